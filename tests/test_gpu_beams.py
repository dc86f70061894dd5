"""GPU parity of select_beams against oracle/cache4.select in 64 bits.

Parents and tokens are equal where the oracle's candidates lie more than 1e-6 apart or are equal
exactly.  Scores: exponentials in fp32 (an argument d = l - top rounded twice, the constant once and
the instruction's own step: 2^-23 (1 + 1.25 |d|) of terms that weigh exp(d) in the sum, so at
most 2.3 2^-23 of it), sums of eight of them in fp32 (7 2^-24), and one rounding of the score.
"""

import numpy as np
import pytest
import torch

from oracle import cache4
from soupsuck_amd.kernels.beams import select_beams

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
SUM_ERROR = 6 * 2.0 ** -23


def _check(logits, scores, count):
    got = select_beams(logits, scores, count)
    assert [t.dtype for t in got] == [F32, torch.int32, torch.int64]
    assert all(t.shape == (logits.shape[0], count) for t in got)
    x, s = logits.double().cpu().numpy(), scores.double().cpu().numpy()
    for row in range(x.shape[0]):
        want, parents, tokens = cache4.select(x[row], s[row], count)
        value = got[0][row].double().cpu().numpy()
        fine = np.isfinite(want)
        np.testing.assert_array_equal(value[~fine], want[~fine])
        assert (np.abs(value - want)[fine] <= SUM_ERROR + 2.0 ** -24 * np.abs(want[fine])).all()
        np.testing.assert_array_equal(got[1][row].cpu().numpy(), parents)
        np.testing.assert_array_equal(got[2][row].cpu().numpy(), tokens)
    return got


def _logits(shape, dtype, device, seed, std=2.5):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype) \
        .to(device)


def _scores(rows, beams, device, seed):
    return (-8 * torch.rand((rows, beams), generator=torch.Generator().manual_seed(seed))).to(device)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,beams,vocab,count", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 2, 6), (1, 4, 63, 8), (3, 2, 64, 4), (2, 5, 1000, 10),
    (1, 4, 2049, 8), (2, 4, 8191, 64), (1, 2, 32003, 2), (1, 16, 4097, 32), (1, 64, 333, 32),
    (1, 3, 50257, 6),
])
def test_select(device, dtype, rows, beams, vocab, count):
    _check(_logits((rows, beams, vocab), dtype, device, vocab), _scores(rows, beams, device, 1),
           count)


def test_select_large_slices(device):
    """Enough rows that every thread holds its most loads."""
    logits = _logits((48, 8, 40001), BF16, device, 3)
    scores = _scores(48, 8, device, 4)
    got = select_beams(logits, scores, 16)
    for row in (0, 17, 47):
        one = _check(logits[row:row + 1], scores[row:row + 1], 16)
        assert torch.equal(got[1][row], one[1][0]) and torch.equal(got[2][row], one[2][0])
        assert (got[0][row] - one[0][0]).abs().max() <= 2 * SUM_ERROR + 2.0 ** -20


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_select_strides(device, dtype):
    wide = _logits((3, 9, 1111), dtype, device, 5)
    _check(wide[:, 1:9:2, 7:1008], _scores(3, 4, device, 6), 8)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_select_first_step_and_ruled_out_tokens(device, dtype):
    logits = _logits((2, 4, 3001), dtype, device, 7)
    scores = torch.full((2, 4), float("-inf"), device=device)
    scores[:, 0] = 0
    logits[..., 100:2900] = float("-inf")
    _check(logits, scores, 8)
    logits[..., 3:] = float("-inf")                     # three tokens left: the rest are -inf
    _check(logits, scores, 8)
    logits[:] = float("-inf")                           # none
    _check(logits, scores, 8)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_select_equal_logits(device, dtype):
    """Ties everywhere: the lowest beam, then the lowest token."""
    for value in (0.0, -3.0, 11.0):
        logits = torch.full((1, 3, 20011), value, dtype=dtype, device=device)
        _check(logits, torch.zeros((1, 3), device=device), 40)
    logits = torch.zeros((1, 3, 20011), dtype=dtype, device=device)
    logits[..., ::2] = -0.0
    _check(logits, torch.zeros((1, 3), device=device), 40)


@pytest.mark.parametrize("reverse", [False, True])
def test_select_sorted_logits(device, reverse):
    """The best tokens side by side: one thread's own, or one slice's."""
    line = torch.arange(30000, dtype=F32, device=device) * 1e-3
    logits = (line.flip(0) if reverse else line).repeat(2, 3, 1)
    logits = logits + torch.arange(3, device=device)[:, None] * 0.1
    _check(logits.contiguous(), _scores(2, 3, device, 2), 64)
    # and spread so that a few lanes hold them all
    spread = torch.full((1, 1, 32768), -50.0, device=device)
    for lane in range(8):
        at = torch.arange(8, device=device)[:, None] * 2048 + lane * 8 + torch.arange(
            8, device=device)
        spread[0, 0, at.flatten()] = torch.arange(64, dtype=F32, device=device) * 0.01 + lane
    _check(spread, torch.zeros((1, 1), device=device), 64)
    _check(spread.to(F16), torch.zeros((1, 1), device=device), 64)


def test_select_not_numbers(device):
    logits = _logits((6, 3, 2500), F32, device, 9)
    logits[0, 1, 77] = float("nan")                     # its beam counts as -inf
    logits[1, 0, 2000] = float("inf")
    logits[2, :, 5] = float("nan")                      # all of them
    logits[3, 2] = float("-inf")
    logits[4, 0] = float("nan")
    scores = _scores(6, 3, device, 10)
    scores[5, 1] = float("nan")
    scores[3, 0] = float("inf")
    _check(logits, scores, 12)


def test_select_extreme_scores(device):
    """Large logits; beams that are told apart by fp32's last bit; scores that swallow logits."""
    logits = _logits((1, 1, 3000), F16, device, 11).repeat(1, 4, 1).contiguous()
    scores = torch.tensor([[-5.0, -5.0 - 2.0 ** -21, -5.0, -5.0 + 2.0 ** -21]], device=device)
    _check(logits, scores, 24)
    _check(logits * 2000, scores, 24)
    _check(logits.float() * 1e30, scores, 24)
    _check(logits.float(), torch.tensor([[-1e9, -1e9, 0.0, -1e30]], device=device), 24)


def test_select_no_rows(device):
    got = select_beams(torch.zeros((0, 2, 10), device=device), torch.zeros((0, 2), device=device), 4)
    assert [t.shape for t in got] == [(0, 4)] * 3


def test_select_replayed(device):
    logits, scores = _logits((2, 4, 9001), BF16, device, 12), _scores(2, 4, device, 13)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        select_beams(logits, scores, 8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = select_beams(logits, scores, 8)
    for seed in (1, 2, 3):
        logits.copy_(_logits((2, 4, 9001), BF16, device, 50 + seed))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, select_beams(logits, scores, 8)):
            assert torch.equal(a, b)
