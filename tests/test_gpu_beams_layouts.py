"""select_beams in every layout of its launches, next to production vocabularies.

How many rounds a slice has, how many slices a line, and whether a join holds its lines' firsts in
registers, go by the sizes: the cases below name what they reach.  Best tokens and ties are planted
in late rounds, at the ends of slices and in the line's last tokens.

Oracle: the definition in 64 bits.  Candidates that are more than 1e-6 apart, or equal, stand in its
order; closer ones (the kernel's log-sums are good to that) in any.  Scores: an exponential's error
and its sums', 6 2^-23 (see tests/test_gpu_beams.py), and one rounding.
"""

import numpy as np
import pytest
import torch

from soupsuck_amd.kernels.beams import select_beams

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
SUM_ERROR = 6 * 2.0 ** -23
CLOSE = 1e-6
THREADS = 256


def _select(logits, scores, count):
    """(scores, parents, tokens) of the `count` first, or all, of one row in 64 bits."""
    entries = []
    for b, line in enumerate(logits):
        with np.errstate(invalid="ignore"):
            top = line.max()
            whole = top + np.log(np.exp(line - top).sum())
        own = np.where(np.isnan(line), -np.inf, line)
        n = min(count, len(own))
        least = np.partition(own, len(own) - n)[len(own) - n]
        above = np.flatnonzero(own > least)
        tokens = np.concatenate([above, np.flatnonzero(own == least)[:n - len(above)]])
        with np.errstate(invalid="ignore"):
            v = line[tokens] - whole + scores[b]
        v = np.where(np.isnan(v), -np.inf, v)
        entries.append((v, np.full(n, b), own[tokens], tokens))
    v, parents, own, tokens = (np.concatenate(x) for x in zip(*entries))
    order = np.lexsort((tokens, -own, parents, -v))[:count]
    return v[order], parents[order], tokens[order]


def _check_row(got, logits, scores, count):
    want, parents, tokens = _select(logits.double().cpu().numpy(), scores.double().cpu().numpy(),
                                    count + 16)
    value, parent, token = (t.cpu().numpy() for t in got)
    n, fine = count, np.isfinite(want[:count])
    np.testing.assert_array_equal(value[~fine], want[:n][~fine].astype(np.float32))
    error = np.abs(value.astype(np.float64) - want[:n])[fine]
    assert (error <= SUM_ERROR + 2.0 ** -24 * np.abs(want[:n][fine])).all()
    # Runs of candidates that lie close: in any order within the run, unless all are equal.
    with np.errstate(invalid="ignore"):
        gaps = -np.diff(want)
    i = 0
    while i < n:
        end = i + 1
        while end < len(want) and gaps[end - 1] <= CLOSE:
            end += 1
        if (gaps[i:end - 1] > 0).any():
            expected = set(zip(parents[i:end].tolist(), tokens[i:end].tolist()))
            here = list(zip(parent[i:end].tolist(), token[i:end].tolist()))
            assert len(set(here)) == len(here) and set(here) <= expected, f"places {i} .. {end}"
        else:                                   # a place of its own, or equal ones
            last = min(end, n)
            np.testing.assert_array_equal(parent[i:last], parents[i:last])
            np.testing.assert_array_equal(token[i:last], tokens[i:last])
        i = end


def _logits(shape, dtype, device, seed):
    gen = torch.Generator(device).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=device) * 2.5).to(dtype)


def _scores(rows, beams, device, seed):
    return (-8 * torch.rand((rows, beams), generator=torch.Generator().manual_seed(seed))).to(device)


def _places(vocab, slices, width):
    """Ends of the line and of its slices, and the last rounds of each."""
    piece = 16 // width
    each = -(-vocab // slices)
    places = {0, vocab - 1, vocab - 2, vocab - piece, vocab // 2}
    for s in range(slices):
        end = min((s + 1) * each, vocab)
        places |= {s * each, end - 1, max(end - THREADS * piece, 0), (s * each + end) // 2}
    return sorted(p for p in places if 0 <= p < vocab)


@pytest.mark.parametrize("rows,beams,vocab,count,dtype", [
    (1, 4, 151936, 8, F16),             # 75 slices of a line, more than a wave has lanes
    (1, 4, 151935, 5, F32),             # 75 slices of two loads
    (1, 8, 151936, 16, BF16),           # 38 slices, 608 firsts in registers
    (64, 8, 151936, 16, BF16),          # 10 rounds a slice
    (64, 16, 151936, 32, BF16),         # 16 rounds, all that are kept, and 512 candidates at last
    (96, 8, 100003, 3, F32),            # 16 rounds, cut to them
    (1, 1, 400003, 64, F32),            # 832 firsts, reloaded
    (2, 1, 5000017, 64, F32),           # 153 slices, 9792 firsts
    (1, 2, 3000001, 33, BF16),          # 46 slices of 16 rounds, 1518 firsts
])
def test_layouts(device, rows, beams, vocab, count, dtype):
    print(f"case layouts {rows} {beams} {vocab} {count} {dtype}", flush=True)
    logits, scores = _logits((rows, beams, vocab), dtype, device, vocab), _scores(rows, beams,
                                                                                 device, 1)
    got = select_beams(logits, scores, count)
    for row in {0, rows // 2, rows - 1}:
        _check_row([t[row] for t in got], logits[row], scores[row], count)
    # The best of all, equal, where each slice begins and ends (of several numbers of slices).
    for slices in (1, 3, 4, 10, 13, 75):
        places = _places(vocab, slices, logits.element_size())
        row, beam = slices % rows, slices % beams
        logits[row, beam, places] = 15.0
        if beam:
            logits[row, 0, places[::2]] = 15.5
    got = select_beams(logits, scores, count)
    for row in {s % rows for s in (1, 3, 4, 10, 13, 75)}:
        _check_row([t[row] for t in got], logits[row], scores[row], count)


@pytest.mark.parametrize("vocab,count,lines,dtype", [
    (151936, 16, 512, BF16), (151936, 32, 1024, BF16), (100003, 8, 768, F32), (400003, 64, 1, F32)])
def test_best_tokens_of_each_round(device, vocab, count, lines, dtype):
    """A line's best tokens are all in one round, of one thread or of all, each round in turn."""
    print(f"case best tokens of each round {vocab} {count} {lines} {dtype}", flush=True)
    base = _logits((lines, 1, vocab), dtype, device, 3)
    scores = torch.zeros((lines, 1), device=device)
    pass_tokens = THREADS * (16 // base.element_size()) * 2
    starts = list(range(0, vocab - count, pass_tokens))
    for turn in range(0, len(starts), 8):
        logits = base.clone()
        rows = []
        for i, start in enumerate(starts[turn:turn + 8]):
            row = (turn + 7 * i) % lines
            if row in rows:
                continue
            rows.append(row)
            at = torch.arange(count, device=device)
            spread = at if i % 2 else at * ((min(pass_tokens, vocab - start) - 1) // count)
            logits[row, 0, start + spread] = (14 + (at * 7 % count) / 16).to(dtype)
        got = select_beams(logits, scores, count)
        for row in rows:
            _check_row([t[row] for t in got], logits[row], scores[row], count)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("beams,count", [(16, 32), (33, 60), (64, 32), (9, 64), (40, 50)])
@pytest.mark.parametrize("value", [0.0, float("-inf")])
def test_equal_candidates_of_many_beams(device, beams, count, value, dtype):
    """More equal candidates than the last ranking has room for: the lines are merged."""
    vocab = 2049
    logits = torch.full((2, beams, vocab), value, dtype=dtype, device=device)
    for scores in (torch.zeros((2, beams), device=device),
                   torch.full((2, beams), float("-inf"), device=device)):
        got = select_beams(logits, scores, count)
        for row in range(2):
            _check_row([t[row] for t in got], logits[row], scores[row], count)
    # Equal but for some beams: ahead of the others, behind them, not there at all.
    scores = torch.zeros((2, beams), device=device)
    scores[0, 3], scores[0, beams - 1], scores[0, 1] = 1.0, -1.0, float("-inf")
    scores[1, ::2] = float("-inf")
    logits[1, 1, 5:11] = 3.0
    got = select_beams(logits, scores, count)
    for row in range(2):
        _check_row([t[row] for t in got], logits[row], scores[row], count)


def test_few_logits_of_many_beams(device):
    """Lines of fewer tokens than are wanted, all of which are candidates at last."""
    logits = _logits((3, 64, 7), F32, device, 5)
    scores = _scores(3, 64, device, 6)
    got = select_beams(logits, scores, 32)
    for row in range(3):
        _check_row([t[row] for t in got], logits[row], scores[row], 32)
