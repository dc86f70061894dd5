"""GPU parity of verify_drafts against oracle/cache.py in 64 bits: whole numbers, so equal.

A result can differ only where a number lies within fp64's rounding of a border (about
1e-11 for a vocabulary of 151936); the seeds here have none.
"""

import numpy as np
import pytest
import torch

from oracle import cache as ocache
from soupsuck_amd.kernels.verify import verify_drafts

pytestmark = pytest.mark.gpu


def _case(rows, drafts, vocab, dtype, device, seed, temperature, looked_up, layout="plain"):
    gen = torch.Generator().manual_seed(seed)
    target = (torch.randn((rows, drafts + 1, vocab), generator=gen) * 3).to(dtype)
    draft = (target[:, :drafts].float() + torch.randn((rows, drafts, vocab), generator=gen)).to(dtype)
    source = target[:, :drafts].float() * 2 if looked_up else draft.float()
    noise = torch.rand(source.shape, generator=gen).clamp_(1e-20, 1 - 1e-7)
    tokens = (source / (temperature or 1.0) - noise.log().neg().log()).argmax(-1) if drafts \
        else torch.zeros((rows, 0), dtype=torch.int64)
    uniform = torch.rand((rows, drafts + 1), generator=gen)

    def place(t):
        if layout == "plain":
            return t.to(device)
        wide = torch.full((t.shape[0], t.shape[1] + 1, t.shape[2] + 3), float("nan"), dtype=dtype,
                          device=device)
        view = wide[:, 1:, 1:1 + t.shape[2]]
        view.copy_(t)
        return view

    return place(target), tokens.to(device), uniform.to(device), None if looked_up else place(draft)


def _check(target, tokens, uniform, draft, counts, temperature):
    accepted, out = verify_drafts(target, tokens, uniform, draft_logits=draft, draft_counts=counts,
                                  temperature=temperature)
    host = [None if t is None else t.detach().double().cpu().numpy() for t in (target, draft)]
    seen = set()
    for b in range(target.shape[0]):
        n, want = ocache.verify(host[0][b], tokens[b].tolist(),
                                [0.0] * (tokens.shape[1] + 1) if uniform is None
                                else uniform[b].tolist(),
                                None if draft is None else host[1][b],
                                None if counts is None else int(counts[b]), temperature)
        assert accepted[b].item() == n and out[b].tolist() == want, b
        seen.add(n)
    return accepted, out, seen


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,drafts,vocab,temperature,looked_up,ragged,layout", [
    (3, 4, 1000, 1.0, False, False, "plain"),
    (40, 5, 517, 0.7, False, True, "plain"),
    (40, 3, 64, 1.3, True, True, "plain"),
    (2, 2, 8192, 1.0, False, False, "odd"),
    (2, 2, 8193, 1.0, False, False, "plain"),
    (3, 2, 16389, 0.9, True, False, "odd"),
    (3, 0, 700, 1.0, False, False, "plain"),
    (5, 7, 1, 1.0, False, True, "plain"),
    (20, 4, 333, 0.0, False, True, "plain"),
    (4, 3, 20000, 0.0, True, False, "odd"),
])
def test_matches_oracle(device, rows, drafts, vocab, temperature, looked_up, ragged, layout, dtype):
    print(f"case verify {rows} {drafts} {vocab} {temperature} {looked_up} {layout}", flush=True)
    target, tokens, uniform, draft = _case(rows, drafts, vocab, dtype, device, rows * 7 + drafts,
                                           temperature, looked_up, layout)
    counts = None
    if ragged:
        counts = (torch.arange(rows) % (drafts + 3) - 1).to(torch.int32).to(device)  # -1 .. G + 1
    _check(target, tokens, uniform, draft, counts, temperature)


def test_large_vocabulary(device):
    args = _case(6, 4, 151936, torch.float16, device, 5, 1.0, False)
    _, _, seen = _check(*args, None, 1.0)
    assert len(seen) > 1


@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_logits_that_are_no_ordinary_numbers(device, temperature):
    inf, nan = float("inf"), float("nan")
    target, tokens, uniform, draft = _case(8, 2, 40, torch.float32, device, 2, 1.0, False)
    target[0, 0] = -inf                  # nothing to draw from
    target[1, 0] = nan
    target[2, 0, 5:9] = inf              # the whole shared by four
    tokens[2, 0] = 7
    target[3, :, 1:] = -inf              # one token left
    target[4, 0, ::2] = nan
    draft[5] = -inf                      # a draft without a distribution
    draft[6, 0, 3] = inf
    tokens[6, 0] = 3
    target[7] = draft[7, 0]              # p = q: accepted for every u below 1
    draft[7] = draft[7, 0].clone()
    _, out, _ = _check(target, tokens, uniform, draft, None, temperature)
    assert out[0].tolist() == [-1, -1, -1] and out[1].tolist() == [-1, -1, -1]


def test_tokens_outside_the_vocabulary_are_refused(device):
    target, tokens, uniform, draft = _case(4, 2, 40, torch.float16, device, 3, 1.0, False)
    tokens[0, 0], tokens[1, 1], tokens[2, 0], tokens[3, 0] = -1, 40, 2 ** 40, -2 ** 40
    for d in (draft, None):
        accepted, out, _ = _check(target, tokens, uniform, d, None, 1.0)
        assert accepted.tolist()[0] == 0 and ((out >= -1) & (out < 40)).all()


def test_uniform_at_its_ends(device):
    target, tokens, uniform, draft = _case(3, 2, 300, torch.float16, device, 4, 1.0, False)
    for value in (0.0, 1.0 - 2.0 ** -24, 1.0):
        uniform.fill_(value)
        _check(target, tokens, uniform, draft, None, 1.0)


def test_equal_largest_logits_take_the_lowest(device):
    target = torch.zeros((2, 2, 20000), dtype=torch.float16, device=device)
    target[0, :, [9000, 150, 12000]] = 3.0
    tokens = torch.tensor([[150], [9000]], device=device)
    accepted, out = verify_drafts(target, tokens, temperature=0.0)
    assert accepted.tolist() == [1, 0] and out.tolist() == [[150, 150], [0, -1]]


def test_replays_of_a_graph(device):
    target, tokens, uniform, draft = _case(4, 3, 9000, torch.float16, device, 6, 0.8, False)
    verify_drafts(target, tokens, uniform, draft_logits=draft, temperature=0.8)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = verify_drafts(target, tokens, uniform, draft_logits=draft, temperature=0.8)
    for seed in (7, 8, 9):
        fresh = _case(4, 3, 9000, torch.float16, device, seed, 0.8, False)
        for a, b in zip((target, tokens, uniform, draft), fresh):
            a.copy_(b)
        graph.replay()
        want = verify_drafts(target, tokens, uniform, draft_logits=draft, temperature=0.8)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_frequencies(device):
    """Accepted and drawn tokens together are distributed as p: 4000 checks, 5 deviations."""
    n, vocab = 4000, 12
    gen = torch.Generator().manual_seed(1)
    rows = torch.randn((2, vocab), generator=gen)
    p, q = (torch.softmax(r.double() / 0.9, 0) for r in rows)
    target = rows[0].expand(n, 2, vocab).contiguous().to(device)
    draft = rows[1].expand(n, 1, vocab).contiguous().to(device)
    tokens = torch.multinomial(q, n, replacement=True, generator=gen)[:, None].to(device)
    uniform = torch.rand((n, 2), generator=gen).to(device)
    _, out = verify_drafts(target, tokens, uniform, draft_logits=draft, temperature=0.9)
    seen = np.bincount(out[:, 0].cpu().numpy(), minlength=vocab)
    p = p.numpy()
    assert (np.abs(seen - n * p) < 5 * np.sqrt(n * p * (1 - p))).all()
