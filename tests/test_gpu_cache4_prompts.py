"""Attention over a 4-bit cache of whole prompts, and of calls whose sequences bring different numbers
of tokens: what a session's first pass and its later ones make of it.

Oracle: the formula in 64 bits; tests/cache_util.attention_bound.
"""

import pytest
import torch

from oracle import cache4
from soupsuck_amd.kernels.paged import PagedCache4, append_kv, cached_attention, read_kv
from tests.cache4_util import NAMES, build4, tokens
from tests.cache_util import DIM, attention_bound, host, offsets

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SCALE = DIM ** -0.5


def _check(device, cache, c, lengths, new, q, cu, window=None, sinks=0):
    """Against the formula over the rows that the cache holds, sequence by sequence."""
    out = cached_attention(q, cache, c.table, c.lengths, cu, max(new), max(lengths), SCALE,
                           window=window, sinks=sinks)
    whole = offsets(lengths, device)
    k, v = read_kv(cache, c.table, c.lengths, whole, sum(lengths))
    group = q.shape[1] // cache.kv_heads
    start = at = 0
    for n, length in zip(new, lengths):
        rows = torch.arange(length, device=device)
        own = torch.arange(length - n, length, device=device)[:, None]
        seen = rows <= own
        if window:
            seen &= (rows > own - window) | (rows < sinks)
        for h in range(q.shape[1]):
            x = q[at:at + n, h].double()
            keys, vals = (t[start:start + length, h // group].double() for t in (k, v))
            s = (x @ keys.t().contiguous() * SCALE).masked_fill(~seen, float("-inf"))
            p = torch.softmax(s, -1) if n else s
            ref, spread = p @ vals, p @ vals.abs()
            reach = float((x.abs() @ keys.abs().t().contiguous()).max() * SCALE) if n else 0.0
            bound = attention_bound(q.dtype, ref, spread, reach, length)
            assert ((out[at:at + n, h].double() - ref).abs() <= bound).all(), (n, length, h)
        start += length
        at += n
    return out


@pytest.mark.parametrize("new,past,hq,hk,page,dtype", [
    ((512,), (0,), 12, 2, 64, F16),
    ((2048,), (1777,), 7, 1, 16, BF16),
    ((1500, 33, 700), (0, 2000, 64), 4, 2, 32, BF16),
    ((1025, 1025), (0, 1), 8, 8, 16, F16),
])
@pytest.mark.parametrize("window,sinks", [(None, 0), (300, 40)])
def test_whole_prompts(device, new, past, hq, hk, page, dtype, window, sinks):
    """A prompt enters the cache and sees itself and what was there, in one call each."""
    print(f"case whole prompts {new} {past} {dtype} {window}", flush=True)
    lengths = [a + b for a, b in zip(new, past)]
    c = build4(lengths, hk, page, device, seed=sum(lengths))
    cache, cu = PagedCache4(c.data, dtype), offsets(new, device)
    k, v = (tokens(sum(new), hk, dtype, device, s) for s in (1, 2))
    q = tokens(sum(new), hq, dtype, device, 3)
    append_kv(cache, k, v, c.table, c.lengths, cu)
    held, _ = read_kv(cache, c.table, c.lengths, cu, sum(new))
    rows = [0, sum(new) // 2, sum(new) - 1]
    assert (host(held[rows]) == cache4.held(host(k[rows]), NAMES[dtype])).all()
    _check(device, cache, c, lengths, new, q, cu, window, sinks)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("others,piece", [(63, 256), (20, 40), (7, 9), (130, 33)])
def test_sequences_of_one_token_beside_a_long_piece(device, others, piece, dtype):
    print(f"case one token beside a long piece {others} {piece} {dtype}", flush=True)
    lengths = [1 + 37 * i % 900 for i in range(others)]
    new = [1] * others
    lengths.insert(others // 2, piece + 511)
    new.insert(others // 2, piece)
    new[0], new[-1] = 0, 0                               # some bring nothing
    c = build4(lengths, 2, 16, device, seed=others)
    q = tokens(sum(new), 14, dtype, device, 3)
    _check(device, PagedCache4(c.data, dtype), c, lengths, new, q, offsets(new, device))
