"""Attention over the paged cache where its work is cut: every block of query rows, ranges that
end inside a sequence, bounds far above the lengths, values that some tokens must not meet.

Oracle and bounds as in tests/test_gpu_cache.py; weights are checked with the outputs.
"""

import numpy as np
import pytest
import torch

from oracle import cache as ocache
from soupsuck_amd.kernels.paged import PagedCache, append_kv, cached_attention, evict_kv
from tests.cache_util import DIM, attention_bound, build, host, offsets
from tests.test_gpu_cache import SCALE, _check_attention, _evict, _tokens

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,new,hq,hk,page,window,sinks,layout", [
    ((2500, 1, 1025, 40), (1, 1, 1, 1), 14, 2, 16, None, 0, "head"),       # 16 rows a block
    ((2500, 1, 1025, 40), (1, 1, 1, 1), 14, 2, 64, 700, 5, "row"),
    ((1400, 33, 1100), (4, 4, 4), 14, 2, 32, None, 0, "head"),             # 32
    ((1400, 1040), (4, 2), 14, 2, 48, 600, 40, "head"),
    ((1300, 50, 1029), (7, 7, 0), 14, 2, 16, None, 0, "row"),              # 64
    ((1300, 1029), (7, 3), 14, 2, 16, 64, 3, "head"),
    ((1111, 700), (19, 13), 14, 2, 64, None, 0, "head"),                   # 128, two blocks
    ((1500,), (70,), 6, 1, 16, 333, 17, "head"),                           # four blocks
    ((1300, 1299), (1, 1), 130, 1, 16, None, 0, "head"),                   # a token over blocks
])
def test_blocks(device, lengths, new, hq, hk, page, window, sinks, layout, dtype):
    print(f"case blocks {lengths} {new} {hq}/{hk} {page} {window} {sinks} {layout}", flush=True)
    c, q, cu, out, _ = _check_attention(device, lengths, new, hq, hk, page, dtype, window, sinks,
                                        layout)
    again = cached_attention(q, PagedCache(c.k, c.v), c.table, c.lengths, cu, max(new),
                             max(lengths), SCALE, window=window, sinks=sinks)
    assert torch.equal(out, again)


@pytest.mark.parametrize("new", [1, 9])
def test_more_sequences_than_lanes(device, new):
    """Seventy lines of ragged lengths, several to a range and ranges inside the long ones."""
    lengths = tuple(new + (1900 if i % 23 == 5 else 13 * i % 210) for i in range(70))
    _check_attention(device, lengths, (new,) * 70, 7, 1, 16, F16, None, 0)


@pytest.mark.parametrize("bound", [4000, 131072, 3 * 10 ** 6, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [1, 4])
def test_bounds_far_above_the_lengths(device, bound, new):
    """Large bounds choose loads past the caches, and keep no scores for the weights."""
    print(f"case bound {bound} {new}", flush=True)
    _check_attention(device, (700, new, 90, 1200), (new,) * 4, 12, 2, 16, BF16, None, 0,
                     max_length=bound)


def test_lengths_beyond_the_bound_are_cut(device):
    c = build((1500, 20), 2, 16, F16, device, seed=2)
    q = _tokens(2, 6, F16, device, 1)
    args = (q, PagedCache(c.k, c.v), c.table, c.lengths, offsets((1, 1), device), 1)
    got = cached_attention(*args, 1100, SCALE)
    # the token's place stays: it sees all of the rows that are left
    want, spread, reach, _ = ocache.attention(
        host(q), host(c.k), host(c.v), c.table.tolist(), [1100, 20], [0, 1, 2], SCALE)
    assert (np.abs(host(got) - want) <= attention_bound(F16, want, spread, reach, 1100)).all()


@pytest.mark.parametrize("bound", [60, 1500])
def test_tokens_outside_the_offsets_and_the_bound_are_zero(device, bound):
    """Packed tokens that no sequence has, and a sequence's tokens past max_new."""
    c = build((50, 40), 2, 16, F16, device, seed=2)
    cache = PagedCache(c.k, c.v)
    q = _tokens(11, 6, F16, device, 1)
    cu = torch.tensor([2, 5, 8], dtype=torch.int32, device=device)
    out = cached_attention(q, cache, c.table, c.lengths, cu, 3, bound, SCALE)
    assert (out[:2] == 0).all() and (out[8:] == 0).all() and (out[2:8] != 0).any(-1).all()
    inner = cached_attention(q[2:8], cache, c.table, c.lengths, offsets((3, 3), device), 3, bound,
                             SCALE)
    assert torch.equal(out[2:8], inner)
    fewer = cached_attention(q, cache, c.table, c.lengths, cu, 2, bound, SCALE)
    assert (fewer[4] == 0).all() and (fewer[7] == 0).all()
    for t in (2, 3, 5, 6):
        assert np.allclose(host(fewer[t]), host(inner[t - 2]), atol=2e-3)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,new,hq", [
    ((75, 60), 6, 6), ((1400, 1105), 6, 6), ((1400, 1105), 9, 12), ((1300, 70), 2, 6),
    ((1500,), 40, 6)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_values_that_some_tokens_see(device, lengths, new, hq, dtype, bad):
    """One infinite or NaN value in the row of a token: the tokens before it are bit for bit as
    without it, those from it on get the value in that column and are as before elsewhere."""
    print(f"case values {lengths} {new} {hq} {dtype} {bad}", flush=True)
    c = build(lengths, 2, 16, dtype, device, seed=3)
    b = len(lengths)
    cu, q = offsets((new,) * b, device), _tokens(new * b, hq, dtype, device, 8)
    args = (q, PagedCache(c.k, c.v), c.table, c.lengths, cu, new, max(lengths), SCALE)
    clean = cached_attention(*args).float()
    which = new // 2
    for row, n in enumerate(lengths):
        j = n - new + which
        c.v[c.table[row, j // 16].item(), :, j % 16, 77] = bad
    out = cached_attention(*args).float()
    for row in range(b):
        seen = slice(new * row + which, new * (row + 1))
        assert torch.equal(out[new * row:seen.start], clean[new * row:seen.start])
        hit = out[seen, :, 77]
        assert torch.isnan(hit).all() if bad != bad else (hit == bad).all()
        rest = [d for d in range(DIM) if d != 77]
        assert torch.equal(out[seen][..., rest], clean[seen][..., rest])


def test_a_window_leaves_bad_rows_behind(device):
    """Rows before some tokens' windows hold infinities and NaN; a missing page lies between."""
    c = build((1400,), 2, 16, F16, device, seed=3)
    cu, q = offsets((8,), device), _tokens(8, 6, F16, device, 8)
    args = (q, PagedCache(c.k, c.v), c.table, c.lengths, cu, 8, 1400, SCALE)
    c.table[0, 40] = -1
    clean = cached_attention(*args, window=1200, sinks=3)
    low = 1400 - 8 - 1200 + 1                     # the first token's lowest row
    for i, bad in ((0, float("nan")), (1, float("inf"))):
        j = low + i                               # seen by tokens 0 .. i
        c.v[c.table[0, j // 16].item(), :, j % 16] = bad
    out = cached_attention(*args, window=1200, sinks=3)
    assert torch.isnan(out[0]).all() and (out[1] == float("inf")).all()
    assert torch.equal(out[2:], clean[2:])


@pytest.mark.parametrize("new", [1, 12])
def test_replays_follow_the_lengths_through_the_cut(device, new):
    """A captured split call with weights: ranges are cut anew from each replay's lengths."""
    c = build((3000, 1700, 90), 2, 16, F16, device, seed=4)
    cu = offsets((new,) * 3, device)
    q = _tokens(3 * new, 12, F16, device, 5)
    cache = PagedCache(c.k, c.v)
    shape = (3, 2, c.table.shape[1] * 16)
    sums, want = (torch.zeros(shape, device=device) for _ in range(2))
    args = (q, cache, c.table, c.lengths, cu, new, 3000, SCALE)
    cached_attention(*args, weights=sums, weights_out=sums)      # warm
    sums.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = cached_attention(*args, weights=sums, weights_out=sums)
    for step, lens in enumerate(((3000, 1700, 90), (20, 1700, 0), (33, 64, 65), (2999, new, 90))):
        c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(_tokens(3 * new, 12, F16, device, 50 + step))
        graph.replay()
        eager = cached_attention(*args, weights=want, weights_out=want)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), step
        assert torch.equal(sums, want), step


def test_a_table_line_of_its_own_stride_and_shared_pages(device):
    """Two sequences with a start in common, named through a table with a gap between lines."""
    c = build((1200, 640), 2, 16, BF16, device, seed=6)
    wide = torch.full((2, 200), -9, dtype=torch.int32, device=device)
    table = wide[:, 7:7 + c.table.shape[1]]
    table.copy_(c.table)
    table[1, :20] = table[0, :20]
    q = _tokens(2, 12, BF16, device, 5)
    cu = offsets((1, 1), device)
    out = cached_attention(q, PagedCache(c.k, c.v), table, c.lengths, cu, 1, 1200, SCALE)
    want, spread, reach, _ = ocache.attention(host(q), host(c.k), host(c.v), table.tolist(),
                                              [1200, 640], [0, 1, 2], SCALE)
    assert (np.abs(host(out) - want) <= attention_bound(BF16, want, spread, reach, 1200)).all()


@pytest.mark.parametrize("length,budget,sinks,recent", [
    (16500, 9000, 4, 100), (16500, 16400, 0, 16), (40000, 5000, 10, 2000)])
def test_evict_around_the_staged_rows(device, length, budget, sinks, recent):
    """More and fewer rows between the ends than LDS holds keys of."""
    _evict(device, (length, 300), 2, 64, F16, budget, sinks, recent)


def test_evict_keeps_the_order_of_equal_weights(device):
    def fill(w):
        w[0] = 0.5
        w[0, 0, 100:200] = 0.5 + 2.0 ** -24
        w[0, 1, 5::7] = -0.25

    _evict(device, (3000,), 2, 16, BF16, 700, 1, 30, fill=fill)


def test_calls_on_streams_of_their_own(device):
    """Append, attention and eviction in order on one side stream equal those on the main one."""
    def run(c):
        k, v = (_tokens(2, 2, F16, device, s) for s in (1, 2))
        cu = offsets((1, 1), device)
        cache = PagedCache(c.k, c.v)
        append_kv(cache, k, v, c.table, c.lengths, cu)
        sums = torch.zeros((2, 2, c.table.shape[1] * 16), device=device)
        out = cached_attention(_tokens(2, 6, F16, device, 3), cache, c.table, c.lengths, cu, 1,
                               1300, SCALE, weights_out=sums)
        to = torch.tensor(c.free[:16], dtype=torch.int32, device=device).view(2, 8)
        return (out, sums, *evict_kv(cache, c.table, c.lengths, sums, to, 128, 1300, sinks=4))

    want = run(build((1300, 40), 2, 16, F16, device, seed=4, spare=16, poison=0.0))
    c = build((1300, 40), 2, 16, F16, device, seed=4, spare=16, poison=0.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(c)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
