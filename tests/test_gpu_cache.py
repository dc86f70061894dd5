"""GPU parity of the paged cache: append, attention of new tokens, eviction.

Oracle: oracle/cache.py in 64 bits on the same inputs.  Appended keys: the rotation's two
products and one sum in fp32 (3 half steps of fp32 of |x cos| + |x sin|) and one rounding;
values bit for bit.  Attention: tests/cache_util.attention_bound.  Accumulated weights: fp32 sums of
probabilities.  Eviction: exact.  Rows that no query sees are NaN in every cache here.
"""

import numpy as np
import pytest
import torch

from oracle import cache as ocache
from soupsuck_amd.kernels.paged import PagedCache, append_kv, cached_attention, evict_kv
from tests.cache_util import DIM, HALF_STEP, attention_bound, build, host, offsets

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
SCALE = DIM ** -0.5


def _tokens(count, heads, dtype, device, seed, layout="plain"):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((count, heads, DIM), generator=gen).to(dtype)
    if layout == "plain":
        return x.to(device)
    wide = torch.full((count, heads + 2, DIM + 16), float("nan"), dtype=dtype, device=device)
    view = wide[:, 1:1 + heads, 8:8 + DIM]
    view.copy_(x)
    return view


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("new,past,hq,hk,page,dtype,cs,layout", [
    ((1,), (0,), 12, 2, 16, F16, F16, "head"),
    ((1,), (63,), 12, 2, 64, F16, F16, "head"),
    ((1, 1, 1, 1, 1), (0, 15, 16, 17, 129), 28, 4, 16, BF16, BF16, "row"),
    ((7, 0, 40, 1), (5, 9, 0, 100), 6, 2, 32, BF16, torch.float32, "head"),
    ((33, 16), (15, 1), 4, 4, 48, F16, torch.float32, "row"),
    ((5,), (0,), 3, 1, 16, F16, F16, "row"),
])
def test_append(device, new, past, hq, hk, page, dtype, cs, layout):
    lens = [a + b for a, b in zip(new, past)]
    c = build(lens, hk, page, dtype, device, seed=sum(lens), layout=layout)
    cu, total = offsets(new, device), sum(new)
    k, v = (_tokens(total, hk, dtype, device, i, layout) for i in (1, 2))
    q = _tokens(total, hq, dtype, device, 3, layout)
    angle = torch.rand((total, DIM), generator=torch.Generator().manual_seed(4)) * 6.3
    cos, sin = (f(angle).to(cs).to(device) for f in (torch.cos, torch.sin))
    args = (host(c.k), host(c.v), host(k), host(v), c.table.tolist(), lens, cu.tolist())
    plain_k, want_v = ocache.append(*args)
    want_k, _ = ocache.append(*args, host(cos), host(sin))
    bystander = host(c.k)
    got = append_kv(PagedCache(c.k, c.v), k, v, c.table, c.lengths, cu, q=q, cos=cos, sin=sin)
    np.testing.assert_array_equal(host(c.v), want_v)

    def close(actual, want, size):
        bound = HALF_STEP[dtype] * np.abs(want) * 1.001 + 3 * 2.0 ** -24 * size
        assert (np.abs(actual - want) <= bound + 2.0 ** -25).all()

    wrote = ~((plain_k == bystander) | (np.isnan(plain_k) & np.isnan(bystander)))
    rest = ~wrote & ~np.isnan(want_k)
    np.testing.assert_array_equal(np.isnan(host(c.k)), np.isnan(want_k))
    close(host(c.k)[wrote], want_k[wrote], 10.0)
    close(host(c.k)[rest], want_k[rest], 10.0)
    close(host(got), ocache.rotate(host(q), host(cos)[:, None], host(sin)[:, None]), 10.0)
    # unrotated: bit for bit
    assert append_kv(PagedCache(c.k, c.v), k, v, c.table, c.lengths, cu) is None
    np.testing.assert_array_equal(host(c.k), plain_k)


def test_append_skips_rows_that_no_page_holds(device):
    c = build([20, 20, 20], 2, 16, F16, device, seed=1)
    c.table[0, 1] = -1
    c.table[1, 1] = 10 ** 6
    c.lengths[2] = 50                      # its rows 46 .. 49 lie behind the table
    before = c.k.clone(), c.v.clone()
    k = _tokens(12, 2, F16, device, 1)
    append_kv(PagedCache(c.k, c.v), k, k, c.table, c.lengths, offsets([4, 4, 4], device))
    for now, then in zip((c.k, c.v), before):
        assert torch.equal(now.view(torch.int16), then.view(torch.int16))
    # more tokens than rows: only the last two have one
    c.lengths[:] = torch.tensor([2, 0, -3], dtype=torch.int32)
    append_kv(PagedCache(c.k, c.v), k, k, c.table, c.lengths, offsets([4, 4, 4], device))
    assert torch.equal(c.k[c.table[0, 0].item(), :, :2], k[2:4].transpose(0, 1))
    changed = (c.k.view(torch.int16) != before[0].view(torch.int16)).any(-1).any(1)
    assert changed.sum().item() == 2


# --------------------------------------------------------------- attention

def _check_attention(device, lengths, new, hq, hk, page, dtype, window, sinks, layout="head",
                     seed=0, weights=True, change=None, scale=SCALE, spread_scale=1.0,
                     max_length=None):
    c = build(lengths, hk, page, dtype, device, seed=seed + 17, layout=layout, extra_pages=1,
              scale=spread_scale)
    if change is not None:
        change(c)
    cu, total = offsets(new, device), sum(new)
    q = _tokens(total, hq, dtype, device, seed, layout)
    ref, spread, reach, w = ocache.attention(host(q), host(c.k), host(c.v), c.table.tolist(),
                                             c.lengths.tolist(), cu.tolist(), scale, window, sinks)
    base = torch.rand(w.shape, generator=torch.Generator().manual_seed(5)).to(device)
    sums = torch.full_like(base, float("nan")) if weights else None
    if max_length is None:
        max_length = max([*lengths, 0])
    out = cached_attention(q, PagedCache(c.k, c.v), c.table, c.lengths, cu, max(new), max_length,
                           scale, window=window, sinks=sinks,
                           weights=base if weights else None, weights_out=sums)
    got = host(out)
    bound = attention_bound(dtype, ref, spread, reach, max_length)
    worst = np.abs(got - ref) / bound if got.size else np.zeros(1)
    assert not np.isnan(got).any() and worst.max() <= 1, f"{worst.max()} of the bound"
    if weights:
        error = 2 * 2.0 ** -24 * (128 * reach + 4 * (1 + reach) + max_length)
        bound = w * error + 2 * 2.0 ** -24 * (host(base) + w) + 1e-12
        assert (np.abs(host(sums) - (host(base) + w)) <= bound).all()
    return c, q, cu, out, sums


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,new,hq,hk,page,window,sinks,layout", [
    ((1,), (1,), 12, 2, 64, None, 0, "head"),
    ((31,), (1,), 12, 2, 16, None, 0, "row"),
    ((32, 33, 64, 65, 127, 128, 129, 1), (1,) * 8, 28, 4, 16, None, 0, "head"),
    ((518,), (1,), 12, 2, 64, None, 0, "head"),
    ((1500, 3, 700), (1, 1, 1), 8, 8, 32, None, 0, "row"),
    ((300, 77), (1, 1), 16, 1, 48, None, 0, "head"),           # one kv head for sixteen
    ((260, 41), (1, 1), 40, 2, 16, None, 0, "head"),           # groups of twenty
    ((90, 5, 200), (5, 5, 5), 12, 2, 32, None, 0, "head"),     # drafts
    ((90, 7, 200, 64), (3, 0, 8, 1), 28, 4, 16, None, 0, "row"),
    ((150,), (150,), 6, 2, 16, None, 0, "head"),               # a whole prompt
    ((400, 129), (70, 33), 7, 1, 64, None, 0, "head"),
    ((700, 40, 1100), (1, 1, 1), 12, 2, 16, 100, 4, "head"),   # window and sinks
    ((700, 40, 1100), (1, 1, 1), 12, 2, 32, 64, 0, "row"),
    ((500, 300), (5, 9), 12, 2, 16, 33, 70, "head"),           # sinks longer than the window
    ((333,), (40,), 4, 2, 16, 1, 0, "head"),                   # only the token itself
    ((333,), (40,), 4, 2, 16, 17, 2, "head"),
])
def test_attention(device, lengths, new, hq, hk, page, window, sinks, layout, dtype):
    print(f"case attention {lengths} {new} {hq}/{hk} {page} {window} {sinks} {layout}", flush=True)
    c, q, cu, out, sums = _check_attention(device, lengths, new, hq, hk, page, dtype, window,
                                           sinks, layout)
    again = cached_attention(q, PagedCache(c.k, c.v), c.table, c.lengths, cu, max(new),
                             max(lengths), SCALE, window=window, sinks=sinks)
    assert torch.equal(out, again)            # weights change nothing, and the order is fixed


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_long_and_many(device, dtype):
    _check_attention(device, (20011, 31, 4097, 1), (1, 1, 1, 1), 14, 2, 64, dtype, None, 0)
    _check_attention(device, tuple(17 * i + 1 for i in range(70)), (1,) * 70, 7, 1, 16, dtype,
                     None, 0)


@pytest.mark.parametrize("new", [1, 4])
def test_rows_that_see_nothing_are_zero(device, new):
    """Empty sequences, sequences shorter than their tokens, sequences without pages."""

    def change(c):
        c.lengths[1] = -5
        c.table[3, :] = -1
        c.table[4, :] = 10 ** 7

    c, _, _, out, sums = _check_attention(device, (0, 0, new - 1, 40, 40, 20), (new,) * 6, 6, 2,
                                          16, F16, None, 0, change=change)
    assert (out[:2 * new] == 0).all() and (out[3 * new:5 * new] == 0).all()
    assert (out[2 * new] == 0).all()


def test_a_missing_page_inside_a_sequence(device):
    def change(c):
        c.table[0, 1] = -1
        c.table[0, 3] = -7

    _check_attention(device, (200,), (3,), 12, 2, 16, BF16, None, 0, change=change)


def test_pages_behind_the_window_may_be_given_back(device):
    def change(c):
        c.table[0, 1:9] = -1               # rows 16 .. 143

    _check_attention(device, (400,), (2,), 12, 2, 16, F16, 200, 4, change=change)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_what_is_not_seen_has_no_part(device, bad, dtype):
    """Unseen rows inside seen tiles: later tokens' rows and rows before the window."""
    lengths, new = (75, 60), (6, 6)

    def change(c):
        # the last token's own row: the five tokens before it must not notice
        for b, n in enumerate(lengths):
            page, row = c.table[b, (n - 1) // 16].item(), (n - 1) % 16
            c.k[page, :, row] = bad
            c.v[page, :, row] = bad

    c = build(lengths, 2, 16, dtype, device, seed=3)
    cu = offsets(new, device)
    q = _tokens(12, 6, dtype, device, 8)
    clean = cached_attention(q, PagedCache(c.k, c.v), c.table, c.lengths, cu, 6, 75, SCALE)
    change(c)
    out = cached_attention(q, PagedCache(c.k, c.v), c.table, c.lengths, cu, 6, 75, SCALE)
    for b in range(2):
        assert torch.equal(out[6 * b:6 * b + 5], clean[6 * b:6 * b + 5])
        assert torch.isnan(out[6 * b + 5]).all() or bad == float("-inf")
    # rows before the window of later tokens, seen by earlier ones
    c = build(lengths, 2, 16, dtype, device, seed=3)
    args = (PagedCache(c.k, c.v), c.table, c.lengths, cu, 6, 75, SCALE)
    clean = cached_attention(q, *args, window=20, sinks=2)
    for b, n in enumerate(lengths):
        j = n - 6 - 19                      # seen by the first token only
        c.k[c.table[b, j // 16].item(), :, j % 16] = bad
        c.v[c.table[b, j // 16].item(), :, j % 16] = bad
    out = cached_attention(q, *args, window=20, sinks=2)
    for b in range(2):
        assert torch.equal(out[6 * b + 1:6 * b + 6], clean[6 * b + 1:6 * b + 6])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_dominating_key_and_a_long_tail(device, dtype):
    """Thousands of weights of 1e-6 beside one of nearly 1: together they count."""
    n = 9000
    c = build((n,), 1, 64, dtype, device, seed=9, scale=0.05)
    q = _tokens(1, 4, dtype, device, 2)
    at = c.table[0, 0].item()
    c.k[at, 0, 7] = (q[0, 0] * 1.2).to(dtype)
    cu = offsets([1], device)
    ref, spread, reach, _ = ocache.attention(host(q), host(c.k), host(c.v), c.table.tolist(), [n],
                                             [0, 1], SCALE)
    out = host(cached_attention(q, PagedCache(c.k, c.v), c.table, c.lengths, cu, 1, n, SCALE))
    assert (np.abs(out - ref) <= attention_bound(dtype, ref, spread, reach, n)).all()


@pytest.mark.parametrize("scale", [0.0, -0.09, 3.0])
def test_scales(device, scale):
    _check_attention(device, (100, 45), (1, 4), 12, 2, 16, F16, 40, 3, scale=scale)


def test_lengths_are_read_when_the_kernel_runs(device):
    """A captured call follows lengths, table and tokens of the moment; weights accumulate."""
    c = build((500, 130), 2, 16, F16, device, seed=4)
    cu = offsets((1, 1), device)
    q = _tokens(2, 12, F16, device, 5)
    cache = PagedCache(c.k, c.v)
    shape = (2, 2, c.table.shape[1] * 16)
    sums = torch.zeros(shape, device=device)
    args = (q, cache, c.table, c.lengths, cu, 1, 500, SCALE)
    cached_attention(*args, weights=sums, weights_out=sums)      # warm
    graph = torch.cuda.CUDAGraph()
    sums.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = cached_attention(*args, weights=sums, weights_out=sums)
    want = torch.zeros(shape, device=device)
    for step, lens in enumerate(((500, 130), (480, 1), (17, 100), (33, 0), (499, 128))):
        c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(_tokens(2, 12, F16, device, 50 + step))
        graph.replay()
        eager = cached_attention(*args, weights=want, weights_out=want)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), step
        assert torch.equal(sums, want), step


def test_another_stream(device):
    c = build((700,), 2, 16, F16, device, seed=4)
    q = _tokens(1, 12, F16, device, 5)
    args = (q, PagedCache(c.k, c.v), c.table, c.lengths, offsets((1,), device), 1, 700, SCALE)
    want = cached_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cached_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_offsets_past_32_bits(device):
    """A sequence in the last pages of a cache of more than 4 GiB a tensor (2^31 elements)."""
    pages = 2 ** 31 // (64 * 4 * DIM) + 40
    k = torch.zeros((pages, 4, 64, DIM), dtype=F16, device=device)
    v = torch.zeros_like(k)
    c = build((150,), 4, 64, F16, device, seed=6)
    order = [pages - 1, pages - 30, 3]
    for i, p in enumerate(order):
        k[p], v[p] = c.k[c.table[0, i]], c.v[c.table[0, i]]
    table = torch.tensor([order], dtype=torch.int32, device=device)
    q = _tokens(1, 8, F16, device, 5)
    cu = offsets((1,), device)
    want = cached_attention(q, PagedCache(c.k, c.v), c.table, c.lengths, cu, 1, 150, SCALE)
    assert torch.equal(cached_attention(q, PagedCache(k, v), table, c.lengths, cu, 1, 150, SCALE),
                       want)
    new = _tokens(1, 4, F16, device, 9)
    append_kv(PagedCache(k, v), new, new, table, torch.tensor([1], dtype=torch.int32,
                                                              device=device), cu)
    assert torch.equal(k[pages - 1, :, 0], new[0]) and torch.equal(v[pages - 1, :, 0], new[0])
    weights = torch.zeros((1, 4, 192), device=device)
    to = torch.tensor([[pages - 2]], dtype=torch.int32, device=device)
    evict_kv(PagedCache(k, v), table, c.lengths, weights, to, 64, 150, recent=64)
    tail = torch.cat((k[pages - 30], k[3]), 1)[:, 150 - 64 - 64:150 - 64]
    assert torch.equal(k[pages - 2], tail)


# ---------------------------------------------------------------- eviction

def _evict(device, lengths, heads, page, dtype, budget, sinks, recent, layout="head", change=None,
           fill=None, max_length=None):
    need = len(lengths) * -(-budget // page)
    c = build(lengths, heads, page, dtype, device, seed=sum(lengths), spare=need + 2,
              layout=layout, extra_pages=1)
    to = torch.tensor(c.free[:need], dtype=torch.int32, device=device).view(len(lengths), -1)
    w = torch.rand((len(lengths), heads, c.table.shape[1] * page),
                   generator=torch.Generator().manual_seed(7))
    w = (w * 40).round() / 40            # many ties
    if fill is not None:
        fill(w)
    w = w.to(device)
    if change is not None:
        change(c, to)
    lens = [min(n, max_length) if max_length is not None else n for n in c.lengths.tolist()]
    want = ocache.evict(host(c.k), host(c.v), c.table.tolist(), lens, w.cpu().numpy(),
                        to.tolist(), budget, sinks, recent)
    got = evict_kv(PagedCache(c.k, c.v), c.table, c.lengths, w, to, budget,
                   max([*lengths, 0]) if max_length is None else max_length, sinks=sinks,
                   recent=recent)
    np.testing.assert_array_equal(got[0].cpu().numpy(), want[0])
    np.testing.assert_array_equal(got[1].cpu().numpy(), want[1])
    np.testing.assert_array_equal(host(c.k), want[2])
    np.testing.assert_array_equal(host(c.v), want[3])
    return c, w, got


@pytest.mark.parametrize("lengths,heads,page,dtype,budget,sinks,recent,layout", [
    ((100,), 2, 16, F16, 40, 4, 16, "head"),
    ((1, 0, 40, 41, 300), 2, 16, BF16, 40, 0, 0, "row"),
    ((65, 64, 63), 1, 32, F16, 64, 4, 60, "head"),     # nothing between the ends
    ((129, 500), 3, 64, F16, 1, 0, 0, "head"),          # a single row
    ((129, 500), 3, 64, F16, 1, 0, 1, "head"),
    ((777, 2000), 4, 16, BF16, 600, 16, 100, "row"),
    ((5000,), 2, 64, F16, 4999, 4, 64, "head"),         # one row goes
    ((9000, 3000), 1, 128, F16, 2000, 0, 0, "head"),
])
def test_evict(device, lengths, heads, page, dtype, budget, sinks, recent, layout):
    _evict(device, lengths, heads, page, dtype, budget, sinks, recent, layout)


def test_evict_weights_that_are_no_ordinary_numbers(device):
    def fill(w):
        w[0, 0, 10:30] = float("inf")
        w[0, 0, 40:50] = float("nan")
        w[0, 1, ::2] = 0.0
        w[0, 1, 1::2] = -0.0                 # equal to 0: the lowest rows stay
        w[0, 1, 60] = -1.0
        w[0, 1, 61] = float("-inf")
        w[0, 1, 62] = -float("nan")
        w[1] = 0.25                          # all equal
        w[2, :, 5] = 1e-42                   # the least there is above 0
        w[2, :, 6] = 0.0

    _evict(device, (90, 80, 70), 2, 16, F16, 33, 2, 5, fill=fill)


def test_evict_bad_pages_and_lengths(device):
    def change(c, to):
        c.table[0, 1] = -1                   # rows that no page holds are kept as zeros
        to[1, 1] = -1                        # rows that have nowhere to go are dropped
        to[2, 0] = 10 ** 6
        c.lengths[3] = 10 ** 6               # cut to the table

    _evict(device, (60, 60, 60, 60), 2, 16, F16, 40, 4, 10, change=change, max_length=10 ** 6)


def test_evict_bound_on_the_length(device):
    _evict(device, (100, 50), 2, 16, F16, 30, 4, 10, max_length=64)


def test_the_cycle_of_a_bounded_cache(device):
    """Append, attend with weights, evict: attention over the compacted cache is attention over
    the kept rows."""
    c, w, (lens, sums) = _evict(device, (300, 200), 2, 16, F16, 128, 4, 32)
    to = torch.tensor(c.free[:16], dtype=torch.int32, device=device).view(2, 8)
    q = _tokens(2, 12, F16, device, 3)
    cu = offsets((1, 1), device)
    out = cached_attention(q, PagedCache(c.k, c.v), to, lens, cu, 1, 128, SCALE, weights=sums,
                           weights_out=sums)
    ref, spread, reach, step = ocache.attention(host(q), host(c.k), host(c.v), to.tolist(),
                                                lens.tolist(), [0, 1, 2], SCALE)
    assert (np.abs(host(out) - ref) <= attention_bound(F16, ref, spread, reach, 128)).all()
    assert np.isclose(step.sum(), 24)
