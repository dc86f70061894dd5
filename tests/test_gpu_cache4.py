"""GPU parity of the 4-bit paged cache: append, reading back, attention of new tokens.

Oracle: oracle/cache4.py and oracle/cache.py in 64 bits.  Codes and scales are exact: the rotation
that they are taken from has exact products and one rounding in fp64, here and there.
Attention is that over a 16-bit cache with the same values, which 16 bits hold exactly:
tests/cache_util.attention_bound.  Rows that no query sees are NaN.
"""

import numpy as np
import pytest
import torch

from oracle import cache as ocache
from oracle import cache4
from soupsuck_amd.kernels.paged import (PagedCache, PagedCache4, append_kv, cached_attention,
                                        read_kv)
from tests.cache4_util import NAMES, build4, random_bytes, tokens, values
from tests.cache_util import DIM, HALF_STEP, attention_bound, build, host, offsets

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
SCALE = DIM ** -0.5


# ------------------------------------------------------------------ append

def _want(data, k, v, table, lengths, cu, dtype):
    """The bytes after append of k / v [T, heads, 128] (64 bits)."""
    out = data.copy()
    pages, heads, groups, _ = data.shape
    size = groups * 16
    for b, length in enumerate(lengths):
        for t in range(cu[b], cu[b + 1]):
            row = length - cu[b + 1] + t
            if not 0 <= row < len(table[b]) * size or not 0 <= table[b][row // size] < pages:
                continue
            for h in range(heads):
                cache4.pack(out, table[b][row // size], h, row % size, k[t, h], v[t, h],
                            NAMES[dtype])
    return out


def _same_bytes(got, want):
    """Equal bytes, the codes of NaN blocks (which count for nothing) and signs of zeros aside."""
    for a, b in zip(cache4.unpack(got), cache4.unpack(want)):
        np.testing.assert_array_equal(a, b)
    np.testing.assert_array_equal(got[..., 2048:], want[..., 2048:])


@pytest.mark.parametrize("new,past,hq,hk,page,dtype,cs,strided", [
    ((1,), (0,), 12, 2, 16, F16, F16, False),
    ((1,), (63,), 12, 2, 64, F16, F16, False),
    ((1, 1, 1, 1, 1), (0, 15, 16, 17, 129), 28, 4, 16, BF16, BF16, True),
    ((7, 0, 40, 1), (5, 9, 0, 100), 6, 2, 32, BF16, torch.float32, False),
    ((33, 16), (15, 1), 4, 4, 48, F16, torch.float32, True),
    ((5,), (0,), 3, 1, 16, F16, F16, True),
])
def test_append(device, new, past, hq, hk, page, dtype, cs, strided):
    lens = [a + b for a, b in zip(new, past)]
    c = build4(lens, hk, page, device, seed=sum(lens), layout="gaps" if strided else "plain")
    cu, total = offsets(new, device), sum(new)
    k, v = (tokens(total, hk, dtype, device, i, strided, scale=3.0) for i in (1, 2))
    q = tokens(total, hq, dtype, device, 3, strided)
    angle = torch.rand((total, DIM), generator=torch.Generator().manual_seed(4)) * 6.3
    cos, sin = (f(angle).to(cs).to(device) for f in (torch.cos, torch.sin))
    before = c.data.cpu().numpy().copy()
    turned = ocache.rotate(host(k), host(cos)[:, None], host(sin)[:, None])
    args = (c.table.tolist(), lens, cu.tolist(), dtype)
    cache = PagedCache4(c.data, dtype)
    got = append_kv(cache, k, v, c.table, c.lengths, cu, q=q, cos=cos, sin=sin)
    _same_bytes(c.data.cpu().numpy(), _want(before, turned, host(v), *args))
    want_q = ocache.rotate(host(q), host(cos)[:, None], host(sin)[:, None])
    assert (np.abs(host(got) - want_q)
            <= HALF_STEP[dtype] * np.abs(want_q) * 1.001 + 3 * 2.0 ** -24 * 10 + 2.0 ** -25).all()
    # read back, bit for bit; then without a rotation
    held_k, held_v = read_kv(cache, c.table, c.lengths, cu, total)
    np.testing.assert_array_equal(host(held_k), cache4.held(turned, NAMES[dtype]))
    np.testing.assert_array_equal(host(held_v), cache4.held(host(v), NAMES[dtype]))
    assert append_kv(cache, k, v, c.table, c.lengths, cu) is None
    _same_bytes(c.data.cpu().numpy(), _want(before, host(k), host(v), *args))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_next_to_borders_and_ends(device, dtype):
    """Ties, blocks of zeros, the ends of the range, infinities and NaN."""
    low, high = cache4.EXPONENTS[NAMES[dtype]]
    top = torch.finfo(dtype).max
    rows = torch.zeros((14, 1, DIM), dtype=torch.float64)
    middles = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    rows[1, 0] = middles.repeat(16)
    rows[2, 0] = middles.repeat(16) * -(2.0 ** 3)
    rows[3, 0] = middles.repeat(16) * 2.0 ** low          # 0.25 2^low is not zero in the type
    rows[4, 0, ::3] = top
    rows[5, 0, 5], rows[5, 0, 99] = -top, top / 2
    rows[6, 0, 7] = float("inf")
    rows[7, 0, 70] = float("nan")
    rows[8, 0, 127], rows[8, 0, 3] = float("-inf"), 2.0
    rows[9, 0] = torch.finfo(dtype).tiny
    rows[10, 0] = torch.finfo(dtype).smallest_normal / 2
    rows[11, 0] = 1.5 * 4 * (1 + torch.finfo(dtype).eps)  # just past 6
    rows[12, 0] = 6.0
    rows[13, 0] = 7.0
    k = rows.to(dtype).to(device)
    c = build4([14], 1, 16, device, seed=1)
    before = c.data.cpu().numpy().copy()
    cu = offsets([14], device)
    cache = PagedCache4(c.data, dtype)
    append_kv(cache, k, -k, c.table, c.lengths, cu)
    _same_bytes(c.data.cpu().numpy(),
                _want(before, host(k), -host(k), c.table.tolist(), [14], [0, 14], dtype))
    held_k, held_v = read_kv(cache, c.table, c.lengths, cu, 14)
    np.testing.assert_array_equal(host(held_k), cache4.held(host(k), NAMES[dtype]))
    np.testing.assert_array_equal(host(held_v), cache4.held(-host(k), NAMES[dtype]))
    # a rotation past the type's range is no infinity
    cos = torch.ones((14, DIM), dtype=torch.float32, device=device)
    append_kv(cache, k, k, c.table, c.lengths, cu, cos=cos, sin=-cos)
    turned = ocache.rotate(host(k), host(cos)[:, None], -host(cos)[:, None])
    held_k, _ = read_kv(cache, c.table, c.lengths, cu, 14)
    np.testing.assert_array_equal(host(held_k), cache4.held(turned, NAMES[dtype]))


def test_append_rotation_is_not_rounded_before_the_codes(device):
    """Sums that lie next to a border by less than fp32 can tell."""
    k = torch.zeros((4, 1, DIM), dtype=BF16)
    k[:, 0, 0] = 6.0                                     # scale 1
    k[:, 0, 1], k[:, 0, 65] = 2.5, 1.0
    cos, sin = torch.ones((4, DIM)), torch.zeros((4, DIM))
    sin[:, 1] = torch.tensor([2.0 ** -30, -(2.0 ** -30), 0.0, 2.0 ** -24])
    c = build4([4], 1, 16, device, seed=1)
    cu = offsets([4], device)
    cache = PagedCache4(c.data, BF16)
    append_kv(cache, k.to(device), k.to(device), c.table, c.lengths, cu, cos=cos.to(device),
              sin=sin.to(device))
    held, _ = read_kv(cache, c.table, c.lengths, cu, 4)
    assert held[:, 0, 1].tolist() == [2.0, 3.0, 2.0, 2.0]


def test_append_skips_rows_that_no_page_holds(device):
    c = build4([20, 20, 20], 2, 16, device, seed=1)
    c.table[0, 1] = -1
    c.table[1, 1] = 10 ** 6
    c.lengths[2] = 50                      # its rows 46 .. 49 lie behind the table
    before = c.data.clone()
    cache = PagedCache4(c.data, F16)
    k = tokens(12, 2, F16, device, 1)
    cu = offsets([4, 4, 4], device)
    append_kv(cache, k, k, c.table, c.lengths, cu)
    assert torch.equal(c.data, before)
    held_k, held_v = read_kv(cache, c.table, c.lengths, cu, 12)
    assert (held_k == 0).all() and (held_v == 0).all()
    # more tokens than rows: only the last two have one
    c.lengths[:] = torch.tensor([2, 0, -3], dtype=torch.int32)
    append_kv(cache, k, k, c.table, c.lengths, cu)
    want = before.cpu().numpy().copy()
    for row in range(2):
        for h in range(2):
            cache4.pack(want, c.table[0, 0].item(), h, row, host(k[2 + row, h]),
                        host(k[2 + row, h]), "float16")
    _same_bytes(c.data.cpu().numpy(), want)


# -------------------------------------------------------------------- read

@pytest.mark.parametrize("four", [True, False])
def test_read_whole_sequences_of_several_layers(device, four):
    lens = [40, 0, 17, 1]
    layers = 67                                          # more than a launch takes
    c = build4(lens, 2, 16, device, seed=5) if four else build(lens, 2, 16, F16, device, seed=5)
    c.table[0, 1] = -1                                   # rows 16 .. 31 are not held
    total = sum(lens)
    cu = offsets([*lens], device)
    caches, want = [], []
    for layer in range(layers):
        if four:
            data = torch.from_numpy(random_bytes(tuple(c.data.shape), layer)).to(device)
            caches.append(PagedCache4(data, BF16))
            k, v = values(data) if layer in (0, 1, 63, 64, 66) else (None, None)
        else:
            k, v = torch.randn_like(c.k), torch.randn_like(c.v)
            caches.append(PagedCache(k, v))
            k, v = host(k), host(v)
        want.append((k, v))
    k, v = read_kv(caches, c.table, c.lengths, cu, total + 2)
    assert k.shape == v.shape == (layers, total + 2, 2, DIM)
    one = read_kv(caches[3], c.table, c.lengths, cu, total + 2)
    assert torch.equal(one[0], k[3]) and torch.equal(one[1], v[3])
    table = c.table.tolist()
    for layer, (wk, wv) in enumerate(want):
        if wk is None:
            continue
        for got, ref in ((host(k[layer]), wk), (host(v[layer]), wv)):
            rows = [ref[table[b][j // 16], :, j % 16] if table[b][j // 16] >= 0
                    else np.zeros((2, DIM)) for b, n in enumerate(lens) for j in range(n)]
            np.testing.assert_array_equal(got[:total], np.array(rows))
            assert (got[total:] == 0).all()              # tokens that no sequence has


# --------------------------------------------------------------- attention

def check_attention(device, lengths, new, hq, hk, page, dtype, window=None, sinks=0,
                    strided=False, seed=0, change=None, scale=SCALE, max_length=None, max_new=None,
                    spread=2):
    c = build4(lengths, hk, page, device, seed=seed + 17, extra_pages=1, spread=spread,
               layout="gaps" if strided else "plain")
    if change is not None:
        change(c)
    cu, total = offsets(new, device), sum(new)
    q = tokens(total, hq, dtype, device, seed, strided)
    k, v = values(c.data)
    ref, reach_of, reach, _ = ocache.attention(host(q), k, v, c.table.tolist(),
                                               c.lengths.tolist(), cu.tolist(), scale, window,
                                               sinks)
    if max_length is None:
        max_length = max([*lengths, 0])
    cache = PagedCache4(c.data, dtype)
    out = cached_attention(q, cache, c.table, c.lengths, cu, max_new or max(new), max_length, scale,
                           window=window, sinks=sinks)
    got = host(out)
    bound = attention_bound(dtype, ref, reach_of, reach, max_length)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(ref))
    fine = ~np.isnan(ref)
    worst = (np.abs(got - ref) / bound)[fine] if fine.any() else np.zeros(1)
    assert worst.max(initial=0.0) <= 1, f"{worst.max()} of the bound"
    again = cached_attention(q, cache, c.table, c.lengths, cu, max_new or max(new), max_length,
                             scale, window=window, sinks=sinks)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    return c, q, cu, out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,new,hq,hk,page,window,sinks,strided", [
    ((1,), (1,), 12, 2, 64, None, 0, False),
    ((31,), (1,), 12, 2, 16, None, 0, True),
    ((32, 33, 64, 65, 127, 128, 129, 1), (1,) * 8, 28, 4, 16, None, 0, False),
    ((518,), (1,), 12, 2, 64, None, 0, False),
    ((1500, 3, 700), (1, 1, 1), 8, 8, 32, None, 0, True),
    ((300, 77), (1, 1), 16, 1, 48, None, 0, False),
    ((260, 41), (1, 1), 40, 2, 16, None, 0, False),
    ((90, 5, 200), (5, 5, 5), 12, 2, 32, None, 0, False),
    ((90, 7, 200, 64), (3, 0, 8, 1), 28, 4, 16, None, 0, True),
    ((150,), (150,), 6, 2, 16, None, 0, False),
    ((400, 129), (70, 33), 7, 1, 64, None, 0, False),
    ((700, 40, 1100), (1, 1, 1), 12, 2, 16, 100, 4, False),
    ((700, 40, 1100), (1, 1, 1), 12, 2, 32, 64, 0, True),
    ((500, 300), (5, 9), 12, 2, 16, 33, 70, False),
    ((333,), (40,), 4, 2, 16, 1, 0, False),
    ((333,), (40,), 4, 2, 16, 17, 2, False),
    ((0, 4, 0), (0, 1, 2), 6, 2, 16, None, 0, False),            # nothing to see
    ((3, 2), (5, 9), 6, 2, 16, None, 0, False),                  # more tokens than rows
    ((3000, 2050), (1, 6), 14, 2, 16, None, 0, False),           # cut over the keys
])
def test_attention(device, lengths, new, hq, hk, page, dtype, window, sinks, strided):
    check_attention(device, lengths, new, hq, hk, page, dtype, window, sinks, strided,
                    seed=sum(lengths))


@pytest.mark.parametrize("new", [1, 4, 20])
def test_attention_long_and_cut(device, new):
    check_attention(device, (9001, 17, 4000), (new,) * 3, 28, 4, 64, BF16, seed=new)


@pytest.mark.parametrize("scale", [0.0, -SCALE, 30.0, 1e-6])
def test_attention_scales(device, scale):
    check_attention(device, (200, 70), (3, 1), 12, 2, 16, F16, scale=scale, seed=8)


@pytest.mark.parametrize("new,hq,hk", [(1, 6, 2), (9, 6, 2)])
@pytest.mark.parametrize("dtype,rise", [(F16, 0.98), (F16, 1.0), (BF16, 7.9), (BF16, 8.1)])
def test_attention_maxima_that_rise_by_little(device, new, hq, hk, dtype, rise):
    """Every eighth tile the scores rise by a power of two next to the one that sums are kept to."""
    length = 8 * 32 * 7 - 5
    c = build4([length], hk, 16, device, seed=3)
    for j in range(0, length, 16):
        page = c.table[0, j // 16].item()
        keys = c.data[page, :, 0, :1024].view(hk, 4, 16, 16)
        keys.zero_()
        keys[:, 0, :, :j // 256] = 0x11                    # a score of one each: 0.5 + 0.5
        c.data[page, :, 0, 2048:2112] = 127
    cu = offsets([new], device)
    q = torch.ones(new, hq, DIM, dtype=dtype, device=device)
    scale = rise * np.log(2.0)
    k, v = values(c.data)
    ref, reach_of, reach, _ = ocache.attention(host(q), k, v, c.table.tolist(),
                                               c.lengths.tolist(), cu.tolist(), scale, None, 0)
    got = host(cached_attention(q, PagedCache4(c.data, dtype), c.table, c.lengths, cu, new, length,
                                scale))
    bound = attention_bound(dtype, ref, reach_of, reach, length)
    assert (np.abs(got - ref) / bound).max() <= 1


def test_attention_pages_that_are_not_held(device):
    def change(c):
        c.table[0, 2] = -1
        c.table[0, 5] = 10 ** 6
        c.table[1, :] = -1
        c.lengths[2] = 1000                              # behind the table

    check_attention(device, (200, 70, 90), (3, 2, 1), 12, 2, 16, BF16, change=change,
                    max_length=2000)


def test_attention_bounds_below_what_is_there(device):
    """max_new and max_length cut: tokens behind are zeros, rows behind are not read."""
    c = build4([300, 40], 2, 16, device, seed=3)
    cache = PagedCache4(c.data, F16)
    q = tokens(9, 6, F16, device, 1)
    cu = offsets([6, 3], device)
    # (Other bounds may lay a call out in another way, whose sums come in another order.)
    k, v = values(c.data)
    ref, reach_of, reach, _ = ocache.attention(host(q), k, v, c.table.tolist(),
                                               c.lengths.tolist(), cu.tolist(), SCALE)
    bound = attention_bound(F16, ref, reach_of, reach, 300)
    got = cached_attention(q, cache, c.table, c.lengths, cu, 4, 1000, SCALE)
    all_of = cached_attention(q, cache, c.table, c.lengths, cu, 6, 1000, SCALE)
    assert (got[4:6] == 0).all() and (np.abs(host(all_of) - ref) <= bound).all()
    seen = [0, 1, 2, 3, 6, 7, 8]
    assert (np.abs(host(got) - ref) <= bound)[seen].all()
    k[c.table[0, 16:].tolist()], v[c.table[0, 16:].tolist()] = np.nan, np.nan
    short = cached_attention(q, cache, c.table, c.lengths, cu, 6, 256, SCALE)
    assert not torch.isnan(short).any()
    # tokens outside the offsets
    cu2 = torch.tensor([1, 4, 7], dtype=torch.int32, device=device)
    got = cached_attention(q, cache, c.table, c.lengths, cu2, 6, 1000, SCALE)
    assert (got[0] == 0).all() and (got[7:] == 0).all() and not (got[1:7] == 0).all(-1).any()


@pytest.mark.parametrize("new,length", [(1, 100), (5, 100), (5, 3000), (40, 90)])
def test_attention_nan_blocks_reach_those_that_see_them(device, new, length):
    """A NaN block of values spoils its 32 columns of the tokens that see its row, one of keys
    all columns; nobody else's."""
    def change(c):
        # the last row of the sequence: only the last token sees it
        row = length - 1
        page = c.table[0, row // 16].item()
        c.data[page, 0, 0, 2112 + 2 * 16 + row % 16] = 255           # values, block 2, head 0
        if new > 2:
            row = length - 3
            page = c.table[0, row // 16].item()
            c.data[page, 1, 0, 2048 + 0 * 16 + row % 16] = 255       # keys, block 0, head 1

    check_attention(device, (length, 50), (new, 1), 12, 2, 16, BF16, change=change)


@pytest.mark.parametrize("window,sinks", [(64, 4), (64, 0)])
def test_attention_nan_blocks_before_the_window(device, window, sinks):
    def change(c):
        for row in (2, 10, 100):
            page = c.table[0, row // 16].item()
            c.data[page, :, 0, 2112 + row % 16] = 255
            c.data[page, :, 0, 2048 + 16 + row % 16] = 255

    def clean(c):
        change(c)
        page = c.table[0, 0].item()
        c.data[page, :, 0, [2112 + 2, 2048 + 16 + 2]] = 126

    check_attention(device, (300,), (4,), 12, 2, 16, F16, window, sinks, change=clean)
    if sinks:
        with pytest.raises(AssertionError):              # row 2 is seen: NaN, as the oracle has it
            c, _, _, out = check_attention(device, (300,), (4,), 12, 2, 16, F16, window, sinks,
                                           change=change)
            assert not torch.isnan(out).any()


def test_attention_wide_scales_and_the_ends_of_the_range(device):
    def change(c):
        c.data[..., 2048:2112][c.data[..., 2048:2112] != 255] = 127 - 13
        c.data[..., 2112:][c.data[..., 2112:] != 255] = 127 + 13

    check_attention(device, (90, 40), (3, 1), 12, 2, 16, F16, change=change)

    def far(c):
        c.data[..., 2048:2112][c.data[..., 2048:2112] != 255] = 127 - 125
        c.data[..., 2112:][c.data[..., 2112:] != 255] = 127 + 100

    check_attention(device, (90, 40), (3, 1), 12, 2, 16, BF16, change=far)


def test_without_sequences_or_tokens(device):
    cache = PagedCache4.empty(4, 2, 16, F16, device)
    table = torch.zeros((0, 3), dtype=torch.int32, device=device)
    none = torch.zeros(0, dtype=torch.int32, device=device)
    cu = torch.zeros(1, dtype=torch.int32, device=device)
    q = tokens(3, 4, F16, device, 1)
    assert (cached_attention(q, cache, table, none, cu, 1, 10, SCALE) == 0).all()
    assert cached_attention(q[:0], cache, table, none, cu, 0, 10, SCALE).shape == (0, 4, DIM)
    k = tokens(3, 2, F16, device, 2)
    cos = torch.ones((3, DIM), device=device)
    turned = append_kv(cache, k, k, table, none, cu, q=q, cos=cos, sin=cos * 0)
    assert torch.equal(turned, q)
    held = read_kv(cache, table, none, cu, 3)
    assert (held[0] == 0).all() and held[0].shape == (3, 2, DIM)
    assert read_kv(cache, table, none, cu, 0)[0].shape == (0, 2, DIM)


# ------------------------------------------------------- as they are used

def test_append_and_attention_replayed_and_on_another_stream(device):
    """A captured step, replayed as the sequences grow, gives what eager calls give."""
    steps, rows, hk, hq, page = 4, 3, 2, 12, 16
    lens = [15, 200, 31]
    table = torch.arange(rows * 20, dtype=torch.int32, device=device).view(rows, 20)
    data = torch.from_numpy(random_bytes((rows * 20, hk, 1, 2176), 9)).to(device)
    other = data.clone()
    lengths = torch.tensor(lens, dtype=torch.int32, device=device)
    cu = offsets([1] * rows, device)
    q, k, v = (tokens(rows, h, BF16, device, i) for i, h in enumerate((hq, hk, hk)))
    cos = torch.ones((rows, DIM), dtype=BF16, device=device)
    sin = cos * 0.5

    def step(cache):
        turned = append_kv(cache, k, v, table, lengths, cu, q=q, cos=cos, sin=sin)
        return cached_attention(turned, cache, table, lengths, cu, 1, 300, SCALE)

    graphed, eager = PagedCache4(data, BF16), PagedCache4(other, BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graphed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed)
    other.copy_(data)                                    # with the row that the first step wrote
    for i in range(steps):
        lengths += 1
        q.copy_(tokens(rows, hq, BF16, device, 20 + i))
        k.copy_(tokens(rows, hk, BF16, device, 40 + i))
        v.copy_(tokens(rows, hk, BF16, device, 60 + i))
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
