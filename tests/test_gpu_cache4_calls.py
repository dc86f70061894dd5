"""The 4-bit cache's, fork's and selection's calls made in other ways: the native bodies against the
Python ones, units over many ranges, two calls at once, offsets past 32 bits."""

import contextlib

import numpy as np
import pytest
import torch

from oracle import cache as ocache
from soupsuck_amd import _lib
from soupsuck_amd.kernels.beams import select_beams
from soupsuck_amd.kernels.paged import (PagedCache, PagedCache4, append_kv, cached_attention,
                                        fork_kv, read_kv)
from tests.cache4_util import build4, random_bytes, tokens, values
from tests.cache_util import DIM, attention_bound, build, host, offsets
from tests.test_gpu_cache4 import check_attention

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SCALE = DIM ** -0.5


@contextlib.contextmanager
def python_bodies():
    _lib.hooks["none"] = None
    try:
        yield
    finally:
        del _lib.hooks["none"]


def _same(a, b):
    a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride()
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("angles", [None, torch.float32, "cache"])
def test_append_and_read(device, dtype, angles):
    c = build4([40, 9], 2, 16, device, seed=1)
    other = c.data.clone()
    cu = offsets([5, 9], device)
    k, v = (tokens(14, 2, dtype, device, s) for s in (2, 3))
    q = cos = sin = None
    if angles is not None:
        kind = dtype if angles == "cache" else angles
        q = tokens(14, 6, dtype, device, 4)
        cos, sin = (tokens(14, 1, kind, device, s)[:, 0] for s in (5, 6))
    caches = PagedCache4(c.data, dtype), PagedCache4(other, dtype)
    got = append_kv(caches[0], k, v, c.table, c.lengths, cu, q=q, cos=cos, sin=sin)
    with python_bodies():
        want = append_kv(caches[1], k, v, c.table, c.lengths, cu, q=q, cos=cos, sin=sin)
    assert got is None and want is None if q is None else torch.equal(got, want)
    assert torch.equal(c.data, other)
    for which in (caches[0], list(caches), caches):
        read = read_kv(which, c.table, c.lengths, cu, 14)
        with python_bodies():
            _same(read, read_kv(which, c.table, c.lengths, cu, 14))


def test_attention_fork_and_select(device):
    c = build4([300, 90], 2, 16, device, seed=2)
    cache = PagedCache4(c.data, F16)
    q, cu = tokens(6, 12, F16, device, 1), offsets([4, 2], device)

    def attend():
        return cached_attention(q, cache, c.table, c.lengths, cu, 4, 300, SCALE, window=100,
                                sinks=4)

    wide = build([20, 9], 2, 16, F16, device, seed=1, poison=0.0)
    layers = [PagedCache(wide.k, wide.v), PagedCache(wide.v.clone(), wide.k.clone())]
    parents, spare = (torch.tensor(x, dtype=torch.int32, device=device)
                      for x in ([1, 0, 1], wide.free[:3]))

    def fork():
        return fork_kv(layers, wide.table, wide.lengths, parents, spare)

    logits = tokens(3, 5, BF16, device, 3).contiguous()
    scores = torch.rand((3, 5), device=device)

    def select():
        return select_beams(logits, scores, 7)

    for call in (attend, fork, select):
        got = call()
        with python_bodies():
            _same(got, call())


def test_subclasses_are_caches_too(device):
    class Mine(PagedCache4):
        pass

    c = build4([40], 2, 16, device, seed=1)
    cu = offsets([40], device)
    got = read_kv([Mine(c.data, F16)], c.table, c.lengths, cu, 40)
    want = read_kv([PagedCache4(c.data, F16)], c.table, c.lengths, cu, 40)
    _same(got, want)


@pytest.mark.parametrize("rows,new,hq,hk", [(70, 1, 4, 2), (130, 2, 8, 8), (9, 3, 28, 4),
                                            (5, 1, 6, 1), (33, 1, 8, 8)])
def test_attention_over_many_ranges(device, rows, new, hq, hk):
    """More lines than are looked at together; units in equal parts and not; short ones between."""
    rng = np.random.default_rng(rows)
    lengths = rng.integers(new, 1400, rows).tolist()
    lengths[::7] = [0] * len(lengths[::7])
    lengths[1] = 2500
    check_attention(device, lengths, (new,) * rows, hq, hk, 16, BF16, seed=rows)


@pytest.mark.parametrize("rows,new,hq,hk,window", [
    (70, 3, 64, 8, None), (70, 3, 64, 8, 40),          # blocks of 32 rows on two waves
    (36, 7, 128, 16, None), (36, 7, 128, 16, 40),      # of 64 rows on two waves
    (68, 1, 8, 8, None), (150, 1, 8, 8, 40),           # of 16 rows on two waves
    (40, 3, 64, 8, None), (40, 3, 64, 8, 40),          # each on four
    (40, 7, 64, 8, None), (40, 7, 64, 8, 40),
    (40, 1, 8, 8, None), (40, 1, 64, 8, 40),
])
def test_attention_of_many_short_units(device, rows, new, hq, hk, window):
    rng = np.random.default_rng(rows)
    lengths = rng.integers(1, 200, rows).tolist()
    lengths[::9] = [0] * len(lengths[::9])
    lengths[2] = 270

    def change(c):
        # NaN blocks of values in a row that the last token alone sees, and in one that all see
        for b, row in ((2, 269), (4, 0)):
            page = c.table[b, row // 16].item()
            if page >= 0:
                c.data[page, 0, 0, 2112 + 16 + row % 16] = 255

    check_attention(device, lengths, (new,) * rows, hq, hk, 16, F16, window, 2, seed=rows,
                    change=change)


@pytest.mark.parametrize("window", [None, 500])
def test_attention_of_equal_parts(device, window):
    """Eight sequences whose units are cut into as many parts each."""
    check_attention(device, (3000, 2900, 3100, 2800) * 2, (2,) * 8, 16, 8, 32, F16, window, 4,
                    seed=3)


@pytest.mark.parametrize("new,hq,hk", [(5, 8, 2), (9, 8, 2), (11, 14, 2)])
def test_attention_of_one_long_among_short_ones(device, new, hq, hk):
    """Its units have more parts than are joined row by row; blocks of 20, 36, 64 and 13 rows."""
    lengths = [70 + 5 * i for i in range(24)]
    lengths[5], lengths[6], lengths[20] = 20000, 0, 900
    news = [new] * 24
    news[7], news[8] = 0, 1
    check_attention(device, lengths, news, hq, hk, 16, BF16, seed=new)


@pytest.mark.parametrize("new", [5, 12, 40, 90])
def test_attention_bounds_far_above_the_lengths(device, new):
    """Bounds that ask for the split where the sequences are short, or have nothing."""
    check_attention(device, (100, 0, 33), (new, 0, 3), 14, 2, 16, BF16, seed=4, max_length=100000,
                    max_new=new + 7)


def test_two_streams_at_once(device):
    """Calls on two streams have workspaces of their own."""
    c = build4([5000, 3000], 2, 16, device, seed=6)
    cache = PagedCache4(c.data, F16)
    cu = offsets([1, 1], device)
    qs = [tokens(2, 12, F16, device, i) for i in range(4)]
    logits = torch.randn((2, 4, 30000), device=device)
    scores = torch.zeros((2, 4), device=device)

    def both(q):
        return (cached_attention(q, cache, c.table, c.lengths, cu, 1, 5000, SCALE),
                *select_beams(logits + q.float().mean(), scores, 8))

    want = [both(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(both(q))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        _same(a, b)


def test_offsets_past_32_bits(device):
    """A cache of more than 4 GiB: rows on its first and its last pages."""
    pages, heads, page = 31000, 8, 128
    data = torch.empty((pages, heads, page // 16, 2176), dtype=torch.uint8, device=device)
    assert data.numel() > 2 ** 32
    cache = PagedCache4(data, BF16)
    table = torch.tensor([[pages - 1, 0], [pages - 2, 1]], dtype=torch.int32, device=device)
    lengths = torch.tensor([200, 130], dtype=torch.int32, device=device)
    cu = offsets([200, 130], device)
    k, v = (tokens(330, heads, BF16, device, s) for s in (1, 2))
    append_kv(cache, k, v, table, lengths, cu)
    held_k, held_v = read_kv(cache, table, lengths, cu, 330)
    few = PagedCache4.empty(4, heads, page, BF16, device)
    near = torch.tensor([[3, 0], [2, 1]], dtype=torch.int32, device=device)
    append_kv(few, k, v, near, lengths, cu)
    _same((held_k, held_v), read_kv(few, near, lengths, cu, 330))
    q, one = tokens(2, 16, BF16, device, 3), offsets([1, 1], device)
    _same(cached_attention(q, cache, table, lengths, one, 1, 200, SCALE),
          cached_attention(q, few, near, lengths, one, 1, 200, SCALE))
    parents, spare = (torch.tensor(x, dtype=torch.int32, device=device)
                      for x in ([1, 0], [pages - 3, 2]))
    new, sizes = fork_kv(cache, table, lengths, parents, spare)
    assert new.tolist() == [[pages - 2, pages - 3], [pages - 1, 2]] and sizes.tolist() == [130, 200]
    turned = read_kv(cache, new, sizes, offsets([130, 200], device), 330)
    assert torch.equal(turned[0][:130], held_k[200:]) and torch.equal(turned[0][130:], held_k[:200])


@pytest.mark.parametrize("sinks", [0, 3])
def test_attention_rows_and_columns_of_one_query(device, sinks):
    """Each weight on its own row: keys that single one value out (which column goes where)."""
    c = build4([64], 1, 16, device, seed=7)
    cache = PagedCache4(c.data, F16)
    k = torch.zeros((64, 1, DIM), dtype=F16, device=device)
    k[torch.arange(64), 0, 2 * torch.arange(64)] = 6.0
    v = (torch.arange(64 * DIM, device=device).view(64, 1, DIM) % 13 - 6).to(F16)
    cu = offsets([64], device)
    append_kv(cache, k, v, c.table, c.lengths, cu)
    keys, vals = values(c.data)
    for row in (0, 1, 15, 16, 31, 32, 63):
        q = torch.zeros((1, 2, DIM), dtype=F16, device=device)
        q[0, :, 2 * row] = 100.0
        out = cached_attention(q, cache, c.table, c.lengths, offsets([1], device), 1, 64, 1.0,
                               sinks=sinks)
        page, inside = c.table[0, row // 16].item(), row % 16
        assert np.array_equal(host(out)[0, 0], vals[page, 0, inside])
        ref, spread, reach, _ = ocache.attention(host(q), keys, vals, c.table.tolist(), [64],
                                                 [0, 1], 1.0)
        assert (np.abs(host(out) - ref) <= attention_bound(F16, ref, spread, reach, 64)).all()


def test_random_bytes_hold_every_code(device):
    """All 256 bytes and both types: what is read back is what the bytes say."""
    data = torch.from_numpy(random_bytes((3, 2, 2, 2176), 1, spread=20)).to(device)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=device)
    lengths = torch.tensor([96], dtype=torch.int32, device=device)
    keys, vals = values(data)
    for dtype in (F16, BF16):
        some = data.clone()
        if dtype == F16:
            some[..., 2048:] = some[..., 2048:].clamp(127 - 13, 127 + 13)
        k, v = values(some)
        got = read_kv(PagedCache4(some, dtype), table, lengths, offsets([96], device), 96)
        order = [2, 0, 1]
        for a, b in zip(got, (k, v)):
            want = np.concatenate([b[p].transpose(1, 0, 2) for p in order])
            np.testing.assert_array_equal(host(a), want)
    assert np.isfinite(keys).all() and np.isfinite(vals).all()
