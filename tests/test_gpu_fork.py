"""GPU parity of fork_kv: tables, lengths and copied rows, exactly (oracle/cache4.py)."""

import numpy as np
import pytest
import torch

from oracle import cache4
from soupsuck_amd.kernels.paged import PagedCache, PagedCache4, fork_kv
from tests.cache4_util import random_bytes

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _caches(four, layers, pages, heads, page, dtype, device, strided=False):
    out = []
    for i in range(layers):
        if four:
            data = torch.from_numpy(random_bytes((pages, heads, page // 16, 2176), i)).to(device)
            if strided:
                wide = torch.zeros((pages, heads + 1, page // 16, 2192), dtype=torch.uint8,
                                   device=device)
                wide[:, :heads, :, :2176] = data
                data = wide[:, :heads, :, :2176]
            out.append(PagedCache4(data, dtype))
            continue
        gen = torch.Generator().manual_seed(i)
        k, v = (torch.randn((pages, page, heads, 128), generator=gen).to(dtype).to(device)
                for _ in range(2))
        out.append(PagedCache(*((k.transpose(1, 2), v.transpose(1, 2)) if strided else
                                (t.transpose(1, 2).contiguous() for t in (k, v)))))
    return out


def _tensors(cache):
    return (cache.data,) if isinstance(cache, PagedCache4) else (cache.k, cache.v)


def _check(device, four, table, lengths, parents, spare, page, pages, heads=2, layers=2,
           dtype=F16, strided=False):
    caches = _caches(four, layers, pages, heads, page, dtype, device, strided)
    want, want_lengths, copies = cache4.fork(table, lengths, parents, spare, page, pages)
    expected = []
    for cache in caches:
        for t in _tensors(cache):
            t = t.clone()
            old = t.clone()
            for a, b, n in copies:
                if four:
                    t[b, :, :-(-n // 16)] = old[a, :, :-(-n // 16)]
                else:
                    t[b, :, :n] = old[a, :, :n]
            expected.append(t)
    got, got_lengths = fork_kv(caches, _int32(table, device), _int32(lengths, device),
                               _int32(parents, device), _int32(spare, device))
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    np.testing.assert_array_equal(got_lengths.cpu().numpy(), want_lengths)
    for t, ref in zip((t for c in caches for t in _tensors(c)), expected):
        assert torch.equal(t, ref)


@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("table,lengths,parents,spare,page,pages", [
    ([[0, 1], [2, 3]], [20, 27], [1, 0], [4, 5], 16, 6),
    ([[0, 1], [2, 3]], [20, 27], [1, 1], [4, 5], 16, 6),             # both continue one
    ([[0, 1], [2, 3]], [16, 32], [0, 1], [4, 5], 16, 6),             # at a page's end, full
    ([[0, 1], [2, 3]], [0, 1], [0, 1], [4, 5], 16, 6),               # empty, one row
    ([[0, 1, -1]], [70], [0] * 5, [2, 3, 4, 5, 6], 64, 7),           # one into five
    ([[0, 1], [2, 3], [4, 5]], [33, 31, 90], [2], [6], 48, 7),       # three into one
    ([[0, 1], [2, 3]], [20, 27], [-1, 2], [4, 5], 16, 6),            # parents that are none
    ([[0, -1], [2, 99]], [20, 27], [0, 1], [4, 5], 16, 6),           # open pages not held
    ([[0, 1], [2, 3]], [20, 27], [0, 1], [-1, 77], 16, 6),           # spares that are none
    ([[0, 1], [2, 3]], [-4, 999], [0, 1], [4, 5], 16, 6),            # lengths cut
    ([[0, 1], [2, 3]], [100, 127], [1, 0], [4, 5], 128, 6),
])
def test_fork(device, four, table, lengths, parents, spare, page, pages):
    _check(device, four, table, lengths, parents, spare, page, pages)


@pytest.mark.parametrize("four", [True, False])
def test_fork_many_layers_heads_and_strides(device, four):
    _check(device, four, [[0, 1], [2, 3]], [20, 27], [1, 0], [4, 5], 16, 6, layers=130)
    _check(device, four, [[0, 1], [2, 3]], [50, 40], [1, 0], [4, 5], 32, 6, heads=7, dtype=BF16,
           strided=True)


def test_fork_random(device):
    rng = np.random.default_rng(5)
    rows, width, page = 24, 9, 32
    pages = rows * width + rows
    order = rng.permutation(pages)
    table = order[:rows * width].reshape(rows, width).tolist()
    _check(device, True, table, rng.integers(0, page * width + 1, rows).tolist(),
           rng.integers(0, rows, rows).tolist(), order[rows * width:].tolist(), page, pages,
           heads=3, layers=3)


def test_fork_without_rows_and_with_a_single_cache(device):
    cache = _caches(True, 1, 4, 2, 16, F16, device)[0]
    none = torch.zeros(0, dtype=torch.int32, device=device)
    table, lengths = fork_kv(cache, _int32([[0, 1]], device), _int32([5], device), none, none)
    assert table.shape == (0, 2) and lengths.shape == (0,)
    empty = torch.zeros((0, 2), dtype=torch.int32, device=device)
    table, lengths = fork_kv(cache, empty, none, _int32([0], device), _int32([3], device))
    assert table.tolist() == [[3, -1]] and lengths.tolist() == [0]


@pytest.mark.parametrize("four", [True, False])
def test_fork_replayed(device, four):
    """A captured fork sees the tables, lengths and parents of the moment."""
    caches = _caches(four, 2, 12, 2, 16, F16, device)
    table, lengths = _int32([[0, 1, 2], [3, 4, 5]], device), _int32([20, 40], device)
    parents, spare = _int32([1, 0], device), _int32([6, 7], device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fork_kv(caches, table, lengths, parents, spare)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, out_lengths = fork_kv(caches, table, lengths, parents, spare)
    for i, (n, p, s) in enumerate((([20, 40], [1, 0], [6, 7]), ([31, 5], [1, 1], [8, 9]),
                                   ([48, 16], [0, 0], [10, 11]))):
        lengths.copy_(_int32(n, device))
        parents.copy_(_int32(p, device))
        spare.copy_(_int32(s, device))
        before = [t.clone() for c in caches for t in _tensors(c)]
        graph.replay()
        torch.cuda.synchronize()
        want, want_lengths, copies = cache4.fork(table.tolist(), n, p, s, 16, 12)
        np.testing.assert_array_equal(out.cpu().numpy(), want)
        np.testing.assert_array_equal(out_lengths.cpu().numpy(), want_lengths)
        for t, ref in zip((t for c in caches for t in _tensors(c)), before):
            for a, b, rows in copies:
                rows = slice(None) if four else slice(0, rows)
                ref[b, :, rows] = ref[a, :, rows]
            assert torch.equal(t, ref)
