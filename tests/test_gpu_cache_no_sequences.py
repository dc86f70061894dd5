"""Calls with tokens and no sequences: queries are rotated and see nothing, the cache stays."""

import pytest
import torch

from oracle import cache as ocache
from soupsuck_amd import _lib
from soupsuck_amd.kernels.paged import PagedCache, append_kv, cached_attention, evict_kv
from tests.cache_util import DIM, HALF_STEP, build, host
from tests.test_gpu_cache import _tokens

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(params=[F16, BF16])
def call(request, device):
    c = build((40,), 2, 16, request.param, device, seed=1)
    return (request.param, PagedCache(c.k, c.v), c.table[:0], c.lengths[:0],
            torch.zeros(1, dtype=torch.int32, device=device))


@pytest.mark.parametrize("count", [1, 37])
def test_append(device, call, count):
    dtype, cache, table, lengths, cu = call
    before = cache.k.clone(), cache.v.clone()
    k, q = _tokens(count, 2, dtype, device, 1), _tokens(count, 6, dtype, device, 2)
    cos, sin = (_tokens(count, 1, dtype, device, s)[:, 0] for s in (3, 4))
    got = append_kv(cache, k, k, table, lengths, cu, q=q, cos=cos, sin=sin)
    want = ocache.rotate(host(q), host(cos)[:, None], host(sin)[:, None])
    size = abs(host(q)).max() * 2 * abs(host(cos)).max() + abs(host(sin)).max() * abs(host(q)).max()
    # one rounding, and 3 half steps of fp32 of the two products
    assert (abs(host(got) - want) <= HALF_STEP[dtype] * abs(want) * 1.001
            + 3 * 2.0 ** -24 * size + 2.0 ** -25).all()
    assert append_kv(cache, k, k, table, lengths, cu) is None
    for now, then in zip((cache.k, cache.v), before):
        assert torch.equal(now.view(torch.int16), then.view(torch.int16))


@pytest.mark.parametrize("count", [0, 1, 37])
def test_attention(device, call, count):
    dtype, cache, table, lengths, cu = call
    q = _tokens(count, 6, dtype, device, 2, "row")
    weights = torch.zeros((0, 2, table.shape[1] * 16), device=device)
    for extra in ({}, dict(weights_out=weights), dict(window=5, sinks=2)):
        got = cached_attention(q, cache, table, lengths, cu, 3, 40, 0.1, **extra)
        assert got.shape == (count, 6, DIM) and (got == 0).all()


@pytest.mark.parametrize("count", [1, 37])
def test_the_c_entry_point(device, call, count):
    """Outputs of any strides are written, what lies between them is not."""
    dtype, cache, _, _, _ = call
    q = _tokens(count, 6, dtype, device, 2)
    wide = torch.full((count, 7, DIM + 8), 3.0, dtype=dtype, device=device)
    out = wide[:, :6, :DIM]
    _lib.call("ss_cached_attention", cache._pointer, q.data_ptr(), q.stride(0), q.stride(1), 6,
              None, 3, 3, None, None, 0, count, 1, 40, 0.1, 0, 0, None, None, out.data_ptr(),
              out.stride(0), out.stride(1), None, 0, _lib.stream(device))
    assert (out == 0).all() and (wide[:, 6] == 3).all() and (wide[:, :, DIM:] == 3).all()


def test_evict(device, call):
    _, cache, table, lengths, _ = call
    weights = torch.zeros((0, 2, table.shape[1] * 16), device=device)
    got = evict_kv(cache, table, lengths, weights, table, 16, 40)
    assert got[0].shape == (0,) and got[1].shape == weights.shape
