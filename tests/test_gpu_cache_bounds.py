"""Cached attention at the edges of its bounds: lengths cut by max_length, windows that leave
nothing of a sequence, workspaces with a guard behind them.

Oracle: oracle/cache.py in 64 bits, given only the table's pages that the bound leaves (a cut
sequence's tokens keep their places).  Tolerances: tests/cache_util.attention_bound and, for
accumulated weights, the scores' error on each weight and one rounding of each sum.
"""

import numpy as np
import pytest
import torch

from oracle import cache as ocache
from soupsuck_amd import _lib
from soupsuck_amd.kernels.paged import PagedCache, cached_attention
from tests.cache_util import attention_bound, build, host, offsets
from tests.test_gpu_cache import SCALE, _tokens

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
GUARD = 4096


def _attention(cache, q, table, lengths, cu, max_new, max_length, window, sinks, weights):
    """(out, weights_out) of the C entry point with a guard behind the workspace, which must
    come back as it was."""
    rows, tokens, heads = table.shape[0], q.shape[0], q.shape[1]
    out = torch.full_like(q, float("nan"))
    need = _lib.load().ss_cached_attention_workspace_size(
        rows, tokens, heads, cache.k.shape[1], max_new, max_length, 1)
    scratch = torch.full((need + GUARD,), 0xA5, dtype=torch.uint8, device=q.device)
    sums = torch.full_like(weights, float("nan"))
    _lib.call("ss_cached_attention", cache._pointer, q.data_ptr(), q.stride(0), q.stride(1), heads,
              table.data_ptr(), table.stride(0), table.shape[1], lengths.data_ptr(), cu.data_ptr(),
              rows, tokens, max_new, max_length, SCALE, window, sinks, weights.data_ptr(),
              sums.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), scratch.data_ptr(),
              need, _lib.stream(q.device))
    assert (scratch[need:] == 0xA5).all()
    return out, sums


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,hq", [(1, 14), (2, 12), (3, 12)])      # scores kept; keys again
@pytest.mark.parametrize("bound", [64, 1024, 2048])                  # one workgroup a unit; cut
@pytest.mark.parametrize("sinks", [0, 3])
def test_windows_past_the_bound(device, bound, new, hq, sinks, dtype):
    """Lengths so far past max_length that a window leaves nothing, beside ordinary sequences:
    before, between and behind them."""
    print(f"case window past the bound {bound} {new} {hq} {sinks} {dtype}", flush=True)
    window = 100
    lengths = (bound + 500, bound - 4, bound + window + new, 40, bound + 900)
    c = build(lengths, 2, 16, dtype, device, seed=bound + new)
    cu = offsets((new,) * len(lengths), device)
    q = _tokens(new * len(lengths), hq, dtype, device, 3)
    base = torch.rand((len(lengths), 2, c.table.shape[1] * 16),
                      generator=torch.Generator().manual_seed(5)).to(device)
    out, sums = _attention(PagedCache(c.k, c.v), q, c.table, c.lengths, cu, new, bound, window,
                           sinks, base)
    ref, spread, reach, w = ocache.attention(
        host(q), host(c.k), host(c.v), c.table[:, :bound // 16].tolist(), lengths, cu.tolist(),
        SCALE, window, sinks)
    assert (np.abs(host(out) - ref) <= attention_bound(dtype, ref, spread, reach, bound)).all()
    if not sinks:
        for row in (0, 2, 4):
            assert (out[row * new:(row + 1) * new] == 0).all()
    want = host(base)
    want[:, :, :bound] += w
    error = np.zeros_like(want)
    error[:, :, :bound] = w * 2 * 2.0 ** -24 * (128 * reach + 4 * (1 + reach) + bound)
    assert (np.abs(host(sums) - want) <= error + 2 * 2.0 ** -24 * want + 1e-12).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bound", [4000, 131072, 3 * 10 ** 6, 2 ** 31 - 1])
@pytest.mark.parametrize("new,hq", [(1, 12), (2, 14), (4, 12), (20, 6)])
def test_the_bound_has_no_part_in_the_result(device, bound, new, hq, dtype):
    """Large bounds choose loads past the caches and keep no scores for the weights; what is
    summed, and so the tolerance, is the sequences' own rows."""
    print(f"case bound {bound} {new} {hq} {dtype}", flush=True)
    lengths = (700, new, 90, 1200)
    c = build(lengths, 2, 16, dtype, device, seed=17)
    cu = offsets((new,) * 4, device)
    q = _tokens(new * 4, hq, dtype, device, 0)
    base = torch.rand((4, 2, c.table.shape[1] * 16),
                      generator=torch.Generator().manual_seed(5)).to(device)
    sums = torch.full_like(base, float("nan"))
    out = cached_attention(q, PagedCache(c.k, c.v), c.table, c.lengths, cu, new, bound, SCALE,
                           weights=base, weights_out=sums)
    ref, spread, reach, w = ocache.attention(host(q), host(c.k), host(c.v), c.table.tolist(),
                                             lengths, cu.tolist(), SCALE)
    rows = max(lengths)
    assert (np.abs(host(out) - ref) <= attention_bound(dtype, ref, spread, reach, rows)).all()
    want = host(base) + w
    error = w * 2 * 2.0 ** -24 * (128 * reach + 4 * (1 + reach) + rows)
    assert (np.abs(host(sums) - want) <= error + 2 * 2.0 ** -24 * want + 1e-12).all()
