"""Attention over a 4-bit cache where masks and bounds meet blocks that are not numbers.

Rows behind max_length are NaN on the device, and so are rows before a window; sinks may be NaN
themselves, all of a row (a block of its keys) or 32 columns (a block of its values).  What is NaN in
the result has to be what the formula makes NaN.

Oracle: the formula in 64 bits, with a bound on the rows; tests/cache_util.attention_bound.
"""

import numpy as np
import pytest
import torch

from soupsuck_amd.kernels.paged import PagedCache4, cached_attention
from tests.cache4_util import build4, tokens, values
from tests.cache_util import DIM, attention_bound, host, offsets
from tests.test_gpu_cache4 import check_attention

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SCALE = DIM ** -0.5


def _reference(q, k, v, table, lengths, cu, window, sinks, bound):
    """(o, sums of |p v|, greatest sum of |q k| scale) with rows from `bound` on left out."""
    size, heads = k.shape[2], k.shape[1]
    group = q.shape[1] // heads
    out, spread, reach = np.zeros_like(q), np.zeros_like(q), 0.0
    for b, length in enumerate(lengths):
        there = np.arange(min(length, bound, len(table[b]) * size))
        if not len(there):
            continue
        page = np.array(table[b])[there // size]
        keys, vals = (x[page, :, there % size] for x in (k, v))       # [rows, heads, 128]
        for t in range(cu[b], cu[b + 1]):
            at = length - cu[b + 1] + t
            seen = (there <= at) & ((there > at - window) | (there < sinks) if window else True)
            if not seen.any():
                continue
            for h in range(q.shape[1]):
                ks, vs = keys[seen, h // group], vals[seen, h // group]
                s = ks @ q[t, h] * SCALE
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h], spread[t, h] = p @ vs, p @ np.abs(vs)
                reach = max(reach, float(np.nanmax(np.abs(ks) @ np.abs(q[t, h])) * SCALE))
    return out, spread, reach


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,hq", [(1, 6), (3, 16), (20, 4)])
@pytest.mark.parametrize("bound", [1, 64, 250, 256, 1009, 4000, 5001])    # whole units; split
@pytest.mark.parametrize("window,sinks", [(None, 0), (1500, 40)])
def test_rows_behind_max_length_are_not_read(device, bound, window, sinks, new, hq, dtype):
    print(f"case rows behind max_length {bound} {new} {window} {dtype}", flush=True)
    lengths = (bound + 300, max(bound - 4, 0), 40, bound + 1, bound + 900)
    c = build4(lengths, 2, 16, device, seed=bound + new)
    for b in range(len(lengths)):
        for j in range(bound, min(bound + 64, lengths[b])):           # rows of the next tiles
            page = c.table[b, j // 16].item()
            c.data[page, :, 0, 2048 + j % 16::16] = 255
    cu = offsets([new] * len(lengths), device)
    q = tokens(new * len(lengths), hq, dtype, device, 3)
    got = host(cached_attention(q, PagedCache4(c.data, dtype), c.table, c.lengths, cu, new, bound,
                                SCALE, window=window, sinks=sinks))
    ref, spread, reach = _reference(host(q), *values(c.data), c.table.tolist(), lengths,
                                    cu.tolist(), window, sinks, bound)
    assert np.isfinite(ref).all() and np.isfinite(got).all()
    assert (np.abs(got - ref) <= attention_bound(dtype, ref, spread, reach, bound)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,hq", [(1, 12), (4, 12), (40, 4)])
@pytest.mark.parametrize("length", [300, 5000])                       # one workgroup a unit; split
@pytest.mark.parametrize("sinks", [3, 40, 70])                        # inside a tile; a tile and more
@pytest.mark.parametrize("which", ["keys", "values"])
def test_nan_blocks_of_sinks(device, which, sinks, length, new, hq, dtype):
    """Row 2 is a sink and NaN: in a block of keys for every column, in one of values for 32."""
    print(f"case nan blocks of sinks {which} {sinks} {length} {new} {dtype}", flush=True)

    def change(c):
        page = c.table[0, 0].item()
        if which == "keys":
            c.data[page, 0, 0, 2048 + 16 + 2] = 255
        else:
            c.data[page, 0, 0, 2112 + 2 * 16 + 2] = 255
        for row in (75, 100):                                         # neither sinks nor in a window
            page = c.table[0, row // 16].item()
            c.data[page, :, 0, 2048 + row % 16::16] = 255

    _, _, _, out = check_attention(device, (length, 50), (new, 1), hq, 2, 16, dtype, 64, sinks,
                                   seed=length, change=change)
    nan = torch.isnan(out).cpu()                                      # as the formula has it, spelled out
    want = torch.zeros_like(nan)
    columns = slice(0, 128) if which == "keys" else slice(64, 96)
    want[:new, :hq // 2, columns] = True
    assert torch.equal(nan, want)
