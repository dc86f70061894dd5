"""Cached attention where the scaled scores pass 2^24, at which fp32 counts in whole powers of two.

The inputs make every product and sum exact in fp32 (whole multiples of 32 below 2^29), so what the
kernel has beside 64 bits is: the scale's and the exponent's rounding (3 half steps of fp32 of an
exponent of at most REACH), the exponential's (2), the sums over the rows, each twice (numerator
and sum), the rounding of a probability to 16 bits twice and the output's.
"""

import numpy as np
import pytest
import torch

from oracle import cache as ocache
from soupsuck_amd.kernels.paged import PagedCache, cached_attention
from tests.cache_util import HALF_STEP, build, host, offsets

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SCALE, STEPS = 0.05, 20
REACH = 32 * SCALE * STEPS          # exponents within this of the greatest


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", [1024.0, 1500.0, 2000.0])
@pytest.mark.parametrize("new,length", [(1, 1), (1, 1300), (4, 1300), (40, 1300)])
def test_equal_keys_give_their_value(device, size, new, length, dtype):
    """Rows with one value in common: whatever the weights' shares, it is the result."""
    c = build((length,), 2, 16, dtype, device, seed=1)
    c.k.fill_(size)
    c.v.copy_(c.v[c.table[0, 0].item(), :, :1][None])
    cu = offsets((min(new, length),), device)
    q = torch.full((min(new, length), 12, 128), size, dtype=dtype, device=device)
    out = cached_attention(q, PagedCache(c.k, c.v), c.table, c.lengths, cu, new, length,
                           128 ** -0.5)
    want = c.v[c.table[0, 0].item(), :, 0].repeat_interleave(6, 0)[None].double()
    # equal weights: their sum's rounding (length half steps of fp32, twice) and the output's
    error = HALF_STEP[dtype] + 2 * 2.0 ** -24 * length
    assert ((out.double() - want).abs() <= error * want.abs()).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("lengths,new,hq", [
    ((40, 9), 1, 14), ((3000, 40, 700), 1, 14), ((3000, 700), 2, 14), ((1400, 300), 8, 12),
    ((1500, 90), 40, 12)])
def test_weights_of_close_keys(device, lengths, new, hq, sign, dtype):
    """q . k = 127 * 2000^2 + 32 a, a = 0 .. 20: close keys under a large common part."""
    print(f"case close keys {lengths} {new} {hq} {sign} {dtype}", flush=True)
    c = build(lengths, 2, 16, dtype, device, seed=2)
    rows, gen = len(lengths), torch.Generator().manual_seed(3)
    steps = torch.randint(0, STEPS + 1, c.k.shape[:3], generator=gen).to(dtype).to(device)
    c.k.fill_(2000.0)
    c.k[..., 127] = steps
    q = torch.full((rows * new, hq, 128), sign * 2000.0, dtype=dtype, device=device)
    q[..., 127] = sign * 32.0
    cu = offsets((new,) * rows, device)
    sums = torch.zeros((rows, 2, c.table.shape[1] * 16), device=device)
    args = (q, PagedCache(c.k, c.v), c.table, c.lengths, cu, new, max(lengths), sign * SCALE)
    out = cached_attention(*args, weights_out=sums)
    assert torch.equal(out, cached_attention(*args))
    ref, spread, _, w = ocache.attention(host(q), host(c.k), host(c.v), c.table.tolist(),
                                         lengths, cu.tolist(), sign * SCALE)
    step = HALF_STEP[dtype]
    error = 2 * 2.0 ** -24 * (3 * REACH + 2 + max(lengths))
    bound = step * np.abs(ref) + spread * (2 * step + error) + 1e-7
    assert (np.abs(host(out) - ref) <= bound).all()
    error += 2.0 ** -24 * new * hq // 2
    assert (np.abs(host(sums) - w) <= w * error + 1e-12).all()
