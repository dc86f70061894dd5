"""Attention over a 4-bit cache of bf16 at the ends of the type's range.

What the cache holds are numbers of its type up to 6 2^125 and down to 2^-126, and attention over
them is an average, so no output lies outside of what the values span: none may be an infinity,
and none may vanish.  Keys single out one row, whose score lies next to the power of two that the
running sums are kept to, in a later tile of a wave than others: there a probability is the
farthest from the maximum that the sums refer to.

Oracle: oracle/cache.py in 64 bits, of values taken times a power of two (exact), and
tests/cache_util.attention_bound with an absolute part that goes with them: products and their sums are
rounded to 2^-150 at worst (fp32's subnormal half step) in a scale of at least 2^-8 of the result's,
once for each row and again for each of 16 partial sums, and the output to 2^-134.
"""

import numpy as np
import pytest
import torch

from oracle import cache as ocache
from soupsuck_amd.kernels.paged import PagedCache, PagedCache4, cached_attention
from tests.cache4_util import build4, values
from tests.cache_util import attention_bound, host, offsets

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
# Rows of one wave's third tile whether a workgroup has eight waves, four or two, and of a range.
LENGTH, CHOSEN = 32 * 24 - 7, 32 * 16 + 5


def _chosen(device, hk, exponent, others):
    """A cache of rows that score 0 but for one that scores 1; value scales 2^exponent there and
    2^others elsewhere."""
    c = build4([LENGTH], hk, 16, device, seed=5)
    held = c.data[..., 2048:] != 255
    c.data[..., :1024] = 0
    c.data[..., 2048:2112][held[..., :64]] = 127
    c.data[..., 2112:][held[..., 64:]] = 127 + others
    page, row = c.table[0, CHOSEN // 16].item(), CHOSEN % 16
    c.data[page, :, 0, row * 16] = 0x11                     # 0.5 in two dimensions of block 0
    for block in range(4):
        c.data[page, :, 0, 2112 + block * 16 + row] = 127 + exponent
    return c


def _check(device, c, hq, new, rise, exponent, max_length):
    q = torch.ones((new, hq, 128), dtype=BF16, device=device)
    cu, scale = offsets([new], device), rise * np.log(2.0)
    got = host(cached_attention(q, PagedCache4(c.data, BF16), c.table, c.lengths, cu, new, max_length,
                                scale))
    k, v = values(c.data)
    v = v * 2.0 ** -exponent
    ref, spread, reach, _ = ocache.attention(host(q), k, v, c.table.tolist(), [LENGTH], [0, new],
                                             scale)
    small = (2.0 ** -134 + 2.0 ** (8 - 150) * (LENGTH + 16)) * 2.0 ** -exponent
    bound = attention_bound(BF16, ref, spread, reach, LENGTH) - 1e-7 + small
    assert np.isfinite(got).all()
    assert (np.abs(got * 2.0 ** -exponent - ref) / bound).max() <= 1


@pytest.mark.parametrize("max_length", [LENGTH, 100000])          # one workgroup a unit; split
@pytest.mark.parametrize("new,hq,hk", [(1, 6, 2), (9, 6, 2), (40, 4, 2), (40, 64, 32)])
@pytest.mark.parametrize("rise", [0.5, 7.9, 8.1, 20.0])
def test_values_at_the_top(device, rise, new, hq, hk, max_length):
    """6 2^123 with nearly all of the weight (and 2^112 elsewhere) are no infinity."""
    print(f"case values at the top {rise} {new} {hq} {max_length}", flush=True)
    c = _chosen(device, hk, 123, 112)
    _check(device, c, hq, new, rise, 123, max_length)


@pytest.mark.parametrize("max_length", [LENGTH, 100000])
@pytest.mark.parametrize("new,hq,hk", [(1, 6, 2), (9, 6, 2), (40, 4, 2), (40, 64, 32)])
@pytest.mark.parametrize("rise", [0.5, 7.9, 8.1])
def test_values_at_the_bottom(device, rise, new, hq, hk, max_length):
    """2^-126, the least normal number of the type, does not vanish."""
    print(f"case values at the bottom {rise} {new} {hq} {max_length}", flush=True)
    c = _chosen(device, hk, -125, -125)
    _check(device, c, hq, new, rise, -125, max_length)


@pytest.mark.parametrize("exponent,others", [(123, 112), (-125, -125)])
def test_as_over_16_bits(device, exponent, others):
    """The same rows in a 16-bit cache: results are an ordinary case's rounding apart."""
    c = _chosen(device, 2, exponent, others)
    k, v = (torch.from_numpy(np.nan_to_num(x)).to(BF16).contiguous().to(device) for x in values(c.data))
    q, cu = torch.ones((1, 6, 128), dtype=BF16, device=device), offsets([1], device)
    args = (c.table, c.lengths, cu, 1, LENGTH, 7.9 * np.log(2.0))
    four, wide = (host(cached_attention(q, cache, *args)) * 2.0 ** -exponent
                  for cache in (PagedCache4(c.data, BF16), PagedCache(k, v)))
    size = np.abs(values(c.data)[1][c.table[0, CHOSEN // 16].item(), :, CHOSEN % 16]).max()
    assert (np.abs(four - wide) <= 4 * 2.0 ** -8 * size * 2.0 ** -exponent).all()
