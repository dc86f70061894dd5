"""The oracle of the 4-bit cache, forks and beam selection against independent statements (CPU)."""

import itertools

import numpy as np
import pytest

from oracle import cache4


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_what_a_block_can_hold_it_keeps(dtype):
    low, high = cache4.EXPONENTS[dtype]
    values = np.concatenate((cache4.STEPS, -cache4.STEPS))
    for e in (low, low + 1, 0, 3, high):
        x = np.resize(values, 128) * 2.0 ** e
        np.testing.assert_array_equal(cache4.held(x, dtype), x)


def test_held_is_the_nearest_of_what_the_scale_allows():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((500, 128)) * np.exp(rng.uniform(-5, 5, (500, 1)))
    got = cache4.held(x, "bfloat16")
    blocks, held = x.reshape(-1, 32), got.reshape(-1, 32)
    for block, values in zip(blocks[:300], held):
        top = np.abs(block).max()
        scale = next(2.0 ** e for e in itertools.count(-30) if 6 * 2.0 ** e >= top)
        grid = np.concatenate((cache4.STEPS, -cache4.STEPS)) * scale
        near = grid[np.abs(block[:, None] - grid).argmin(-1)]
        np.testing.assert_allclose(np.abs(block - values), np.abs(block - near), rtol=0, atol=0)
    np.testing.assert_array_equal(cache4.held(got, "bfloat16"), got)


def test_ties_go_to_even_codes():
    x = np.zeros(128)
    x[:8] = 6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5
    np.testing.assert_array_equal(cache4.held(x, "float16")[:8], [6, 0, 1, 1, 2, 2, 4, 4])
    np.testing.assert_array_equal(cache4.held(-x, "float16")[:8], [-6, 0, -1, -1, -2, -2, -4, -4])


def test_ends_of_the_range_and_numbers_that_are_none():
    x = np.zeros((3, 128))
    x[0, :2] = 60000, 2.0 ** -14
    x[1, 3] = np.inf
    x[2, 40] = np.nan
    got = cache4.held(x, "float16")
    assert got[0, 0] == 6 * 2.0 ** 13 and got[0, 1] == 0
    assert np.isnan(got[1, :32]).all() and (got[1, 32:] == 0).all()
    assert np.isnan(got[2, 32:64]).all() and (got[2, :32] == 0).all()
    small = np.full(128, 2.0 ** -14 * 0.5)
    assert (cache4.held(small, "float16") == 0).all()          # half of the least step: to even
    assert (cache4.held(small * 1.01, "float16") == 2.0 ** -14).all()


def test_bytes():
    data = np.zeros((2, 1, 2, 2176), np.uint8)
    k, v = np.zeros(128), np.zeros(128)
    k[33], v[9] = 3.0, -1.5
    cache4.pack(data, 1, 0, 18, k, v, "bfloat16")
    group = data[1, 0, 1]                       # row 18 is row 2 of the second group
    assert group[1 * 256 + 2 * 16 + 0] == 0x70  # dimension 33: high half, code of 6 at scale 1/2
    assert group[2048 + 1 * 16 + 2] == 126
    assert group[1024 + 0 + 1 * 16 + 2 * 4 + 0] == 0xF0
    assert group[2112 + 0 + 2] == 125
    keys, values = cache4.unpack(data)
    np.testing.assert_array_equal(keys[1, 0, 18], k)
    np.testing.assert_array_equal(values[1, 0, 18], v)
    assert np.count_nonzero(keys) == np.count_nonzero(values) == 1


def test_fork():
    table = [[3, 4, -1], [5, 6, 7]]
    new, lengths, copies = cache4.fork(table, [20, 48], [1, 0, 0, -1], [8, 9, 10, 11], 16, 12)
    np.testing.assert_array_equal(new, [[5, 6, 7], [3, 9, -1], [3, 10, -1], [11, -1, -1]])
    np.testing.assert_array_equal(lengths, [48, 20, 20, 0])
    assert copies == [(4, 9, 4), (4, 10, 4)]


def test_select():
    rng = np.random.default_rng(2)
    x, scores = rng.standard_normal((3, 11)), np.array([-1.0, -1.5, -9.0])
    p = np.log(np.exp(x) / np.exp(x).sum(-1, keepdims=True)) + scores[:, None]
    want = np.sort(p, None)[::-1][:6]
    got, parents, tokens = cache4.select(x, scores, 6)
    np.testing.assert_allclose(got, want, rtol=1e-12)
    np.testing.assert_allclose(p[parents, tokens], want, rtol=1e-12)
    _, parents, tokens = cache4.select(np.zeros((2, 4)), np.zeros(2), 5)
    assert parents.tolist() == [0, 0, 0, 0, 1] and tokens.tolist() == [0, 1, 2, 3, 0]
