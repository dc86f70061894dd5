"""The cache and verification oracle against independent statements of the same things (CPU)."""

import numpy as np
import pytest

from oracle import attention as oattn
from oracle import cache as ocache
from oracle import rope as orope


def paged(x, size, order):
    """[T, H, D] rows laid into pages in the given order."""
    t, h, d = x.shape
    pages = np.full((max(order) + 1, h, size, d), np.nan)
    for j in range(t):
        pages[order[j // size], :, j % size] = x[j]
    return pages


@pytest.fixture
def prompt():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((37, 6, 16)), *rng.standard_normal((2, 37, 2, 16))
    order = [2, 0, 4]
    return q, k, v, paged(k, 16, order), paged(v, 16, order), [order]


def test_a_whole_prompt_is_causal_attention(prompt):
    q, k, v, kc, vc, table = prompt
    ref, _ = oattn.forward(q, k, v, [37], 0.25)
    got, _, _, weights = ocache.attention(q, kc, vc, table, [37], [0, 37], 0.25)
    np.testing.assert_allclose(got, ref, rtol=1e-12, atol=1e-12)
    assert weights.sum() == pytest.approx(37 * 6) and (weights[:, :, 37:] == 0).all()


@pytest.mark.parametrize("window,sinks", [(37, 0), (5, 37), (1000, 3)])
def test_masks_that_hide_nothing(prompt, window, sinks):
    q, _, _, kc, vc, table = prompt
    args = (q[:9], kc, vc, table, [37], [0, 9], 0.25)
    np.testing.assert_allclose(ocache.attention(*args, window, sinks)[0],
                               ocache.attention(*args)[0], rtol=0, atol=0)


def test_window_of_one_without_sinks_is_the_row_itself(prompt):
    q, _, v, kc, vc, table = prompt
    got = ocache.attention(q, kc, vc, table, [37], [0, 37], 0.25, 1, 0)[0]
    np.testing.assert_allclose(got, np.repeat(v, 3, 1), rtol=1e-12)


def test_rotation_is_the_training_rotation_up_to_its_roundings():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((1, 4, 7, 128)).astype(np.float32)
    angle = rng.uniform(0, 6, (1, 7, 64)).astype(np.float32)
    cos, sin = (np.concatenate([f(angle)] * 2, -1) for f in (np.cos, np.sin))
    ref = orope.rope_forward(x, cos, sin)
    got = ocache.rotate(x, cos[:, None], sin[:, None])
    np.testing.assert_allclose(got, ref, rtol=0, atol=4 * 2.0 ** -24 * 8)


def test_evict_keeps_ends_and_heaviest():
    k = np.arange(4 * 1 * 16 * 1, dtype=np.float64).reshape(4, 1, 16, 1)
    w = np.zeros((1, 1, 32), np.float32)
    w[0, 0, [5, 9, 20]] = [1.0, 3.0, 1.0]      # 5 and 20 tie: the lower row stays
    n, nw, kc, _ = ocache.evict(k, k, [[1, 0]], [25], w, [[3]], 6, 2, 2)
    assert n.tolist() == [6]
    assert kc[3, 0, :6, 0].tolist() == [16, 17, 16 + 5, 16 + 9, 7, 8]
    assert nw[0, 0, :7].tolist() == [0, 0, 1, 3, 0, 0, 0]


@pytest.mark.parametrize("looked_up", [False, True])
def test_verified_tokens_are_distributed_as_the_target(looked_up):
    """The first token of many checks: frequencies within 4.5 standard deviations of p."""
    rng = np.random.default_rng(11)
    target, draft = rng.standard_normal((2, 2, 6)) * 1.5
    p, q = (ocache.probabilities(x[0], 0.8) for x in (target, draft))
    runs = 20000
    seen = np.zeros(6)
    for _ in range(runs):
        x = 2 if looked_up else rng.choice(6, p=q)
        _, out = ocache.verify(target, [x], rng.random(2), None if looked_up else draft[:1],
                               temperature=0.8)
        seen[out[0]] += 1
    assert (np.abs(seen - runs * p) < 4.5 * np.sqrt(runs * p * (1 - p))).all()


def test_a_planted_mistake_is_seen():
    """Drawing from p instead of max(p - q, 0) is far outside the same bound."""
    rng = np.random.default_rng(11)
    target, draft = rng.standard_normal((2, 2, 6)) * 1.5
    p, q = (ocache.probabilities(x[0], 0.8) for x in (target, draft))
    seen = np.zeros(6)
    for _ in range(20000):
        x = rng.choice(6, p=q)
        seen[x if rng.random() * q[x] < p[x] else ocache.draw(p, rng.random())] += 1
    assert (np.abs(seen - 20000 * p) > 4.5 * np.sqrt(20000 * p * (1 - p))).any()
