"""Sizes that the paged cache's kernels refuse before any launch (CPU)."""

import ctypes

import pytest

from soupsuck_amd import _lib
from tests.test_cache_refusals import _attention, raw  # noqa: F401


@pytest.mark.parametrize("field", ["k_row", "v_row"])
@pytest.mark.parametrize("value", [2 ** 26, 2 ** 40, -128])
def test_rows_far_apart(raw, field, value):  # noqa: F811
    lib, cache, at, _ = raw
    setattr(cache, field, value)
    assert _attention(lib, cache, at) == _lib.ERR_INVALID_ARGUMENT
    assert "2^26" in lib.ss_last_error().decode()


@pytest.mark.parametrize("change,needle", [
    (dict(max_new=0), "max_new"), (dict(pages=2 ** 27, stride=2 ** 27), "rows"),
    (dict(tokens=2 ** 28, max_new=2 ** 28, heads=2), "too many"),
])
def test_attention(raw, change, needle):  # noqa: F811
    lib, cache, at, _ = raw
    assert _attention(lib, cache, at, **change) == _lib.ERR_INVALID_ARGUMENT
    assert needle in lib.ss_last_error().decode()


def test_workspace_is_bounded_by_the_tokens_and_the_scores(raw):  # noqa: F811
    """Bounds far above what a call brings do not ask for memory in their proportion."""
    size = raw[0].ss_cached_attention_workspace_size
    few = size(4, 4, 12, 2, 1, 2048, 1)
    assert size(4, 4, 12, 2, 2 ** 30, 2048, 1) <= 8 * few + 2 ** 20
    assert size(64, 64, 28, 4, 1, 2 ** 31 - 1, 1) < 2 ** 27
    assert size(0, 4, 12, 2, 1, 2048, 1) == 0 == size(4, 4, 12, 5, 1, 2048, 1)
    assert ctypes.sizeof(ctypes.c_size_t) == 8
