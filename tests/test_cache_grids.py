"""Cache calls whose grids would have 2^32 threads or more are refused before any launch (CPU).

A launch has whole workgroups, so what counts is the number of threads rounded up to them.
"""

import ctypes

import pytest

from soupsuck_amd import _lib
from tests.test_cache4_refusals import raw as raw4  # noqa: F401
from tests.test_cache_refusals import raw  # noqa: F401

GROUP = 256


def _too_many(lib, rc):
    assert rc == _lib.ERR_INVALID_ARGUMENT
    assert "too many" in lib.ss_last_error().decode()


def _append(call, cache, at, tokens, q_heads=0):
    q = (at, 1024, 128, q_heads) if q_heads else (None, 0, 0, 0)
    angles = (at, 128, at, 128) if q_heads else (None, 0, None, 0)
    out = (at, 1024, 128) if q_heads else (None, 0, 0)
    return call(ctypes.byref(cache), at, 256, 128, at, 256, 128, *q, *angles, _lib.F32, at, 3, 3,
                at, at, 2, tokens, *out, None)


@pytest.mark.parametrize("q_heads", [0, 3, 12])
def test_append(raw, raw4, q_heads):  # noqa: F811
    """Eight threads for each row of a head, or for four query heads of a row (4 bits)."""
    lib, cache, at, _ = raw
    _, cache4, at4, _ = raw4
    for call, struct, base, queries in ((lib.ss_kv_append, cache, at, q_heads),
                                        (lib.ss_kv_append4, cache4, at4, -(-q_heads // 4))):
        items = queries + 2 * struct.kv_heads
        most = (2 ** 32 // GROUP - 1) * (GROUP // 8)
        for tokens in (most // items + 1, 2 ** 32 // 8 // items, 2 ** 31 // (q_heads + 4) - 1):
            _too_many(lib, _append(call, struct, base, tokens, q_heads))


def test_read_of_whole_workgroups(raw4):  # noqa: F811
    """Fewer than 2^32 threads, but not once the last workgroup is whole."""
    lib, cache, at, _ = raw4
    cache.kv_heads = 1
    caches = (ctypes.c_void_p * 1)(ctypes.addressof(cache))
    for tokens in (2 ** 32 // 8 - 1, 2 ** 32 // 8 - 31):
        _too_many(lib, lib.ss_kv_read4(caches, 1, at, 3, 3, at, at, 2, tokens, at, at, None))


def _attention(call, cache, at, tokens, weights):
    return call(ctypes.byref(cache), at, 256, 128, 2, at, 3, 3, None, None, 0, tokens, 1, 48, 0.1,
                0, 0, *weights, at, 256, 128, None, 0, None)


def test_attention_without_sequences(raw, raw4):  # noqa: F811
    """Zeros are written by 16 threads a row of a head."""
    lib, cache, at, _ = raw
    _, cache4, at4, _ = raw4
    for tokens in (2 ** 32 // 16 // 2, 2 ** 30 - 1, 2 ** 32 // 16 // 2 - 7):
        _too_many(lib, _attention(lib.ss_cached_attention, cache, at, tokens, (None, None)))
        _too_many(lib, _attention(lib.ss_cached_attention4, cache4, at4, tokens, ()))


@pytest.mark.parametrize("rows,out_pages", [(2 ** 21, 2), (2 ** 31 - 1, 1), (2 ** 20, 2 ** 3)])
def test_evict(raw, rows, out_pages):  # noqa: F811
    """1024 threads for each kv head of a sequence; 16 for each row that it may keep."""
    lib, cache, at, _ = raw
    rc = lib.ss_kv_evict(ctypes.byref(cache), at, 3, 3, at, rows, 48, at, at, out_pages, out_pages,
                         16, 0, 0, at, at, at, 2 ** 62, None)
    _too_many(lib, rc)
