"""What the 4-bit cache, forks and beam selection refuse, before any launch (CPU)."""

import ctypes

import pytest
import torch

from soupsuck_amd import _lib
from soupsuck_amd.kernels.beams import select_beams
from soupsuck_amd.kernels.paged import (PagedCache, PagedCache4, append_kv, cached_attention,
                                        evict_kv, fork_kv, read_kv)

F16, BF16 = torch.float16, torch.bfloat16


def _cache(pages=4, heads=2, size=16, dtype=F16):
    return PagedCache4.empty(pages, heads, size, dtype, "cpu")


def _int32(*values):
    return torch.tensor(values, dtype=torch.int32)


def _bytes(*shape, dtype=torch.uint8):
    return torch.zeros(shape, dtype=dtype)


TABLE, LENGTHS, CU = torch.zeros((2, 3), dtype=torch.int32), _int32(5, 6), _int32(0, 1, 2)
ROWS = torch.zeros((2, 2, 128), dtype=F16)


@pytest.mark.parametrize("data,dtype,needle", [
    (_bytes(4, 2, 1, 2176, dtype=torch.int8), F16, "uint8"),
    (_bytes(4, 2, 1, 2048), F16, "2176"),
    (_bytes(4, 2, 2176), F16, "uint8"),
    (None, F16, "data"),
    (_bytes(4, 2, 1, 2176), torch.float32, "dtype"),
    (_bytes(4, 2, 1, 2176), None, "dtype"),
    (_bytes(0, 2, 1, 2176), F16, "at least one page"),
    (_bytes(4, 2, 0, 2176), F16, "at least one page"),
    (_bytes(4, 2, 1, 2184)[..., :2176], F16, "strides"),
    (_bytes(4, 2, 1, 2192)[..., 8:2184], F16, "aligned"),
    (_bytes(4, 2, 1, 4352)[..., ::2], F16, "strides"),
])
def test_caches(data, dtype, needle):
    with pytest.raises(ValueError, match=needle):
        PagedCache4(data, dtype)


@pytest.mark.parametrize("size", [0, 24, -16, 16.0, True])
def test_page_sizes(size):
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedCache4.empty(4, 2, size, F16, "cpu")


def test_properties():
    cache = _cache(4, 3, 48, BF16)
    assert (cache.page_size, cache.kv_heads, cache.dtype) == (48, 3, BF16)
    assert cache.data.shape == (4, 3, 3, 2176) and cache.device.type == "cpu"
    wide = PagedCache.empty(4, 3, 48, F16, "cpu")
    assert (wide.page_size, wide.kv_heads, wide.dtype) == (48, 3, F16)


@pytest.mark.parametrize("change,needle", [
    (dict(cache=_cache(dtype=BF16)), "k and v"),
    (dict(k=ROWS.float()), "k and v"),
    (dict(k=ROWS[:, :1]), "k and v"),
    (dict(q=ROWS), "q only with them"),
    (dict(cos=torch.zeros((2, 128), dtype=BF16), sin=torch.zeros((2, 128), dtype=BF16)),
     "cos and sin"),
    (dict(block_table=TABLE.long()), "block_table"),
    (dict(), "CUDA"),
])
def test_append(change, needle):
    args = dict(cache=_cache(), k=ROWS, v=ROWS, block_table=TABLE, lengths=LENGTHS, cu_seqlens=CU)
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        append_kv(**args)


@pytest.mark.parametrize("change,needle", [
    (dict(q=ROWS.to(BF16)), "q must be"),
    (dict(q=torch.zeros((2, 3, 128), dtype=F16)), "multiple of the cache"),
    (dict(max_new=0), "max_new"),
    (dict(scale=float("inf")), "scale"),
    (dict(weights_out=torch.zeros(2, 2, 48)), "4-bit cache gives no weights"),
    (dict(), "CUDA"),
])
def test_attention(change, needle):
    args = dict(q=ROWS, cache=_cache(), block_table=TABLE, lengths=LENGTHS, cu_seqlens=CU,
                max_new=1, max_length=48, scale=0.1)
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        cached_attention(**args)


def test_evict():
    with pytest.raises(ValueError, match="must be a PagedCache"):
        evict_kv(_cache(), TABLE, LENGTHS, torch.zeros(2, 2, 48), TABLE, 32, 48)


UNALIKE = [
    (_cache(), _cache(pages=5)), (_cache(), _cache(dtype=BF16)), (_cache(), _cache(heads=1)),
    (PagedCache.empty(4, 2, 16, F16, "cpu"), PagedCache.empty(4, 2, 32, F16, "cpu")),
    (PagedCache.empty(4, 2, 16, F16, "cpu"),
     PagedCache(torch.zeros((4, 16, 2, 128), dtype=F16).transpose(1, 2),
                torch.zeros((4, 2, 16, 128), dtype=F16))),
]


@pytest.mark.parametrize("change,needle", [
    (dict(caches=object()), "caches must be"),
    (dict(caches=[]), "caches must be"),
    (dict(caches=[_cache(), PagedCache.empty(4, 2, 16, F16, "cpu")]), "caches must be"),
    *((dict(caches=list(pair)), "one shape") for pair in UNALIKE),
    (dict(block_table=TABLE[0]), "block_table"),
    (dict(lengths=_int32(5)), "lengths"),
    (dict(cu_seqlens=_int32(0, 1)), "cu_seqlens"),
    (dict(tokens=-1), "tokens"),
    (dict(tokens=2.0), "tokens"),
    (dict(tokens=2 ** 31), "tokens"),
    (dict(), "CUDA"),
])
def test_read(change, needle):
    args = dict(caches=[_cache(), _cache()], block_table=TABLE, lengths=LENGTHS, cu_seqlens=CU,
                tokens=2)
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        read_kv(**args)


@pytest.mark.parametrize("change,needle", [
    (dict(caches=None), "caches must be"),
    *((dict(caches=tuple(pair)), "one shape") for pair in UNALIKE),
    (dict(block_table=TABLE.long()), "block_table"),
    (dict(lengths=LENGTHS.long()), "lengths"),
    (dict(parents=_int32(0, 1).long()), "parents"),
    (dict(parents=_int32(0)), "parents"),
    (dict(spare=_int32(0, 1, 2, 3)[::2]), "parents and spare"),
    (dict(parents=[0, 1]), "parents"),
    (dict(), "CUDA"),
])
def test_fork(change, needle):
    args = dict(caches=[_cache(), _cache()], block_table=TABLE, lengths=LENGTHS,
                parents=_int32(1, 0), spare=_int32(2, 3))
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        fork_kv(**args)


LOGITS, SCORES = torch.zeros((2, 3, 10)), torch.zeros((2, 3))


@pytest.mark.parametrize("change,needle", [
    (dict(logits=LOGITS.double()), "logits"),
    (dict(logits=LOGITS[0]), "logits"),
    (dict(logits=torch.zeros((2, 3, 20))[..., ::2]), "logits"),
    (dict(logits=torch.zeros((2, 3, 0))), "logits"),
    (dict(logits=LOGITS.clone().requires_grad_()), "logits"),
    (dict(logits=torch.zeros((2, 65, 4))), "64 beams"),
    (dict(logits=torch.zeros((2, 0, 4))), "64 beams"),
    (dict(logits=torch.zeros((65536, 1, 1))), "65535"),
    (dict(scores=SCORES.half()), "scores"),
    (dict(scores=SCORES[:, :2]), "scores"),
    (dict(scores=torch.zeros((3, 2)).t()), "scores"),
    (dict(count=0), "count"),
    (dict(count=31), "count"),
    (dict(count=65, logits=torch.zeros((2, 3, 100))), "count"),
    (dict(count=2.0), "count"),
    (dict(count=True), "count"),
    (dict(logits=torch.zeros((1, 64, 50)), scores=torch.zeros((1, 64)), count=33), "2048"),
    (dict(), "CUDA"),
])
def test_select(change, needle):
    args = dict(logits=LOGITS, scores=SCORES, count=4)
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        select_beams(**args)


# ------------------------------------------------------ the C entry points themselves

@pytest.fixture
def raw():
    """(library, cache struct, an aligned host address that is never read)."""
    buffer = (ctypes.c_uint8 * 256)()
    at = (ctypes.addressof(buffer) + 63) // 64 * 64
    cache = _lib.PagedCache4Struct(at, 8704, 4352, 2176, 4, 32, 2, 128, _lib.F16)
    return _lib.load(), cache, at, buffer


def _attention(lib, cache, at, **change):
    names = ("q q_tok q_head heads table stride pages lengths cu rows tokens max_new max_length "
             "scale window sinks o o_tok o_head ws ws_bytes stream").split()
    values = dict(zip(names, (at, 1024, 128, 4, at, 3, 3, at, at, 2, 2, 1, 48, 0.1, 0, 0,
                              at, 1024, 128, at, 0, None)))
    values.update(change)
    return lib.ss_cached_attention4(ctypes.byref(cache) if cache else None, *values.values())


def _refused(lib, rc, needle):
    assert rc == _lib.ERR_INVALID_ARGUMENT and needle in lib.ss_last_error().decode()


@pytest.mark.parametrize("change,needle", [
    (dict(heads=3), "multiple"), (dict(heads=0), "multiple"), (dict(q=None), "null"),
    (dict(o=None), "null"), (dict(table=None), "null"), (dict(cu=None), "null"),
    (dict(lengths=None), "null"), (dict(stride=2), "block table"), (dict(rows=-1), "block table"),
    (dict(tokens=-1), "negative"), (dict(window=-1), "negative"), (dict(sinks=-1), "negative"),
    (dict(q_tok=4), "aligned"), (dict(o_head=12), "aligned"), (dict(max_new=0), "max_new"),
    (dict(pages=2 ** 30, stride=2 ** 30), "rows"), (dict(tokens=2 ** 31), "too many"),
])
def test_c_attention(raw, change, needle):
    lib, cache, at, _ = raw
    _refused(lib, _attention(lib, cache, at, **change), needle)


def test_c_attention_workspace(raw):
    lib, cache, at, _ = raw
    need = lib.ss_cached_attention4_workspace_size(2, 2, 4, 2, 1, 100000)
    assert need > 0
    _refused(lib, _attention(lib, cache, at, max_length=100000, ws_bytes=need - 1), "workspace")


@pytest.mark.parametrize("field,value,needle", [
    ("data", None, "null"), ("dtype", _lib.F32, "dtype"), ("head_dim", 64, "head_dim"),
    ("pages", 0, "pages"), ("kv_heads", 0, "heads"), ("page_size", 24, "multiple of 16"),
    ("group", 2180, "aligned"), ("page", 8, "aligned"),
])
def test_c_caches(raw, field, value, needle):
    lib, cache, at, _ = raw
    setattr(cache, field, value)
    _refused(lib, _attention(lib, cache, at), needle)
    _refused(lib, _attention(lib, None, at), "null")


def _pointers(*caches):
    return (ctypes.c_void_p * len(caches))(*(ctypes.addressof(c) for c in caches))


def test_c_read_and_fork(raw):
    lib, cache, at, _ = raw
    other = _lib.PagedCache4Struct(at, 8704, 4352, 2176, 5, 32, 2, 128, _lib.F16)

    def read(caches=_pointers(cache), count=1, table=at, lengths=at, cu=at, rows=2, tokens=2, k=at):
        return lib.ss_kv_read4(caches, count, table, 3, 3, lengths, cu, rows, tokens, k, at, None)

    def fork(caches=_pointers(cache), count=1, table=at, rows=2, parents=at, spare=at, new=2,
             out=at):
        return lib.ss_kv_fork4(caches, count, table, 3, 3, at, rows, parents, spare, new, out, at,
                               None)

    for call in (read, fork):
        _refused(lib, call(count=0), "needs a cache")
        _refused(lib, call(caches=None), "needs a cache")
        _refused(lib, call(caches=_pointers(cache, other), count=2), "not like the first")
        _refused(lib, call(table=None), "null")
        _refused(lib, call(rows=-1), "block table")
    _refused(lib, read(cu=None), "null")
    _refused(lib, read(k=None), "null")
    _refused(lib, read(k=at + 8), "aligned")
    _refused(lib, read(tokens=-1), "negative")
    _refused(lib, read(tokens=2 ** 32), "too many")
    _refused(lib, fork(parents=None), "null")
    _refused(lib, fork(out=None), "null")
    _refused(lib, fork(new=-1), "negative")
    _refused(lib, fork(new=2 ** 31 - 1), "too many")
    assert read(tokens=0) == fork(new=0) == _lib.OK


def test_c_reads_and_forks_past_a_grid(raw):
    """Eight threads a row and head, 256 a new row, head and 16 rows: 2^32 of them are refused."""
    lib, cache, at, _ = raw
    tokens = 2 ** 32 // 8 // cache.kv_heads
    _refused(lib, lib.ss_kv_read4(_pointers(cache), 1, at, 3, 3, at, at, 2, tokens, at, at, None),
             "too many")
    rows = 2 ** 32 // 256 // cache.kv_heads // (cache.page_size // 16)
    _refused(lib, lib.ss_kv_fork4(_pointers(cache), 1, at, 3, 3, at, 2, at, at, rows, at, at, None),
             "too many")


@pytest.mark.parametrize("change,needle", [
    (dict(dtype=7), "dtype"), (dict(rows=-1), "sizes"), (dict(beams=0), "sizes"),
    (dict(beams=65), "sizes"), (dict(vocab=0), "sizes"), (dict(count=0), "sizes"),
    (dict(count=65), "sizes"), (dict(vocab=2 ** 31), "sizes"), (dict(logits=None), "null"),
    (dict(tokens=None), "null"), (dict(ws=None), "workspace"), (dict(ws_bytes=8), "workspace"),
])
def test_c_select(raw, change, needle):
    lib, _, at, _ = raw
    names = ("logits l_seq l_beam dtype scores rows beams vocab count out parents tokens ws ws_bytes "
             "stream").split()
    values = dict(zip(names, (at, 300, 100, _lib.F16, at, 2, 3, 100, 4, at, at, at, at, 0, None)))
    values.update(change)
    _refused(lib, lib.ss_select_beams(*values.values()), needle)


def test_c_append(raw):
    lib, cache, at, _ = raw
    args = [at, 256, 128, at, 256, 128, None, 0, 0, 0, None, 0, None, 0, _lib.F32, at, 3, 3, at, at,
            2, 2, None, 0, 0, None]
    for index, value, needle in ((0, None, "null"), (19, None, "null"), (21, -1, "negative"),
                                 (6, at, "go together"), (10, at, "go together"),
                                 (1, 4, "aligned"), (21, 2 ** 40, "too many")):
        changed = list(args)
        changed[index] = value
        _refused(lib, lib.ss_kv_append4(ctypes.byref(cache), *changed), needle)
