"""What the paged cache and the draft check refuse, before any launch (CPU)."""

import ctypes

import pytest
import torch

from soupsuck_amd import _lib
from soupsuck_amd.kernels.paged import PagedCache, append_kv, cached_attention, evict_kv
from soupsuck_amd.kernels.verify import verify_drafts

F16 = torch.float16


def _cache(pages=4, heads=2, size=16, dtype=F16):
    return PagedCache.empty(pages, heads, size, dtype, "cpu")


def _int32(*values):
    return torch.tensor(values, dtype=torch.int32)


TABLE, LENGTHS, CU = torch.zeros((2, 3), dtype=torch.int32), _int32(5, 6), _int32(0, 1, 2)
ROWS = torch.zeros((2, 2, 128), dtype=F16)


@pytest.mark.parametrize("k,v,needle", [
    (torch.zeros(4, 2, 16, 128), torch.zeros(4, 2, 16, 128), "fp16 or bf16"),
    (torch.zeros(4, 2, 16, 64, dtype=F16), torch.zeros(4, 2, 16, 64, dtype=F16), "128"),
    (torch.zeros(4, 2, 16, 128, dtype=F16), torch.zeros(4, 2, 32, 128, dtype=F16), "one shape"),
    (torch.zeros(4, 2, 16, 128, dtype=F16), torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16),
     "one shape"),
    (torch.zeros(4, 2, 24, 128, dtype=F16),) * 2 + ("multiple of 16",),
    (torch.zeros(0, 2, 16, 128, dtype=F16),) * 2 + ("at least one page",),
    (torch.zeros(4, 2, 16, 129, dtype=F16)[..., :128],) * 2 + ("strides",),
    (torch.zeros(4, 2, 16, 256, dtype=F16)[..., ::2],) * 2 + ("strides",),
    (None, None, "k and v"),
])
def test_caches(k, v, needle):
    with pytest.raises(ValueError, match=needle):
        PagedCache(k, v)


@pytest.mark.parametrize("change,needle", [
    (dict(cache=object()), "PagedCache"),
    (dict(block_table=TABLE.long()), "block_table"),
    (dict(block_table=TABLE[0]), "block_table"),
    (dict(lengths=_int32(5)), "lengths"),
    (dict(lengths=LENGTHS.long()), "lengths"),
    (dict(cu_seqlens=_int32(0, 1)), "cu_seqlens"),
    (dict(k=ROWS.float()), "k and v"),
    (dict(k=ROWS[:, :1]), "k and v"),
    (dict(v=ROWS[:1]), "k and v"),
    (dict(q=ROWS), "q only with them"),
    (dict(cos=torch.zeros(2, 128)), "cos and sin"),
    (dict(cos=torch.zeros(2, 64), sin=torch.zeros(2, 64)), "cos and sin"),
    (dict(cos=torch.zeros(2, 128, dtype=torch.bfloat16),
          sin=torch.zeros(2, 128, dtype=torch.bfloat16)), "cos and sin"),
    (dict(q=ROWS.float(), cos=torch.zeros(2, 128), sin=torch.zeros(2, 128)), "q must be"),
    (dict(k=torch.zeros((2, 2, 132), dtype=F16)[..., :128]), "strides"),
    (dict(), "CUDA"),
])
def test_append(change, needle):
    args = dict(cache=_cache(), k=ROWS, v=ROWS, block_table=TABLE, lengths=LENGTHS, cu_seqlens=CU)
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        append_kv(**args)


@pytest.mark.parametrize("change,needle", [
    (dict(q=ROWS.float()), "q must be"),
    (dict(q=ROWS[..., :64]), "q must be"),
    (dict(q=ROWS.clone().requires_grad_()), "q must be"),
    (dict(q=torch.zeros((2, 3, 128), dtype=F16)), "multiple of the cache"),
    (dict(q=torch.zeros((2, 2, 130), dtype=F16)[..., :128]), "strides"),
    (dict(max_new=0), "max_new"),
    (dict(max_new=True), "max_new"),
    (dict(max_length=-1), "max_length"),
    (dict(max_length=2 ** 31), "max_length"),
    (dict(scale=float("nan")), "scale"),
    (dict(window=0), "window"),
    (dict(window=2.5), "window"),
    (dict(sinks=-1), "sinks"),
    (dict(weights=torch.zeros(2, 2, 48)), "only with weights_out"),
    (dict(weights_out=torch.zeros(2, 2, 47)), "weights"),
    (dict(weights_out=torch.zeros(2, 2, 48, dtype=F16)), "weights"),
    (dict(), "CUDA"),
])
def test_attention(change, needle):
    args = dict(q=ROWS, cache=_cache(), block_table=TABLE, lengths=LENGTHS, cu_seqlens=CU,
                max_new=1, max_length=48, scale=0.1)
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        cached_attention(**args)


@pytest.mark.parametrize("change,needle", [
    (dict(weights=torch.zeros(2, 2, 32)), "weights"),
    (dict(out_table=TABLE[:1]), "out_table"),
    (dict(budget=0), "budget"),
    (dict(budget=49), "budget"),
    (dict(sinks=20, recent=13), "within the budget"),
    (dict(sinks=-1), "sinks"),
    (dict(max_length=-1), "max_length"),
    (dict(), "CUDA"),
])
def test_evict(change, needle):
    args = dict(cache=_cache(), block_table=TABLE, lengths=LENGTHS,
                weights=torch.zeros(2, 2, 48), out_table=TABLE, budget=32, max_length=48)
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        evict_kv(**args)


LOGITS = torch.zeros((2, 3, 10))


@pytest.mark.parametrize("change,needle", [
    (dict(target_logits=LOGITS.double()), "target_logits"),
    (dict(target_logits=LOGITS[0]), "target_logits"),
    (dict(target_logits=torch.zeros((2, 3, 20))[..., ::2]), "target_logits"),
    (dict(target_logits=torch.zeros((2, 3, 0))), "target_logits"),
    (dict(draft_tokens=torch.zeros((2, 2), dtype=torch.int32)), "draft_tokens"),
    (dict(draft_tokens=torch.zeros((2, 3), dtype=torch.int64)), "draft_tokens"),
    (dict(temperature=-0.5), "temperature"),
    (dict(temperature=float("inf")), "temperature"),
    (dict(uniform=None), "uniform"),
    (dict(uniform=torch.zeros((2, 2))), "uniform"),
    (dict(uniform=torch.zeros((2, 3), dtype=torch.float64)), "uniform"),
    (dict(draft_logits=LOGITS), "draft_logits"),
    (dict(draft_logits=LOGITS[:, :2].half()), "draft_logits"),
    (dict(draft_counts=torch.zeros(2, dtype=torch.int64)), "draft_counts"),
    (dict(target_logits=torch.zeros((30000, 3, 1)),
          draft_tokens=torch.zeros((30000, 2), dtype=torch.int64),
          uniform=torch.zeros((30000, 3))), "65535"),
    (dict(), "CUDA"),
])
def test_verify(change, needle):
    args = dict(target_logits=LOGITS, draft_tokens=torch.zeros((2, 2), dtype=torch.int64),
                uniform=torch.zeros((2, 3)))
    args.update(change)
    with pytest.raises(ValueError, match=needle):
        verify_drafts(**args)


# ------------------------------------------------------ the C entry points themselves

@pytest.fixture
def raw():
    """(library, cache struct, an aligned host address that is never read)."""
    buffer = (ctypes.c_uint8 * 256)()
    at = (ctypes.addressof(buffer) + 63) // 64 * 64
    cache = _lib.PagedCacheStruct(at, 4096, 2048, 128, at, 4096, 2048, 128, 4, 16, 2, 128,
                                  _lib.F16)
    return _lib.load(), cache, at, buffer


def _attention(lib, cache, at, **change):
    names = ("q q_tok q_head heads table stride pages lengths cu rows tokens max_new max_length "
             "scale window sinks w_in w_out o o_tok o_head ws ws_bytes stream").split()
    values = dict(zip(names, (at, 1024, 128, 4, at, 3, 3, at, at, 2, 2, 1, 48, 0.1, 0, 0, None,
                              None, at, 1024, 128, at, 0, None)))
    values.update(change)
    return lib.ss_cached_attention(ctypes.byref(cache) if cache else None, *values.values())


@pytest.mark.parametrize("change,needle", [
    (dict(heads=3), "multiple"), (dict(heads=0), "multiple"), (dict(q=None), "null"),
    (dict(o=None), "null"), (dict(table=None), "null"), (dict(cu=None), "null"),
    (dict(lengths=None), "null"), (dict(stride=2), "block table"), (dict(pages=0), "block table"),
    (dict(rows=-1), "block table"), (dict(tokens=-1), "negative"), (dict(window=-1), "negative"),
    (dict(sinks=-1), "negative"), (dict(max_length=-1), "negative"), (dict(q_tok=4), "aligned"),
    (dict(o_head=12), "aligned"), (dict(pages=2 ** 30, stride=2 ** 30), "rows"),
    (dict(tokens=2 ** 31), "too many"),
])
def test_c_attention(raw, change, needle):
    lib, cache, at, _ = raw
    assert _attention(lib, cache, at, **change) == _lib.ERR_INVALID_ARGUMENT
    assert needle in lib.ss_last_error().decode()


def test_c_attention_workspace(raw):
    lib, cache, at, _ = raw
    need = lib.ss_cached_attention_workspace_size(2, 2, 4, 2, 1, 48, 1)
    assert need > 0
    assert _attention(lib, cache, at, w_out=at, ws_bytes=need - 1) == _lib.ERR_INVALID_ARGUMENT
    assert "workspace" in lib.ss_last_error().decode()


@pytest.mark.parametrize("field,value,needle", [
    ("k", None, "null"), ("dtype", _lib.F32, "dtype"), ("head_dim", 64, "head_dim"),
    ("pages", 0, "pages"), ("kv_heads", 0, "heads"), ("page_size", 24, "multiple of 16"),
    ("page_size", 0, "multiple of 16"), ("v_row", 132, "aligned"),
])
def test_c_caches(raw, field, value, needle):
    lib, cache, at, _ = raw
    setattr(cache, field, value)
    assert _attention(lib, cache, at) == _lib.ERR_INVALID_ARGUMENT
    assert needle in lib.ss_last_error().decode()
    assert _attention(lib, None, at) == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("change,needle", [
    (dict(k=None), "null"), (dict(cu=None), "null"), (dict(tokens=-1), "negative"),
    (dict(q=1), "go together"), (dict(cos=1), "go together"), (dict(k_tok=4), "aligned"),
    (dict(tokens=2 ** 40), "too many"),
])
def test_c_append(raw, change, needle):
    lib, cache, at, _ = raw
    names = ("k k_tok k_head v v_tok v_head q q_tok q_head heads cos cos_tok sin sin_tok cs table "
             "stride pages lengths cu rows tokens q_out qo_tok qo_head stream").split()
    values = dict(zip(names, (at, 256, 128, at, 256, 128, None, 0, 0, 0, None, 0, None, 0, 0, at, 3,
                              3, at, at, 2, 2, None, 0, 0, None)))
    values.update({n: at if v == 1 else v for n, v in change.items()})
    assert lib.ss_kv_append(ctypes.byref(cache), *values.values()) == _lib.ERR_INVALID_ARGUMENT
    assert needle in lib.ss_last_error().decode()


@pytest.mark.parametrize("change,needle", [
    (dict(weights=None), "null"), (dict(budget=0), "budget"), (dict(sinks=-1), "budget"),
    (dict(sinks=20, recent=13), "budget"), (dict(recent=2 ** 62, sinks=2 ** 62), "budget"),
    (dict(out_pages=1), "hold"), (dict(out_stride=1), "hold"), (dict(max_length=-1), "max_length"),
    (dict(ws_bytes=8), "workspace"), (dict(ws=None), "workspace"),
])
def test_c_evict(raw, change, needle):
    lib, cache, at, _ = raw
    names = ("table stride pages lengths rows max_length weights out_table out_stride out_pages "
             "budget sinks recent out_lengths out_weights ws ws_bytes stream").split()
    values = dict(zip(names, (at, 3, 3, at, 2, 48, at, at, 2, 2, 32, 0, 0, at, at, at, 2 ** 20,
                              None)))
    values.update(change)
    assert lib.ss_kv_evict(ctypes.byref(cache), *values.values()) == _lib.ERR_INVALID_ARGUMENT
    assert needle in lib.ss_last_error().decode()


@pytest.mark.parametrize("change,needle", [
    (dict(dtype=3), "dtype"), (dict(vocab=0), "bad sizes"), (dict(vocab=2 ** 31), "bad sizes"),
    (dict(drafts=-1), "bad sizes"), (dict(rows=-1), "bad sizes"), (dict(heat=-1.0), "temperature"),
    (dict(heat=float("nan")), "temperature"), (dict(target=None), "null"),
    (dict(uniform=None), "null"), (dict(rows=20000), "too many"), (dict(drafts=40000), "too many"),
    (dict(ws_bytes=8), "workspace"),
])
def test_c_verify(raw, change, needle):
    lib, _, at, _ = raw
    names = ("target t_seq t_row draft d_seq d_row dtype tokens counts uniform rows drafts vocab "
             "heat accepted out ws ws_bytes stream").split()
    values = dict(zip(names, (at, 40, 10, at, 30, 10, 0, at, None, at, 2, 3, 10, 1.0, at, at, at,
                              2 ** 20, None)))
    values.update(change)
    assert lib.ss_verify_drafts(*values.values()) == _lib.ERR_INVALID_ARGUMENT
    assert needle in lib.ss_last_error().decode()
