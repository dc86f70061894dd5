"""Paged key-value cache: append, attention of new tokens, eviction, beams (16 or 4 bits).

What generation with the tuned projections needs beside them; the reference trains only
and has no counterpart.  Keys and values lie in pages ([pages, kv heads, page size, 128]); a
sequence's pages are named by its line of a block table, so sequences grow without copies
and share a start.  New tokens are packed back to back as in
``packed_causal_attention`` (``row_offsets`` builds their offsets) and are each sequence's
last cache rows: ``lengths`` counts them in.

    cache = PagedCache.empty(pages, kv_heads, page_size, dtype, device)
    q = append_kv(cache, k, v, block_table, lengths, cu, q=q, cos=cos, sin=sin)
    o = cached_attention(q, cache, block_table, lengths, cu, max_new, max_length,
                         weights=weights, weights_out=weights)
    lengths, weights = evict_kv(cache, block_table, lengths, weights, fresh, budget, max_length,
                                sinks=4, recent=256)

``PagedCache4`` holds the rows in 4 bits a value (136 bytes a row and head instead of 512) and
stands wherever a ``PagedCache`` does, except in ``evict_kv`` and for attention weights.
``read_kv`` gives rows back as a cache holds them.  ``fork_kv`` lets sequences continue others,
as beams do (``kernels.beams.select_beams`` chooses them):

    scores, parents, tokens = select_beams(logits, scores, beams)
    table, lengths = fork_kv(caches, table, lengths, row_of(parents), spare_pages)

Block tables, lengths and offsets are read on the device: no call waits for it, and all
of them can be captured into a graph whose replays see the lengths of the moment
(``max_new`` and ``max_length`` are bounds, fixed at capture).  A table entry that names no
page of the cache, -1 for instance, is a page the sequence does not hold: nothing is read from or written
to it.
"""

import ctypes

import torch

from .. import _lib, native
from ..contract import Rule, enforce, finite_real

HEAD_DIM = 128
_CODES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _strided(t):
    """16-byte aligned base, unit last stride, other strides multiples of 16 bytes."""
    unit = 16 // t.element_size()
    return (t.data_ptr() % 16 == 0 and t.stride(-1) == 1
            and all(s % unit == 0 for s in t.stride()[:-1]))


def _whole(value, minimum):
    return isinstance(value, int) and not isinstance(value, bool) and value >= minimum


def _index(t):
    """The tensor's GPU, -1 where it is on none."""
    return t.device.index if t.is_cuda else -1


CACHE_RULES = (
    Rule("PagedCache: k and v must be [pages, kv_heads, page_size, 128] fp16 or bf16 tensors of "
         "one shape, dtype and device, without gradients",
         lambda a: all(isinstance(t, torch.Tensor) and t.ndim == 4 and t.shape[3] == HEAD_DIM
                       and t.dtype in (torch.float16, torch.bfloat16) and not t.requires_grad
                       for t in (a.k, a.v))
         and a.k.shape == a.v.shape and a.k.dtype == a.v.dtype and a.k.device == a.v.device),
    Rule("PagedCache: needs at least one page and head and a page size that is a multiple of 16",
         lambda a: a.k.shape[0] > 0 and a.k.shape[1] > 0 and a.k.shape[2] > 0
         and a.k.shape[2] % 16 == 0),
    Rule("PagedCache: k and v need 16-byte aligned bases, a unit last stride and strides that "
         "are multiples of 8", lambda a: _strided(a.k) and _strided(a.v)),
)


class PagedCache:
    """Pages of 16-bit keys and values: the tensors ``k`` and ``v`` [pages, kv_heads, page_size, 128]."""

    def __init__(self, k, v):
        enforce(CACHE_RULES, k=k, v=v)
        self._k, self._v = k, v
        pages, heads, size, dim = k.shape
        self._struct = _lib.PagedCacheStruct(
            k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], pages, size, heads, dim,
            _CODES[k.dtype])
        self._pointer = ctypes.addressof(self._struct)
        self._index = _index(k)

    @classmethod
    def empty(cls, pages, kv_heads, page_size, dtype=torch.float16, device="cuda"):
        """A cache of uninitialised pages."""
        shape = (pages, kv_heads, page_size, HEAD_DIM)
        return cls(torch.empty(shape, dtype=dtype, device=device),
                   torch.empty(shape, dtype=dtype, device=device))

    @property
    def k(self):
        return self._k

    @property
    def v(self):
        return self._v

    @property
    def dtype(self):
        return self._k.dtype

    @property
    def device(self):
        return self._k.device

    @property
    def kv_heads(self):
        return self._k.shape[1]

    @property
    def page_size(self):
        return self._k.shape[2]


GROUP_BYTES = 2176  # of 16 rows: key codes, value codes, key scales, value scales


CACHE4_RULES = (
    Rule("PagedCache4: data must be a uint8 [pages, kv_heads, page_size / 16, 2176] tensor",
         lambda a: isinstance(a.data, torch.Tensor) and a.data.dtype == torch.uint8
         and a.data.ndim == 4 and a.data.shape[3] == GROUP_BYTES),
    Rule("PagedCache4: dtype must be torch.float16 or torch.bfloat16",
         lambda a: a.dtype in (torch.float16, torch.bfloat16)),
    Rule("PagedCache4: needs at least one page and head and a page size that is a multiple of 16",
         lambda a: all(n > 0 for n in a.data.shape[:3])),
    Rule("PagedCache4: data needs a 16-byte aligned base, a unit last stride and strides that "
         "are multiples of 16", lambda a: _strided(a.data)),
)


class PagedCache4:
    """Pages of keys and values in 4 bits: the bytes ``data`` [pages, kv_heads, page_size / 16, 2176].

    Every 32 values of a row share a scale 2^e; a value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times
    it, with a sign.  e is the least with which none is past 6 (-13 to 13 for fp16, -125 to 125
    for bf16: beyond, values are held as 6 2^e); rounding is to nearest even.  A block with an
    infinity or NaN reads as NaN.  ``dtype`` is the type of the tensors around the cache; the
    bytes' layout is in include/soupsuck_amd.h.
    """

    def __init__(self, data, dtype=torch.float16):
        enforce(CACHE4_RULES, data=data, dtype=dtype)
        self._data, self._dtype = data, dtype
        pages, heads, groups, _ = data.shape
        self._struct = _lib.PagedCache4Struct(data.data_ptr(), *data.stride()[:3], pages,
                                              16 * groups, heads, HEAD_DIM, _CODES[dtype])
        self._pointer = ctypes.addressof(self._struct)
        self._index = _index(data)

    @classmethod
    def empty(cls, pages, kv_heads, page_size, dtype=torch.float16, device="cuda"):
        """A cache of uninitialised pages (``page_size`` a multiple of 16)."""
        if not _whole(page_size, 16) or page_size % 16:
            raise ValueError("PagedCache4: page_size must be a multiple of 16")
        return cls(torch.empty((pages, kv_heads, page_size // 16, GROUP_BYTES), dtype=torch.uint8,
                               device=device), dtype)

    @property
    def data(self):
        return self._data

    @property
    def dtype(self):
        return self._dtype

    @property
    def device(self):
        return self._data.device

    @property
    def kv_heads(self):
        return self._data.shape[1]

    @property
    def page_size(self):
        return 16 * self._data.shape[2]


def _table(t):
    return (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.ndim == 2
            and t.shape[1] > 0 and (t.stride(1) == 1 or t.shape[1] == 1)
            and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1))


def _line_stride(t):
    """Stride between the lines of a block table (any value serves where there is one)."""
    return max(t.stride(0), t.shape[1])


def _int32_line(t, n):
    return (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.ndim == 1
            and t.shape[0] == n and (t.is_contiguous()))


def _packed(t, cache, heads=None):
    return (isinstance(t, torch.Tensor) and t.ndim == 3 and t.dtype == cache.dtype
            and t.shape[2] == HEAD_DIM and (heads is None or t.shape[1] == heads)
            and not t.requires_grad)


def _is_cache(cache):
    return isinstance(cache, PagedCache)


def _is_cache4(cache):
    return isinstance(cache, PagedCache4)


def _any_cache(name):
    return Rule(f"{name}: cache must be a PagedCache or a PagedCache4",
                lambda a: _is_cache(a.cache) or _is_cache4(a.cache))


def _rows_rules(name, with_offsets=True, cache_rule=None):
    rules = [
        cache_rule or _any_cache(name),
        Rule(f"{name}: block_table must be int32 [rows, pages a row] with a unit last stride",
             lambda a: _table(a.block_table)),
        Rule(f"{name}: lengths must be a contiguous int32 [rows]",
             lambda a: _int32_line(a.lengths, a.block_table.shape[0])),
    ]
    if with_offsets:
        rules.append(Rule(f"{name}: cu_seqlens must be a contiguous int32 [rows + 1]",
                          lambda a: _int32_line(a.cu_seqlens, a.block_table.shape[0] + 1)))
    return rules


def _one_device(name):
    return Rule(f"{name}: all tensors must be CUDA tensors on the cache's device",
                lambda a: a.cache.device.type == "cuda"
                and all(t is None or t.device == a.cache.device for t in a.tensors))


def _pages(cache):
    """A tensor of the cache's memory."""
    return cache._data if _is_cache4(cache) else cache._k


APPEND_RULES = (
    *_rows_rules("append_kv"),
    Rule("append_kv: k and v must be [tokens, kv_heads, 128] of the cache's type, without "
         "gradients", lambda a: _packed(a.k, a.cache, a.cache.kv_heads)
         and _packed(a.v, a.cache, a.cache.kv_heads) and a.k.shape[0] == a.v.shape[0]),
    Rule("append_kv: cos and sin go together, q only with them",
         lambda a: (a.cos is None) == (a.sin is None) and (a.q is None or a.cos is not None)),
    Rule("append_kv: q must be [tokens, q_heads, 128] of the cache's type, without gradients",
         lambda a: a.q is None or (_packed(a.q, a.cache) and a.q.shape[0] == a.k.shape[0]
                                   and a.q.shape[1] > 0)),
    Rule("append_kv: cos and sin must be [tokens, 128], both of the cache's type or both fp32",
         lambda a: a.cos is None or all(
             isinstance(t, torch.Tensor) and t.shape == (a.k.shape[0], HEAD_DIM)
             and t.dtype == a.cos.dtype and t.dtype in (a.cache.dtype, torch.float32)
             for t in (a.cos, a.sin))),
    Rule("append_kv: q / k / v / cos / sin need 16-byte aligned bases, a unit last stride and "
         "strides that are multiples of 16 bytes",
         lambda a: all(t is None or t.shape[0] == 0 or _strided(t)
                       for t in (a.q, a.k, a.v, a.cos, a.sin))),
    _one_device("append_kv"),
)


def append_kv(cache, k, v, block_table, lengths, cu_seqlens, q=None, cos=None, sin=None):
    """Write the new tokens' k and v [T, kv_heads, 128] into their sequences' last rows.

    With ``cos`` / ``sin`` [T, 128] (a token's angles, as the model's rotary embedding gives
    them) k is rotated on its way and ``q`` [T, q_heads, 128] is rotated too: returns the
    rotated q (None without q).  A token whose row the sequence does not hold is skipped.  A 4-bit
    cache takes its codes from the rotated key before any rounding (see ``read_kv``).
    """
    nodes = native.nodes() if _is_cache(cache) or _is_cache4(cache) else None
    if nodes is not None:
        got = nodes.append_kv(cache._pointer, _pages(cache), _is_cache4(cache), k, v, block_table,
                              lengths, cu_seqlens, q, cos, sin)
        if got is not None:
            return got if q is not None else None
    enforce(APPEND_RULES, cache=cache, k=k, v=v, block_table=block_table, lengths=lengths,
            cu_seqlens=cu_seqlens, q=q, cos=cos, sin=sin,
            tensors=(k, v, block_table, lengths, cu_seqlens, q, cos, sin))
    tokens = k.shape[0]
    out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if tokens == 0:
        return out
    device = k.device
    with torch.cuda.device(device):
        _lib.call("ss_kv_append4" if _is_cache4(cache) else "ss_kv_append", cache._pointer, k.data_ptr(), k.stride(0), k.stride(1),
                  v.data_ptr(), v.stride(0), v.stride(1),
                  *((None, 0, 0, 0) if q is None
                    else (q.data_ptr(), q.stride(0), q.stride(1), q.shape[1])),
                  *((None, 0, None, 0, _lib.F32) if cos is None
                    else (cos.data_ptr(), cos.stride(0), sin.data_ptr(), sin.stride(0),
                          _CODES[cos.dtype])),
                  block_table.data_ptr(), _line_stride(block_table), block_table.shape[1],
                  lengths.data_ptr(), cu_seqlens.data_ptr(), block_table.shape[0], tokens,
                  *((None, 0, 0) if out is None
                    else (out.data_ptr(), out.stride(0), out.stride(1))),
                  _lib.stream(device))
    return out


def _weights(t, table, cache):
    return (isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.is_contiguous()
            and t.shape == (table.shape[0], cache.kv_heads, table.shape[1] * cache.page_size))


ATTENTION_RULES = (
    *_rows_rules("cached_attention"),
    Rule("cached_attention: q must be [tokens, q_heads, 128] of the cache's type, without "
         "gradients", lambda a: _packed(a.q, a.cache)),
    Rule("cached_attention: q_heads must be a multiple of the cache's heads",
         lambda a: a.q.shape[1] > 0 and a.q.shape[1] % a.cache.kv_heads == 0),
    Rule("cached_attention: q needs a 16-byte aligned base, a unit last stride and strides that "
         "are multiples of 8", lambda a: a.q.shape[0] == 0 or _strided(a.q)),
    Rule("cached_attention: max_new and max_length must be whole numbers, max_new from 1 up where "
         "there are tokens",
         lambda a: _whole(a.max_new, 1 if a.q.shape[0] else 0) and _whole(a.max_length, 0)
         and a.max_new < 2 ** 31 and a.max_length < 2 ** 31),
    Rule("cached_attention: scale must be a finite number", lambda a: finite_real(a.scale)),
    Rule("cached_attention: window must be None or a whole number from 1 up, sinks one from 0 up",
         lambda a: (a.window is None or _whole(a.window, 1)) and _whole(a.sinks, 0)
         and (a.window or 0) < 2 ** 62 and a.sinks < 2 ** 62),
    Rule("cached_attention: weights and weights_out must be contiguous fp32 [rows, kv_heads, "
         "pages a row * page_size], weights only with weights_out",
         lambda a: all(t is None or _weights(t, a.block_table, a.cache)
                       for t in (a.weights, a.weights_out))
         and (a.weights is None or a.weights_out is not None)),
    Rule("cached_attention: a 4-bit cache gives no weights",
         lambda a: _is_cache(a.cache) or a.weights_out is None),
    _one_device("cached_attention"),
)


def cached_attention(q, cache, block_table, lengths, cu_seqlens, max_new, max_length, scale,
                     window=None, sinks=0, weights=None, weights_out=None):
    """softmax(scale q k^T) v of the new tokens [T, q_heads, 128] over their sequences' rows.

    A token sees the rows up to its own; with ``window`` only the last ``window`` of them and
    the sequence's first ``sinks``.  A token that sees none gives zeros.  ``max_new`` and
    ``max_length`` bound a sequence's new tokens (those behind it give zeros) and its length.

    ``weights_out`` (fp32 [rows, kv_heads, pages a row * page_size]) receives ``weights`` (None:
    zeros; may be the same tensor) plus every cache row's attention weight, summed over the new tokens
    and the q heads of its kv head: what ``evict_kv`` ranks by.  All of the call's tokens count. Drafted
    ones that may yet be refused are better left out: ask for the weights of the accepted ones in
    a call of their own (their queries, ``lengths`` and offsets without the refused).  A 4-bit
    cache gives none.
    """
    nodes = native.nodes() if _is_cache(cache) or _is_cache4(cache) else None
    if nodes is not None:
        got = nodes.cached_attention(cache._pointer, _pages(cache), _is_cache4(cache), q,
                                     block_table, lengths, cu_seqlens, max_new, max_length, scale,
                                     window, sinks, weights, weights_out)
        if got is not None:
            return got
    enforce(ATTENTION_RULES, q=q, cache=cache, block_table=block_table, lengths=lengths,
            cu_seqlens=cu_seqlens, max_new=max_new, max_length=max_length, scale=scale,
            window=window, sinks=sinks, weights=weights, weights_out=weights_out,
            tensors=(q, block_table, lengths, cu_seqlens, weights, weights_out))
    tokens, heads = q.shape[0], q.shape[1]
    device = q.device
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    rows = block_table.shape[0]
    four = _is_cache4(cache)
    size = (_lib.load().ss_cached_attention4_workspace_size(
                rows, tokens, heads, cache.kv_heads, max_new, max_length) if four else
            _lib.load().ss_cached_attention_workspace_size(
                rows, tokens, heads, cache.kv_heads, max_new, max_length, weights_out is not None))
    with torch.cuda.device(device):
        scratch = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        _lib.call("ss_cached_attention4" if four else "ss_cached_attention", cache._pointer,
                  q.data_ptr(), q.stride(0), q.stride(1), heads, block_table.data_ptr(),
                  _line_stride(block_table), block_table.shape[1], lengths.data_ptr(),
                  cu_seqlens.data_ptr(), rows, tokens, max_new, max_length, scale, window or 0,
                  sinks, *(() if four else (_lib.ptr(weights), _lib.ptr(weights_out))),
                  out.data_ptr(), out.stride(0), out.stride(1), _lib.ptr(scratch), size,
                  _lib.stream(device))
    return out


EVICT_RULES = (
    *_rows_rules("evict_kv", with_offsets=False, cache_rule=Rule(
        "evict_kv: cache must be a PagedCache", lambda a: _is_cache(a.cache))),
    Rule("evict_kv: weights must be contiguous fp32 [rows, kv_heads, pages a row * page_size]",
         lambda a: _weights(a.weights, a.block_table, a.cache)),
    Rule("evict_kv: out_table must be int32 [rows, pages a row] with a unit last stride",
         lambda a: _table(a.out_table) and a.out_table.shape[0] == a.block_table.shape[0]),
    Rule("evict_kv: budget must be a whole number from 1 up that out_table's pages hold",
         lambda a: _whole(a.budget, 1)
         and a.budget <= a.out_table.shape[1] * a.cache.page_size),
    Rule("evict_kv: sinks and recent must be whole numbers from 0 up, together within the budget",
         lambda a: _whole(a.sinks, 0) and _whole(a.recent, 0) and a.sinks + a.recent <= a.budget),
    Rule("evict_kv: max_length must be a whole number",
         lambda a: _whole(a.max_length, 0) and a.max_length < 2 ** 31),
    _one_device("evict_kv"),
)


def evict_kv(cache, block_table, lengths, weights, out_table, budget, max_length, sinks=0,
             recent=0):
    """Keep at most ``budget`` rows of every sequence and kv head, copied to other pages.

    Kept are the first ``sinks``, the last ``recent`` and of the others the heaviest by
    ``weights`` (see ``cached_attention``; equal ones from the lowest row up).  They go in their order into the
    pages of ``out_table``, which must not be pages of ``block_table``: the old pages are left as they
    were, so that a shared start serves its other sequences.  Returns the new lengths (int32 [rows]) and weights
    (fp32 [rows, kv_heads, out pages a row * page_size], 0 behind the kept rows).
    """
    nodes = native.nodes() if _is_cache(cache) else None
    if nodes is not None:
        got = nodes.evict_kv(cache._pointer, cache._k, block_table, lengths, weights, out_table,
                             budget, max_length, sinks, recent)
        if got is not None:
            return got
    enforce(EVICT_RULES, cache=cache, block_table=block_table, lengths=lengths, weights=weights,
            out_table=out_table, budget=budget, sinks=sinks, recent=recent, max_length=max_length,
            tensors=(block_table, lengths, weights, out_table))
    rows, heads = block_table.shape[0], cache.k.shape[1]
    device = cache.k.device
    out_lengths = torch.empty(rows, dtype=torch.int32, device=device)
    out_weights = torch.empty((rows, heads, out_table.shape[1] * cache.page_size),
                              dtype=torch.float32, device=device)
    if rows == 0:
        return out_lengths, out_weights
    size = _lib.load().ss_kv_evict_workspace_size(rows, heads, budget)
    with torch.cuda.device(device):
        scratch = torch.empty(size, dtype=torch.uint8, device=device)
        _lib.call("ss_kv_evict", cache._pointer, block_table.data_ptr(),
                  _line_stride(block_table), block_table.shape[1], lengths.data_ptr(), rows,
                  max_length, weights.data_ptr(), out_table.data_ptr(), _line_stride(out_table),
                  out_table.shape[1], budget, sinks, recent, out_lengths.data_ptr(),
                  out_weights.data_ptr(), scratch.data_ptr(), size, _lib.stream(device))
    return out_lengths, out_weights


def _caches(value):
    """The caches of a call as a tuple (one cache, or a list of them), None if they are none."""
    caches = (value,) if _is_cache(value) or _is_cache4(value) else value
    if not isinstance(caches, (list, tuple)) or not caches:
        return None
    first = caches[0]
    kind = _is_cache if _is_cache(first) else _is_cache4
    return tuple(caches) if all(kind(c) for c in caches) else None


def _alike(caches):
    """One shape, strides, type and device: what a launch over all of them takes for granted."""
    def key(c):
        tensors = (c.data,) if _is_cache4(c) else (c.k, c.v)
        return (c.dtype, c.device, *((t.shape, t.stride()) for t in tensors))

    first = key(caches[0])
    return all(key(c) == first for c in caches[1:])


def _caches_rules(name):
    return (
        Rule(f"{name}: caches must be a PagedCache, a PagedCache4, or a list of either",
             lambda a: a.caches is not None),
        Rule(f"{name}: the caches must have one shape, strides, dtype and device",
             lambda a: _alike(a.caches)),
    )


def _pointers(caches):
    return (ctypes.c_void_p * len(caches))(*(c._pointer for c in caches))


READ_RULES = (
    *_caches_rules("read_kv"),
    *_rows_rules("read_kv"),
    Rule("read_kv: tokens must be a whole number", lambda a: _whole(a.tokens, 0)
         and a.tokens < 2 ** 31),
    _one_device("read_kv"),
)


def read_kv(caches, block_table, lengths, cu_seqlens, tokens):
    """k and v [tokens, kv_heads, 128] of the sequences' last rows, as a cache holds them.

    The rows are those that ``append_kv`` writes when it is given the same ``block_table``,
    ``lengths`` and ``cu_seqlens``; offsets as long as the sequences read them whole.  With a
    list of caches (one a layer, alike) both are [caches, tokens, kv_heads, 128].  Rows that a
    sequence does not hold are zeros.
    """
    several = isinstance(caches, (list, tuple))
    nodes = native.nodes()
    if nodes is not None:
        got = nodes.read_kv(caches if several else (caches,), PagedCache, PagedCache4, block_table,
                            lengths, cu_seqlens, tokens, several)
        if got is not None:
            return got
    caches = _caches(caches)
    enforce(READ_RULES, caches=caches, cache=caches and caches[0], block_table=block_table,
            lengths=lengths, cu_seqlens=cu_seqlens, tokens=tokens,
            tensors=(block_table, lengths, cu_seqlens))
    cache = caches[0]
    shape = (len(caches), tokens, cache.kv_heads, HEAD_DIM)
    k, v = (torch.empty(shape, dtype=cache.dtype, device=cache.device) for _ in range(2))
    if tokens:
        with torch.cuda.device(cache.device):
            _lib.call("ss_kv_read4" if _is_cache4(cache) else "ss_kv_read", _pointers(caches),
                      len(caches), block_table.data_ptr(), _line_stride(block_table),
                      block_table.shape[1], lengths.data_ptr(), cu_seqlens.data_ptr(),
                      block_table.shape[0], tokens, k.data_ptr(), v.data_ptr(),
                      _lib.stream(cache.device))
    return (k, v) if several else (k[0], v[0])


FORK_RULES = (
    *_caches_rules("fork_kv"),
    *_rows_rules("fork_kv", with_offsets=False),
    Rule("fork_kv: parents and spare must be contiguous int32 [new rows]",
         lambda a: isinstance(a.parents, torch.Tensor) and a.parents.ndim == 1
         and all(_int32_line(t, a.parents.shape[0]) for t in (a.parents, a.spare))),
    _one_device("fork_kv"),
)


def fork_kv(caches, block_table, lengths, parents, spare):
    """Sequences that continue others: (block table, lengths) with a row for each of ``parents``.

    Row i continues row ``parents[i]`` (int32 [new rows]; any number of rows may continue
    one, and a parent that is no row counts as an empty sequence): it shares the parent's full
    pages, and page ``spare[i]`` becomes the one that its next tokens go to, with the
    rows that the parent has beyond its full pages copied there in every cache of the list (one a
    layer, alike).  The entries behind are -1.  Spare pages must be nobody's: not in
    ``block_table`` and not named twice.  The parents' own last pages are free again once no
    row of ``block_table`` is used further, unless they are full.
    """
    nodes = native.nodes()
    if nodes is not None:
        got = nodes.fork_kv(caches if isinstance(caches, (list, tuple)) else (caches,), PagedCache,
                            PagedCache4, block_table, lengths, parents, spare)
        if got is not None:
            return got
    caches = _caches(caches)
    enforce(FORK_RULES, caches=caches, cache=caches and caches[0], block_table=block_table,
            lengths=lengths, parents=parents, spare=spare,
            tensors=(block_table, lengths, parents, spare))
    cache, rows = caches[0], parents.shape[0]
    out_table = torch.empty((rows, block_table.shape[1]), dtype=torch.int32, device=cache.device)
    out_lengths = torch.empty(rows, dtype=torch.int32, device=cache.device)
    if rows:
        with torch.cuda.device(cache.device):
            _lib.call("ss_kv_fork4" if _is_cache4(cache) else "ss_kv_fork", _pointers(caches),
                      len(caches), block_table.data_ptr(), _line_stride(block_table),
                      block_table.shape[1], lengths.data_ptr(), block_table.shape[0],
                      parents.data_ptr(), spare.data_ptr(), rows, out_table.data_ptr(),
                      out_lengths.data_ptr(), _lib.stream(cache.device))
    return out_table, out_lengths
