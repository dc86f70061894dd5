"""The serving calls' native bodies against their Python bodies: same kernels, same results,
same refusals.  Any timing hook selects the Python bodies."""

import contextlib

import pytest
import torch

from soupsuck_amd import _lib
from soupsuck_amd.kernels.paged import PagedCache, append_kv, cached_attention, evict_kv
from soupsuck_amd.kernels.verify import verify_drafts
from tests.cache_util import DIM, build, offsets

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@contextlib.contextmanager
def python_bodies():
    _lib.hooks["none"] = None
    try:
        yield
    finally:
        del _lib.hooks["none"]


def _same(a, b):
    a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride()
        assert torch.equal(x, y)


def _randn(*shape, dtype, device, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("angles", [None, torch.float32, "cache"])
def test_append(device, dtype, angles):
    c = build([40, 9], 2, 16, dtype, device, seed=1, poison=0.0)
    other = c.k.clone(), c.v.clone()
    cu = offsets([5, 9], device)
    k, v = (_randn(14, 2, DIM, dtype=dtype, device=device, seed=s) for s in (2, 3))
    q = cos = sin = None
    if angles is not None:
        kind = dtype if angles == "cache" else angles
        q = _randn(14, 6, DIM, dtype=dtype, device=device, seed=4)
        cos, sin = (_randn(14, DIM, dtype=kind, device=device, seed=s) for s in (5, 6))
    got = append_kv(PagedCache(c.k, c.v), k, v, c.table, c.lengths, cu, q=q, cos=cos, sin=sin)
    with python_bodies():
        want = append_kv(PagedCache(*other), k, v, c.table, c.lengths, cu, q=q, cos=cos, sin=sin)
    if q is None:
        assert got is None and want is None
    else:
        _same(got, want)
    _same((c.k, c.v), other)


@pytest.mark.parametrize("window,sinks,weighed", [(None, 0, False), (50, 3, True)])
def test_attention_and_eviction(device, window, sinks, weighed):
    c = build([1500, 90, 300], 2, 16, F16, device, seed=2, spare=12)
    cache, cu = PagedCache(c.k, c.v), offsets([2, 1, 2], device)
    q = _randn(5, 6, DIM, dtype=F16, device=device, seed=3)
    sums = [torch.zeros((3, 2, c.table.shape[1] * 16), device=device) for _ in range(2)] \
        if weighed else [None, None]
    args = (q, cache, c.table, c.lengths, cu, 2, 1500, 0.1)
    got = cached_attention(*args, window=window, sinks=sinks, weights_out=sums[0])
    with python_bodies():
        want = cached_attention(*args, window=window, sinks=sinks, weights_out=sums[1])
    _same(got, want)
    if weighed:
        _same(*sums)
        to = torch.tensor(c.free[:12], dtype=torch.int32, device=device).view(3, 4)
        args = (cache, c.table, c.lengths, sums[0], to, 60, 1500)
        got = evict_kv(*args, sinks=2, recent=20)
        with python_bodies():
            want = evict_kv(*args, sinks=2, recent=20)
        _same(got, want)


@pytest.mark.parametrize("looked_up", [False, True])
def test_verify(device, looked_up):
    target = _randn(3, 5, 999, dtype=F16, device=device, seed=1)
    draft = None if looked_up else _randn(3, 4, 999, dtype=F16, device=device, seed=2)
    tokens = torch.arange(12, device=device).view(3, 4)
    uniform = torch.rand((3, 5), generator=torch.Generator().manual_seed(3)).to(device)
    counts = torch.tensor([4, 0, 2], dtype=torch.int32, device=device)
    got = verify_drafts(target, tokens, uniform, draft, counts, 0.8)
    with python_bodies():
        want = verify_drafts(target, tokens, uniform, draft, counts, 0.8)
    _same(got, want)
    _same(verify_drafts(target, tokens, temperature=0), verify_drafts(target, tokens, uniform,
                                                                     temperature=0.0))


def test_refusals_reach_the_rules(device):
    """What the native bodies are not sure of goes through the rules."""
    c = build([40], 2, 16, F16, device, seed=1)
    cache, cu = PagedCache(c.k, c.v), offsets([1], device)
    q = _randn(1, 4, DIM, dtype=F16, device=device, seed=2)
    for change, text in ((dict(q=q.float()), "q must be"), (dict(q=q.cpu()), "one device|device"),
                         (dict(q=q[..., ::2]), "q must be"), (dict(max_new=True), "max_new"),
                         (dict(scale=float("nan")), "scale"), (dict(window=0), "window"),
                         (dict(lengths=c.lengths.long()), "lengths"), (dict(q=None), "q must be"),
                         (dict(cu_seqlens=cu[:1]), "cu_seqlens"),
                         (dict(weights=torch.zeros(1, device=device)), "weights")):
        args = dict(q=q, cache=cache, block_table=c.table, lengths=c.lengths, cu_seqlens=cu,
                    max_new=1, max_length=40, scale=0.1)
        with pytest.raises(ValueError, match=text):
            cached_attention(**{**args, **change})
    assert cached_attention(q[:0], cache, c.table, c.lengths, offsets([0], device), 1, 40,
                            0.1).shape == (0, 4, DIM)
