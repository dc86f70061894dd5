"""4-bit caches for the tests: pages in random order, NaN where no sequence has a row."""

from types import SimpleNamespace

import numpy as np
import torch

from oracle import cache4
from tests.cache_util import DIM

NAMES = {torch.float16: "float16", torch.bfloat16: "bfloat16"}


def random_bytes(shape, seed, spread=2):
    """Bytes of random codes with scales around 1 ([pages, heads, groups, 2176])."""
    rng = np.random.default_rng(seed)
    data = rng.integers(0, 256, shape, dtype=np.uint8)
    data[..., 2048:] = rng.integers(126 - spread, 127, (*shape[:-1], 128))
    return data


def build4(lengths, heads, page, device, seed, spare=3, extra_pages=0, layout="plain", spread=2):
    """A cache whose sequences hold random rows; every other row is NaN (scale bytes of 255).

    layout "gaps": the groups lie apart, between bytes that are NaN too.
    """
    gen = torch.Generator().manual_seed(seed)
    need = [max(0, -(-n // page)) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen).tolist()
    width = max(max(need, default=0) + extra_pages, 1)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    data = random_bytes((total, heads, page // 16, 2176), seed, spread)
    known = np.zeros((total, page), bool)
    start = 0
    for b, n in enumerate(lengths):
        mine = order[start:start + need[b]]
        start += need[b]
        table[b, :need[b]] = torch.tensor(mine, dtype=torch.int32)
        for i, p in enumerate(mine):
            known[p, :max(0, min(page, n - i * page))] = True
    scales = data[..., 2048:].reshape(total, heads, page // 16, 2, 4, 16)
    scales[np.broadcast_to(~known.reshape(total, 1, page // 16, 1, 1, 16), scales.shape)] = 255
    data[..., 2048:] = scales.reshape(total, heads, page // 16, 128)
    there = torch.from_numpy(data)
    if layout == "gaps":
        wide = torch.full((total, heads + 1, page // 16, 2176 + 48), 255, dtype=torch.uint8,
                          device=device)
        view = wide[:, :heads, :, 16:16 + 2176]
        view.copy_(there)
        there = view
    else:
        there = there.to(device)
    return SimpleNamespace(data=there, table=table.to(device), page=page, free=order[start:],
                           lengths=torch.tensor(lengths, dtype=torch.int32, device=device))


def values(data):
    """(k, v) [pages, heads, page size, 128] in 64 bits."""
    return cache4.unpack(data.cpu().numpy())


def tokens(count, heads, dtype, device, seed, strided=False, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((count, heads, DIM), generator=gen) * scale).to(dtype)
    if not strided:
        return x.to(device)
    wide = torch.full((count, heads + 2, DIM + 16), float("nan"), dtype=dtype, device=device)
    view = wide[:, 1:1 + heads, 8:8 + DIM]
    view.copy_(x)
    return view
