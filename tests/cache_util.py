"""Paged caches for the tests: pages in random order, poisoned where no sequence has a row."""

from types import SimpleNamespace

import torch

DIM = 128
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def host(t):
    return t.detach().double().cpu().numpy()


def build(lengths, heads, page, dtype, device, seed, spare=3, layout="head", extra_pages=0,
          poison=float("nan"), scale=1.0):
    """A cache whose sequences hold random rows; everything else is ``poison``.

    layout "head": [pages, heads, page, 128]; "row": pages of rows of all heads, with a gap
    between rows, seen through strides.  Table lines are ``extra_pages`` longer than any
    sequence needs; those entries are -1.
    """
    gen = torch.Generator().manual_seed(seed)
    need = [max(0, -(-n // page)) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen).tolist()
    width = max(max(need, default=0) + extra_pages, 1)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    tensors = []
    for _ in range(2):
        if layout == "head":
            t = torch.full((total, heads, page, DIM), poison, dtype=dtype)
        else:
            t = torch.full((total, page, heads + 1, DIM + 8), poison, dtype=dtype)
            t = t[:, :, :heads, :DIM].transpose(1, 2)
        tensors.append(t)
    start = 0
    for b, n in enumerate(lengths):
        mine = order[start:start + need[b]]
        start += need[b]
        table[b, :need[b]] = torch.tensor(mine, dtype=torch.int32)
        for t in tensors:
            rows = (torch.randn((max(n, 0), heads, DIM), generator=gen) * scale).to(dtype)
            for i, p in enumerate(mine):
                part = rows[i * page:(i + 1) * page]
                t[p, :, :part.shape[0]] = part.transpose(0, 1)
    free = order[start:]

    def place(t):
        if layout == "head":
            return t.to(device)
        base = t.transpose(1, 2)._base.to(device)
        return base[:, :, :heads, :DIM].transpose(1, 2)

    return SimpleNamespace(k=place(tensors[0]), v=place(tensors[1]), table=table.to(device),
                           lengths=torch.tensor(lengths, dtype=torch.int32, device=device),
                           free=free, page=page)


def offsets(new, device):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=device)


def attention_bound(dtype, reference, spread, reach, rows):
    """Elementwise bound on the kernel's output against 64 bits.

    One rounding of the output; probabilities rounded to 16 bits before the product with the
    values and again in their sum (2 half steps of the values' spread); scores summed over 128
    products in fp32 (a relative 128 half steps of their reach), exponentials of 2 half steps
    and sums over ``rows`` keys in fp32, all twice (numerator and sum).
    """
    step = HALF_STEP[dtype]
    score = 2 * 2.0 ** -24 * (128 * reach + 4 * (1 + reach) + rows)
    return step * abs(reference) + spread * (2 * step + score) + 1e-7
