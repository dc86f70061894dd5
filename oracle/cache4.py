"""The 4-bit paged cache, forks and beam selection -- test infrastructure only.

Restated in float64 numpy from the definitions in include/soupsuck_amd.h (the reference trains
only and has no counterpart).

Pins (tests/test_oracle_cache4.py): every value that a block can hold is kept; what is held is the
nearest of them; bytes against single values set by hand; forks against lists; selection
against a sort of all candidates.
"""

import math

import numpy as np

STEPS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
EXPONENTS = {"float16": (-13, 13), "bfloat16": (-125, 125)}


def encode(x, dtype):
    """(codes 0 .. 15 [..., 128], scale bytes [..., 4]) of x [..., 128] for a cache of `dtype`."""
    low, high = EXPONENTS[dtype]
    x = np.asarray(x, np.float64).reshape(*np.shape(x)[:-1], 4, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max(-1)
    finite = np.isfinite(x).all(-1)
    top = np.where(finite, top, 0.0)
    part, power = np.frexp(top)                       # top = part 2^power, part in [0.5, 1)
    e = np.where(part > 0.75, power - 2, power - 3)   # 6 2^e = 0.75 2^(e + 3)
    e = np.clip(np.where(top == 0, low, e), low, high)
    y = np.where(finite[..., None], x, 0.0) / np.exp2(e)[..., None]
    size = np.minimum(np.abs(y), 6.0)
    middles = (STEPS[1:] + STEPS[:-1]) / 2
    code = np.searchsorted(middles, size, side="left")          # at a middle: the lower one
    tie = (code < 7) & (size == middles[np.minimum(code, 6)]) & (code % 2 == 1)
    code = np.where(tie, code + 1, code) + 8 * (y < 0)
    return code.reshape(*x.shape[:-2], 128), np.where(finite, e + 127, 255)


def decode(codes, scales):
    """The values of codes [..., 128] and scale bytes [..., 4]; NaN for a byte of 255."""
    codes = np.asarray(codes).reshape(*np.shape(codes)[:-1], 4, 32)
    scales = np.asarray(scales, np.float64)
    size = np.where(scales == 255, np.nan, np.exp2(np.where(scales == 255, 0, scales) - 127))
    value = STEPS[codes % 8] * np.where(codes >= 8, -1.0, 1.0) * size[..., None]
    return value.reshape(*codes.shape[:-2], 128)


def held(x, dtype):
    return decode(*encode(x, dtype))


def places(row, dim):
    """(byte of the key's code, of the value's, of the key's scale, of the value's, shift of the
    code in its byte) of one value in its group's 2176 bytes."""
    block = dim // 32
    return (block * 256 + row * 16 + dim % 32 // 2,
            1024 + row // 4 * 256 + dim // 8 * 16 + row % 4 * 4 + dim % 8 // 2,
            2048 + block * 16 + row, 2112 + block * 16 + row, dim % 2 * 4)


_ROW, _DIM = np.divmod(np.arange(16 * 128), 128)
_PLACES = [np.array(p).reshape(16, 128) for p in
           zip(*(places(r, d) for r, d in zip(_ROW.tolist(), _DIM.tolist())))]


def unpack(data):
    """(k, v) [pages, heads, page size, 128] of the bytes [pages, heads, groups, 2176]."""
    data = np.asarray(data)
    pages, heads, groups, _ = data.shape
    out = []
    for code, scale in ((0, 2), (1, 3)):
        codes = data[..., _PLACES[code]] >> _PLACES[4] & 15
        scales = data[..., _PLACES[scale][:, ::32]]
        out.append(decode(codes, scales).reshape(pages, heads, groups * 16, 128))
    return out


def pack(data, page, head, row, k, v, dtype):
    """Writes one row's k and v [128] into the bytes."""
    group = data[page, head, row // 16]
    for x, code_at, scale_at in ((k, 0, 2), (v, 1, 3)):
        codes, scales = encode(x, dtype)
        for dim in range(128):
            at, shift = _PLACES[code_at][row % 16, dim], _PLACES[4][row % 16, dim]
            group[at] = (int(group[at]) & ~(15 << shift) & 255) | int(codes[dim]) << shift
        group[_PLACES[scale_at][row % 16, ::32]] = scales


def fork(table, lengths, parents, spare, page_size, pages):
    """(new table, new lengths, copies): copies are (from page, to page, rows)."""
    width = len(table[0])
    new, sizes, copies = [], [], []
    for parent, free in zip(parents, spare):
        known = 0 <= parent < len(table)
        n = max(0, min(int(lengths[parent]), width * page_size)) if known else 0
        full, rest = divmod(n, page_size)
        line = list(table[parent][:full]) if known else []
        if full < width:
            source = int(table[parent][full]) if rest else -1
            usable = 0 <= source < pages
            if rest and usable and 0 <= free < pages:
                copies.append((source, int(free), rest))
            line.append(-1 if rest and not usable else int(free))
        new.append((line + [-1] * width)[:width])
        sizes.append(n)
    return np.array(new, np.int32).reshape(-1, width), np.array(sizes, np.int32), copies


def select(logits, scores, count):
    """(scores, parents, tokens) of one sequence: logits [beams, vocab], scores [beams]."""
    x = np.array(logits, np.float64)
    beams, vocab = x.shape
    entries = []
    for b in range(beams):
        line = x[b]
        if np.isnan(line).any() or (line == np.inf).any() or (line == -np.inf).all():
            whole = math.nan
        else:
            whole = line.max() + math.log(np.exp(line - line.max()).sum())
        for token in range(vocab):
            v = line[token] - whole + float(scores[b])
            v = -math.inf if math.isnan(v) else v
            own = -math.inf if math.isnan(line[token]) else line[token]
            entries.append((-v, b, -own, token))
    entries.sort()
    best = entries[:count]
    return (np.array([-e[0] for e in best]), np.array([e[1] for e in best], np.int32),
            np.array([e[3] for e in best], np.int64))
