"""Answering with a 4-bit cache and with beams: the operators, and their plain forms.

Kinds of case:

  append4    new tokens' keys (rotated) and values into the pages of a 4-bit cache, the queries
             rotated by the same call, and the new rows read back as the cache holds them
  attention4 new tokens over a 4-bit paged cache, with a sliding window and first tokens that
             stay visible where the case has them
  select     the best continuations of each sequence's beams from logits and running scores
  fork       beams continue the beams they were chosen from: block tables follow, and the rows
             of each layer's last, partly filled page are copied

A row of a 4-bit cache has 128 keys and 128 values of one head, in blocks of 32 that share a scale 2^e:
codes are 1 sign, 2 exponent and 1 mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6), e is the least with which none is
past 6, from -13 to 13 for fp16 and from -125 to 125 for bf16.  Head layouts are those of Qwen2.5
1.5B (12 / 2) and 7B (28 / 4) and generic ones, the vocabulary is theirs; sequences are ragged.
listed() names the cases, draw() gives more of the same ranges, prepare() makes what a
program has in hand, run() is one pass (the framework's calls where ``own`` is true, plain torch
in 32 or 64 bits elsewhere), work() the bytes and flops a pass cannot do without and exact()
the result in 64 bits.
"""

import math
from types import SimpleNamespace

import torch

own = False

HEAD_DIM = 128
BLOCK = 32                           # values of a scale
GROUP_BYTES = 2176                   # of 16 rows: key codes, value codes, key scales, value scales
VOCAB = 151936
HEADS = ((12, 2), (28, 4), (8, 8), (24, 8))
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EXPONENTS = {torch.float16: (-13, 13), torch.bfloat16: (-125, 125)}
SCALE = HEAD_DIM ** -0.5


# ----------------------------------------------------------------- the cases

def listed():
    return [
        # one sequence's next token: the append between two products of a decode step
        {"name": "append4_one", "kind": "append4", "dtype": "fp16", "heads": 12, "kv_heads": 2,
         "page": 64, "new": "1", "past": "517", "angles": "fp16"},
        # prompts of several sequences entering the cache together, some after a shared start
        {"name": "append4_prompts", "kind": "append4", "dtype": "bf16", "heads": 28,
         "kv_heads": 4, "page": 16, "new": "2048,1537,1201,777,350,128,1",
         "past": "0,64,0,333,0,0,5000", "angles": "fp32"},
        # interactive: one short conversation, one token; latency is all
        {"name": "attention4_one_short", "kind": "attention4", "dtype": "fp16", "heads": 12,
         "kv_heads": 2, "page": 64, "new": "1", "lengths": "518", "window": 0, "sinks": 0},
        # one very long document, one token: the cache's length is all the parallelism
        {"name": "attention4_one_long", "kind": "attention4", "dtype": "fp16", "heads": 28,
         "kv_heads": 4, "page": 64, "new": "1", "lengths": "131071", "window": 0, "sinks": 0},
        # a large serving batch of ragged conversations, one token each: what the bytes allow
        {"name": "attention4_batch", "kind": "attention4", "dtype": "bf16", "heads": 28,
         "kv_heads": 4, "page": 64, "new": "1",
         "lengths": ",".join(str(8191 - 37 * i) for i in range(64)), "window": 0, "sinks": 0},
        # long streams kept to a window and their first tokens, drafted tokens verified at once
        {"name": "attention4_window", "kind": "attention4", "dtype": "bf16", "heads": 24,
         "kv_heads": 8, "page": 32, "new": "5",
         "lengths": ",".join(["16111,9001,30003,20011"] * 2), "window": 4096, "sinks": 4},
        # pieces of long prompts, each after what the cache has of its sequence already
        {"name": "attention4_piece", "kind": "attention4", "dtype": "bf16", "heads": 28,
         "kv_heads": 4, "page": 16, "new": "64", "lengths": "4099,3801,6007,1201", "window": 0,
         "sinks": 0},
        # one conversation's four beams
        {"name": "select_one", "kind": "select", "dtype": "fp16", "batch": 1, "beams": 4,
         "count": 8, "vocab": VOCAB, "banned": 0, "first": False},
        # a serving batch's beams, the largest call
        {"name": "select_batch", "kind": "select", "dtype": "bf16", "batch": 64, "beams": 8,
         "count": 16, "vocab": VOCAB, "banned": 64, "first": False},
        # the first step, with one living beam of each, over an odd vocabulary
        {"name": "select_first", "kind": "select", "dtype": "fp32", "batch": 8, "beams": 5,
         "count": 10, "vocab": 32003, "banned": 7, "first": True},
        # every layer's cache after a step of one conversation's beams
        {"name": "fork_one", "kind": "fork", "cache": "16bit", "dtype": "fp16", "kv_heads": 2,
         "page": 64, "beams": 4, "layers": 28, "lengths": "517"},
        # the same for a batch over a 4-bit cache, one text at a page's end; rows read back as held
        {"name": "fork_batch", "kind": "fork", "cache": "4bit", "dtype": "bf16", "kv_heads": 4,
         "page": 64, "beams": 8, "layers": 28, "lengths": "811,1343,256,1087"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], uniform over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _text(values):
    return ",".join(str(int(v)) for v in values)


def draw(rng):
    kind = rng.choice(("append4", "attention4", "attention4", "attention4", "select", "select",
                       "fork"))
    dtype = rng.choice(("fp16", "bf16"))
    heads, kv_heads = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128))
    if kind == "append4":
        total, new = _spread(rng, 1, 6000), []
        while sum(new) < total:
            new.append(min(_spread(rng, 1, 2048), total - sum(new)))
        return {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "page": page,
                "new": _text(new),
                "past": _text(rng.choice((0, _spread(rng, 1, 8000))) for _ in new),
                "angles": rng.choice((dtype, "fp32"))}
    if kind == "attention4":
        new = rng.choice((1, 1, 1, 2, 5, 8, 33))     # one token, drafts, a piece of a prompt
        keys = _spread(rng, 1, 1600000 // (kv_heads * new))          # of the whole batch
        batch = _spread(rng, max(1, keys // 100000), max(1, min(64, keys // 8)))
        mean = max(1, keys // batch)
        lengths = [max(new, _spread(rng, max(1, mean // 4), min(131071, max(1, mean * 3 // 2))))
                   for _ in range(batch)]
        return {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "page": page,
                "new": str(new), "lengths": _text(lengths),
                "window": rng.choice((0, 0, _spread(rng, 16, 8192))),
                "sinks": rng.choice((0, 4, 16))}
    if kind == "select":
        dtype = rng.choice(("fp16", "bf16", "fp32"))
        vocab = rng.choice((VOCAB, VOCAB, _spread(rng, 1000, VOCAB)))
        beams = rng.choice((2, 3, 4, 5, 8, 16))
        most = 64 * 8 * VOCAB * 2 // (beams * vocab * (4 if dtype == "fp32" else 2))
        return {"kind": kind, "dtype": dtype, "batch": _spread(rng, 1, min(64, most)),
                "beams": beams, "count": rng.choice((beams, 2 * beams)), "vocab": vocab,
                "banned": rng.choice((0, _spread(rng, 1, 500))), "first": rng.random() < 0.2}
    beams = rng.choice((2, 4, 5, 8))
    return {"kind": kind, "cache": rng.choice(("4bit", "16bit")), "dtype": dtype,
            "kv_heads": rng.choice((2, 4)), "page": page, "beams": beams,
            "layers": _spread(rng, 2, 28),
            "lengths": _text(_spread(rng, 1, 1400) for _ in range(rng.randint(1, 4)))}


# ------------------------------------------------------------- what is in hand

def _numbers(text):
    return [int(v) for v in text.split(",")]


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _generator(seed):
    return torch.Generator(device=_device()).manual_seed(int(seed))


def _normal(gen, shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device=gen.device).mul_(std).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=_device())


def _offsets(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _pages(gen, lengths, page):
    """(pages in all, block table [rows, most pages] int32): pages handed out in random order."""
    need = [max(1, -(-n // page)) for n in lengths]
    total = sum(need)
    order = torch.randperm(total, generator=gen, device=gen.device).to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device=gen.device)
    start = 0
    for row, n in enumerate(need):
        table[row, :n] = order[start:start + n]
        start += n
    return total, table


def _encode(x, dtype):
    """(codes, scale bytes) uint8 of x [..., 128], codes [..., 4, 32] and scales [..., 4]."""
    x = x.reshape(*x.shape[:-1], HEAD_DIM // BLOCK, BLOCK)
    part, power = torch.frexp(x.abs().amax(-1))
    low, high = EXPONENTS[dtype]
    e = torch.where(part <= 0.75, power - 3, power - 2)          # 6 * 2^e = 0.75 * 2^(e + 3)
    e = torch.where(part == 0, low, e).clamp_(low, high)
    y = torch.ldexp(x, -e[..., None])
    size = y.abs()
    code = torch.zeros_like(size, dtype=torch.uint8)
    for border, even in ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True),
                         (3.5, False), (5.0, True)):             # a tie goes to the even code
        code += size > border if even else size >= border
    code += (y < 0).to(torch.uint8) * 8
    return code, (e + 127).to(torch.uint8)


def _grouped(codes_k, scales_k, codes_v, scales_v):
    """The bytes [..., rows / 16, 2176] of rows' codes [..., rows, 4, 32] and scales [..., rows, 4]."""
    lead = codes_k.shape[:-3]
    rows = codes_k.shape[-3]

    def halves(codes):
        return codes[..., 0::2] | (codes[..., 1::2] << 4)        # [..., rows, 4, 16]

    n = len(lead)
    k = halves(codes_k).reshape(*lead, rows // 16, 16, 4, 16)
    k = k.transpose(n + 1, n + 2)                                # block, row, byte
    v = halves(codes_v).reshape(*lead, rows // 16, 4, 4, 16, 4)
    v = v.transpose(n + 2, n + 3)                                # row quad, chunk, row, byte
    parts = [k, v] + [s.reshape(*lead, rows // 16, 16, 4).transpose(n + 1, n + 2)
                      for s in (scales_k, scales_v)]
    return torch.cat([p.reshape(*lead, rows // 16, -1) for p in parts], -1)


def _cache4(data, dtype):
    if not own:
        return SimpleNamespace(data=data, dtype=dtype)
    from soupsuck_amd.kernels.paged import PagedCache4
    return PagedCache4(data, dtype)


def _cache16(k, v):
    if not own:
        return SimpleNamespace(k=k, v=v)
    from soupsuck_amd.kernels.paged import PagedCache
    return PagedCache(k, v)


def _full_cache4(gen, pages, hk, page, dtype, first=None, common=None):
    """A 4-bit cache whose pages all hold rows; the pages ``first`` begin with a heavy key."""
    data = torch.empty((pages, hk, page // 16, GROUP_BYTES), dtype=torch.uint8, device=gen.device)
    step = max(1, (1 << 23) // (hk * page * HEAD_DIM))
    # Keys have a few wide channels, as those behind a rotation have.
    wide = 1.0 + 4.0 * (torch.rand(HEAD_DIM, generator=gen, device=gen.device) < 0.06)
    heavy = None
    if first is not None:
        heavy = torch.zeros(pages, dtype=torch.bool, device=gen.device)
        heavy[first] = True
    for at in range(0, pages, step):
        n = min(step, pages - at)
        shape = (n, hk, page, HEAD_DIM)
        k = torch.randn(shape, generator=gen, device=gen.device) * wide
        if heavy is not None:
            k[:, :, 0] = torch.where(heavy[at:at + n, None, None], common[:, 0] * 0.6, k[:, :, 0])
        v = torch.randn(shape, generator=gen, device=gen.device)
        data[at:at + n] = _grouped(*_encode(k, dtype), *_encode(v, dtype))
    return data


def prepare(case, seed):
    gen = _generator(seed)
    s = SimpleNamespace(case=case)
    s.dtype = DTYPES[case["dtype"]]
    return {"append4": _prepare_append, "attention4": _prepare_attention,
            "select": _prepare_select, "fork": _prepare_fork}[case["kind"]](case, gen, s)


def _prepare_append(case, gen, s):
    page, hk, dtype = case["page"], case["kv_heads"], s.dtype
    s.new, past = _numbers(case["new"]), _numbers(case["past"])
    s.lens = [a + b for a, b in zip(s.new, past)]
    pages, s.table = _pages(gen, s.lens, page)
    s.total = sum(s.new)
    s.cache = _cache4(torch.zeros((pages, hk, page // 16, GROUP_BYTES), dtype=torch.uint8,
                                  device=gen.device), dtype)
    # The fused projection's rows: q, k and v of a token lie side by side.
    qkv = _normal(gen, (s.total, case["heads"] + 2 * hk, HEAD_DIM), dtype)
    s.q, s.k, s.v = qkv.split((case["heads"], hk, hk), dim=1)
    position = torch.cat([torch.arange(b, a + b) for a, b in zip(s.new, past)]).double()
    inverse = 1e6 ** (-torch.arange(0, HEAD_DIM, 2).double() / HEAD_DIM)
    angle = (position[:, None] * inverse).repeat(1, 2)
    s.cos, s.sin = (f(angle).to(DTYPES[case["angles"]]).to(gen.device)
                    for f in (torch.cos, torch.sin))
    s.lengths, s.cu = _int32(s.lens), _int32(_offsets(s.new))
    s.position = position.long().to(gen.device)
    s.row = torch.repeat_interleave(torch.arange(len(s.new)), torch.tensor(s.new)).to(gen.device)
    return s


def _prepare_attention(case, gen, s):
    page, hk, dtype = case["page"], case["kv_heads"], s.dtype
    s.lens = _numbers(case["lengths"])
    batch = len(s.lens)
    pages, s.table = _pages(gen, s.lens, page)
    s.new = [int(case["new"])] * batch
    # Keys and queries with a direction in common, which the first key holds strongly (the
    # sink of trained models), over noise that leaves a few heavy keys.
    common = torch.randn((hk, 1, HEAD_DIM), generator=gen, device=gen.device)
    s.cache = _cache4(_full_cache4(gen, pages, hk, page, dtype, s.table[:, 0].long(), common),
                      dtype)
    q = torch.randn((sum(s.new), hk, case["heads"] // hk, HEAD_DIM), generator=gen,
                    device=gen.device) + common
    s.q = q.to(dtype).view(sum(s.new), case["heads"], HEAD_DIM)
    s.lengths, s.cu, s.max_new = _int32(s.lens), _int32(_offsets(s.new)), max(s.new)
    s.max_length = max(s.lens)
    return s


def _prepare_select(case, gen, s):
    batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
    s.logits = _normal(gen, (batch, beams, vocab), s.dtype, 2.5)
    if case["banned"]:
        # tokens that the program rules out, the same ones for every beam
        ruled = torch.randperm(vocab, generator=gen, device=gen.device)[:case["banned"]]
        s.logits[..., ruled] = -math.inf
    s.scores = -8.0 * torch.rand((batch, beams), generator=gen, device=gen.device) - 1.0
    s.scores = s.scores.sort(-1, descending=True).values
    if case["first"]:
        s.scores[:, 0] = 0.0
        s.scores[:, 1:] = -math.inf
    return s


def _prepare_fork(case, gen, s):
    page, hk, beams, layers = case["page"], case["kv_heads"], case["beams"], case["layers"]
    s.lens = [n for n in _numbers(case["lengths"]) for _ in range(beams)]
    rows = len(s.lens)
    width = max(s.lens) // page + 1
    # A sequence's beams share the pages of most of its text and have the others for themselves.
    lines, pages = [], 0
    for row, n in enumerate(s.lens):
        line = lines[row - row % beams][:n * 7 // 10 // page] if row % beams else []
        mine = -(-n // page) - len(line)
        lines.append(line + list(range(pages, pages + mine)))
        pages += mine
    total = pages + rows
    order = torch.randperm(total, generator=gen, device=gen.device).to(torch.int32)
    index = torch.tensor([line + [total] * (width - len(line)) for line in lines],
                         device=gen.device)
    s.table = torch.cat((order, _int32([-1])))[index]
    s.spare = order[pages:].clone()
    chosen = torch.randint(0, beams, (rows,), generator=gen, device=gen.device)
    s.parents = (torch.arange(rows, device=gen.device) // beams * beams + chosen).to(torch.int32)
    s.lengths = _int32(s.lens)
    s.open = [n % page for n in s.lens]              # rows of the last page, as parents have them
    s.cu, s.total = _int32(_offsets(s.open)), sum(s.open)
    if case["cache"] == "4bit":
        s.caches = [_cache4(_full_cache4(gen, total, hk, page, s.dtype), s.dtype)
                    for _ in range(layers)]
    else:
        s.caches = [_cache16(*(_normal(gen, (total, hk, page, HEAD_DIM), s.dtype)
                               for _ in range(2))) for _ in range(layers)]
    return s


# ------------------------------------------------------------------- one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    case = s.case
    if case["kind"] == "select":
        from soupsuck_amd.kernels.beams import select_beams
        return select_beams(s.logits, s.scores, case["count"])
    from soupsuck_amd.kernels.paged import append_kv, cached_attention, fork_kv, read_kv
    if case["kind"] == "append4":
        q = append_kv(s.cache, s.k, s.v, s.table, s.lengths, s.cu, q=s.q, cos=s.cos, sin=s.sin)
        return (q, *read_kv(s.cache, s.table, s.lengths, s.cu, s.total))
    if case["kind"] == "attention4":
        return cached_attention(s.q, s.cache, s.table, s.lengths, s.cu, s.max_new, s.max_length,
                                scale=SCALE, window=case["window"] or None, sinks=case["sinks"])
    table, lengths = fork_kv(s.caches, s.table, s.lengths, s.parents, s.spare)
    if case["cache"] == "16bit":
        return (table, lengths, *(t for c in s.caches for t in (c.k, c.v)))
    return (table, lengths, *read_kv(s.caches, table, lengths, s.cu, s.total))


def _run_plain(s):
    return {"append4": _plain_append, "attention4": _plain_attention, "select": _plain_select,
            "fork": _plain_fork}[s.case["kind"]](s)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    low, high = x[..., :half], x[..., half:]
    return torch.cat((low * cos[..., :half] - high * sin[..., :half],
                      high * cos[..., half:] + low * sin[..., half:]), -1)


def _steps(device):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0,
                         -3.0, -4.0, -6.0], device=device)


def _decode(codes, scales):
    """fp32 [..., 128] of codes [..., 4, 32] and scale bytes [..., 4]."""
    size = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    return (_steps(codes.device)[codes.long()] * size[..., None]).flatten(-2)


def _ungrouped(data):
    """Keys' and values' codes [..., rows, 4, 32] and scales [..., rows, 4] of grouped bytes."""
    lead, n = data.shape[:-2], data.dim() - 2
    groups = data.shape[-2]

    def whole(packed):
        return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)

    k, v, sk, sv = data.split((1024, 1024, 64, 64), -1)
    k = k.reshape(*lead, groups, 4, 16, 16).transpose(n + 1, n + 2)
    v = v.reshape(*lead, groups, 4, 16, 4, 4).transpose(n + 2, n + 3)
    sk, sv = (t.reshape(*lead, groups, 4, 16).transpose(n + 1, n + 2).reshape(
        *lead, groups * 16, 4) for t in (sk, sv))
    k, v = (whole(t.reshape(*lead, groups * 16, 4, 16)) for t in (k, v))
    return (k, sk), (v, sv)


def _plain_append(s):
    data, page = s.cache.data, s.case["page"]
    cos, sin = s.cos[:, None], s.sin[:, None]
    q = _rotate(s.q.float(), cos.float(), sin.float()).to(s.q.dtype)
    # Codes are decided next to borders: the rotation that they are taken from is in 64 bits.
    (ck, ek), (cv, ev) = (_encode(t, s.dtype) for t in (
        _rotate(s.k.double(), cos.double(), sin.double()), s.v.float()))
    slot = s.table[s.row, torch.div(s.position, page, rounding_mode="floor")].long()[:, None]
    inside = s.position % page
    group, row = (inside // 16)[:, None], (inside % 16)[:, None]
    head = torch.arange(s.k.shape[1], device=slot.device)
    packed_k, packed_v = (c[..., 0::2] | (c[..., 1::2] << 4) for c in (ck, cv))
    k, v = data[..., :1024], data[..., 1024:2048]
    lead = data.shape[:3]
    k.view(*lead, 4, 16, 16)[slot, head, group, :, row] = packed_k
    v.view(*lead, 4, 16, 4, 4)[slot, head, group, row // 4, :, row % 4] = packed_v.reshape(
        *packed_v.shape[:2], 16, 4)
    data[..., 2048:2112].view(*lead, 4, 16)[slot, head, group, :, row] = ek
    data[..., 2112:].view(*lead, 4, 16)[slot, head, group, :, row] = ev
    return q, _decode(ck, ek).to(s.dtype), _decode(cv, ev).to(s.dtype)


def _plain_attention(s):
    case = s.case
    batch, n, hk = len(s.lens), s.new[0], case["kv_heads"]
    group = case["heads"] // hk
    k, v = (_decode(*part) for part in _ungrouped(
        s.cache.data[s.table.long()].transpose(1, 2).flatten(2, 3)))
    q = s.q.view(batch, n, hk, group, HEAD_DIM).permute(0, 2, 3, 1, 4).float() \
        .reshape(batch, hk, group * n, HEAD_DIM)
    score = (q @ k.transpose(2, 3)).mul_(SCALE).view(batch, hk, group, n, -1)
    key = torch.arange(k.shape[2], device=k.device)
    at = (s.lengths[:, None] - n + torch.arange(n, device=k.device))[:, :, None]
    seen = key <= at
    if case["window"]:
        seen &= (key > at - case["window"]) | (key < case["sinks"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
    out = p.view(batch, hk, group * n, -1) @ v
    out = out.view(batch, hk, group, n, HEAD_DIM).permute(0, 3, 1, 2, 4)
    return out.reshape(batch * n, case["heads"], HEAD_DIM).to(s.q.dtype)


def _plain_select(s):
    count = s.case["count"]
    beams, vocab = s.logits.shape[1:]
    # Of each beam its best tokens, the lowest of equal ones; then of all beams.
    most = min(count, vocab)
    top, token = [], []
    for b in range(beams):
        line = s.logits[:, b].sort(dim=-1, descending=True, stable=True)
        top.append(line.values[:, :most])
        token.append(line.indices[:, :most])
    top, token = torch.stack(top, 1).double(), torch.stack(token, 1)
    # Running scores of different beams may lie close together: in 64 bits.
    peak = top[..., :1]
    mass = torch.stack([(line.double() - high).exp().sum(-1) for line, high in zip(s.logits, peak)])
    score = top - (peak + mass.log()[..., None]) + s.scores.double()[..., None]
    score = torch.where(score.isnan(), -math.inf, score).flatten(1)
    best = score.sort(dim=-1, descending=True, stable=True)
    at = best.indices[:, :count]
    return (best.values[:, :count].float(), (at // most).to(torch.int32),
            token.flatten(1).gather(1, at))


def _plain_fork(s):
    page = s.case["page"]
    parents = s.parents.long()
    lengths, old = s.lengths[parents], s.table[parents]
    full = torch.div(lengths, page, rounding_mode="floor")[:, None]
    entry = torch.arange(s.table.shape[1], device=parents.device)
    table = torch.where(entry < full, old, torch.where(entry == full, s.spare[:, None], -1))
    # The open pages' rows one by one, or the pages whole where rows lie within groups of bytes.
    source = old.gather(1, full.clamp(max=old.shape[1] - 1).long())[:, 0].long()
    moved = (lengths % page > 0).nonzero()[:, 0]
    row, inside = _open_rows(s)
    if s.case["cache"] == "16bit":
        for cache in s.caches:
            for t in (cache.k, cache.v):
                t[s.spare[row].long(), :, inside] = t[source[row], :, inside]
        return (table, lengths, *(t for c in s.caches for t in (c.k, c.v)))
    held = []
    for cache in s.caches:
        cache.data[s.spare[moved].long()] = cache.data[source[moved]]
        held.append([_decode(*part).transpose(1, 2)[row, inside].to(s.dtype)
                     for part in _ungrouped(cache.data[s.spare.long()])])
    return (table, lengths, *(torch.stack(side) for side in zip(*held)))


def _open_rows(s):
    """Sequence and row of the page of every row in the last, partly filled pages."""
    counts = torch.tensor(s.open, device=s.table.device)
    row = torch.repeat_interleave(torch.arange(len(s.open), device=counts.device), counts)
    start = torch.cumsum(counts, 0) - counts
    return row, torch.arange(len(row), device=counts.device) - start[row]


# ------------------------------------------------------------------ the floor

def _visible(case, length, new):
    """Keys of a sequence that at least one of its new tokens sees, and pairs in all."""
    keys = pairs = 0
    window, sinks = case["window"], case["sinks"]
    first = None
    for i in range(new):
        at = length - new + i
        if at < 0:
            continue
        low = max(0, at - window + 1) if window else 0
        held = at + 1 - low + min(sinks, low)
        pairs += held
        if first is None:
            first = low
        keys = at + 1 - first + min(sinks, first)
    return keys, pairs


ROW_BYTES = GROUP_BYTES // 16        # a row's keys and values of one head, scales included


def work(case):
    width = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "append4":
        tokens, hk = sum(_numbers(case["new"])), case["kv_heads"]
        angles = 4 if case["angles"] == "fp32" else 2
        # q in and out, k and v in and, as held, out, their codes, and the angles
        return {"bytes": tokens * ((2 * case["heads"] + 4 * hk) * HEAD_DIM * width
                                   + hk * ROW_BYTES + 2 * HEAD_DIM * angles),
                "flops": 3 * tokens * (case["heads"] + hk) * HEAD_DIM}
    if case["kind"] == "attention4":
        new, lengths = int(case["new"]), _numbers(case["lengths"])
        seen = [_visible(case, n, new) for n in lengths]
        keys, pairs = sum(a for a, _ in seen), sum(b for _, b in seen)
        tokens = new * len(lengths)
        return {"bytes": keys * case["kv_heads"] * ROW_BYTES
                + 2 * tokens * case["heads"] * HEAD_DIM * width,
                "flops": 4 * HEAD_DIM * pairs * case["heads"]}
    if case["kind"] == "select":
        logits = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": logits * width + 4 * case["batch"] * (case["beams"] + 4 * case["count"]),
                "flops": 3 * logits}
    rows = sum(n % case["page"] for n in _numbers(case["lengths"])) * case["beams"]
    heads = rows * case["layers"] * case["kv_heads"]
    if case["cache"] == "16bit":
        return {"bytes": heads * 4 * HEAD_DIM * width, "flops": 0}
    # read and written as codes, then given as the values they stand for
    return {"bytes": heads * (2 * ROW_BYTES + 2 * HEAD_DIM * width), "flops": 0}


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append4": _exact_append, "attention4": _exact_attention, "select": _exact_select,
            "fork": _exact_fork}[case["kind"]](s)


def _held(x, dtype):
    """x [..., 128] in fp64 as a 4-bit cache holds it."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1, keepdim=True)
    low, high = EXPONENTS[dtype]
    size = torch.full_like(top, 2.0 ** low)
    e = torch.floor(torch.log2(top.clamp_min(2.0 ** (low - 3)))) - 3
    for _ in range(3):                       # the least power of two that reaches top / 6
        e = torch.where(6.0 * torch.exp2(e) < top, e + 1, e)
    size = torch.exp2(e.clamp(low, high))
    y = blocks / size
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
    return (torch.round(y / step) * step).clamp(-6, 6).mul(size).flatten(-2)


def _exact_append(s):
    half = HEAD_DIM // 2
    c, t = s.cos.double()[:, None], s.sin.double()[:, None]

    def turned(x):
        x = x.double()
        return x * c + torch.cat((-x[..., half:], x[..., :half]), -1) * t

    return turned(s.q), _held(turned(s.k), s.dtype), _held(s.v.double(), s.dtype)


def _values(data):
    """(keys, values) fp64 [..., groups * 16, 128] of grouped bytes, value by value."""
    lead = data.shape[:-2]
    rows = torch.arange(data.shape[-2] * 16, device=data.device)[:, None]
    dim = torch.arange(HEAD_DIM, device=data.device)
    base = rows // 16 * GROUP_BYTES
    row = rows % 16
    flat = data.reshape(*lead, -1)

    def value(byte, scale):
        nibble = (flat[..., byte] >> (dim % 2 * 4).to(torch.uint8)) & 15
        exponent, mantissa = (nibble >> 1) & 3, (nibble & 1).double()
        size = torch.where(exponent == 0, mantissa / 2,
                           (1 + mantissa / 2) * torch.exp2(exponent.double() - 1))
        size = size * torch.exp2(flat[..., scale].double() - 127)
        return torch.where(nibble >= 8, -size, size)

    block = dim // BLOCK
    keys = value(base + block * 256 + row * 16 + dim % BLOCK // 2, base + 2048 + block * 16 + row)
    values = value(base + 1024 + row // 4 * 256 + dim // 8 * 16 + row % 4 * 4 + dim % 8 // 2,
                   base + 2112 + block * 16 + row)
    return keys, values


def _exact_attention(s):
    case = s.case
    n, hk = s.new[0], case["kv_heads"]
    outs = []
    for row, length in enumerate(s.lens):
        pages = s.table[row, :-(-length // case["page"])].long()
        k, v = (x[:, :length] for x in _values(s.cache.data[pages].transpose(0, 1).flatten(1, 2)))
        q = s.q[row * n:(row + 1) * n].double().view(n, hk, -1, HEAD_DIM)
        kt = k.transpose(1, 2).contiguous()
        key = torch.arange(length, device=k.device)
        for i in range(n):
            at = length - n + i
            if at < 0:
                outs.append(torch.zeros((case["heads"], HEAD_DIM), dtype=torch.float64,
                                        device=k.device))
                continue
            hidden = key > at
            if case["window"]:
                hidden = hidden | ((key <= at - case["window"]) & (key >= case["sinks"]))
            logits = torch.matmul(q[i], kt) * SCALE
            p = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
            outs.append(torch.matmul(p, v).reshape(case["heads"], HEAD_DIM))
    return torch.stack(outs)


def _exact_select(s):
    count = s.case["count"]
    scores, parents, tokens = [], [], []
    for line, running in zip(s.logits, s.scores):
        x = line.double()
        # the largest possible candidates of the whole sequence, in the order of beam and token
        value = torch.log_softmax(x, -1) + running.double()[:, None]
        value = torch.where(value.isnan(), -math.inf, value).flatten()
        least = torch.topk(value, count).values[-1]
        near = (value >= least).nonzero()[:, 0]
        order = near[torch.argsort(value[near], descending=True, stable=True)][:count]
        scores.append(value[order])
        parents.append((order // x.shape[1]).to(torch.int32))
        tokens.append(order % x.shape[1])
    return torch.stack(scores), torch.stack(parents), torch.stack(tokens)


def _exact_fork(s):
    page = s.case["page"]
    parents, old = s.parents.tolist(), s.table.tolist()
    spare = s.spare.tolist()
    table, lengths = [], []
    for row, parent in enumerate(parents):
        n = s.lens[parent]
        line = old[parent][:n // page] + [spare[row]]
        table.append((line + [-1] * len(old[0]))[:len(old[0])])
        lengths.append(n)
    moves = [(old[p][s.lens[p] // page], spare[row], s.lens[p] % page)
             for row, p in enumerate(parents) if s.lens[p] % page]
    out = []
    if s.case["cache"] == "16bit":
        for t in (t for cache in s.caches for t in (cache.k.double(), cache.v.double())):
            for a, b, n in moves:
                t[b, :, :n] = t[a, :, :n]
            out.append(t)
    else:
        none = torch.zeros((0, s.case["kv_heads"], HEAD_DIM), dtype=torch.float64,
                           device=s.table.device)
        parts = [[_values(cache.data[a]) for a, _, _ in moves] for cache in s.caches]
        for side in range(2):
            out.append(torch.stack([
                torch.cat([none] + [p[side][:, :n].transpose(0, 1)
                                    for p, (_, _, n) in zip(layer, moves)]) for layer in parts]))
    return (torch.tensor(table, dtype=torch.int32, device=s.table.device),
            torch.tensor(lengths, dtype=torch.int32, device=s.table.device), *out)
