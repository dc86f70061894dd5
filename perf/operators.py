"""Answering with a tuned model: the paged-cache and drafting operators, and their plain forms.

Kinds of case:

  append     new tokens' keys (rotated) and values into the pages of their sequences, the
             queries rotated by the same call
  attention  new tokens over a paged cache, with a sliding window, first tokens that stay
             visible and each key's accumulated attention weight where the case has them
  evict      the heaviest rows of each kv head copied to other pages
  verify     drafted tokens against the target's logits from given uniform numbers

Head layouts are those of Qwen2.5 1.5B (12 / 2) and 7B (28 / 4), the vocabulary is theirs;
sequences are ragged.  listed() names the cases, draw() gives more of the same ranges,
prepare() makes what a program has in hand, run() is one pass (the framework's calls where
``own`` is true, plain torch in 32 or 64 bits elsewhere), work() the bytes and flops a pass
cannot do without and exact() the result in 64 bits.
"""

import math
from types import SimpleNamespace

import torch

own = False

HEAD_DIM = 128
VOCAB = 151936
SMALL, LARGE = (12, 2), (28, 4)      # q / kv heads of the 1.5B and the 7B model
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SCALE = HEAD_DIM ** -0.5


# ----------------------------------------------------------------- the cases

def listed():
    return [
        # one sequence's next token: the append between two products of a decode step
        {"name": "append_one", "kind": "append", "dtype": "fp16", "heads": 12, "kv_heads": 2,
         "page": 64, "new": "1", "past": "517"},
        # prompts of several sequences entering the cache together, some after a shared start
        {"name": "append_prompts", "kind": "append", "dtype": "bf16", "heads": 28,
         "kv_heads": 4, "page": 16, "new": "2048,1537,1201,777,350,128,1",
         "past": "0,64,0,333,0,0,5000"},
        # interactive: one short conversation, one token; latency is all
        {"name": "attention_one_short", "kind": "attention", "dtype": "fp16", "heads": 12,
         "kv_heads": 2, "page": 64, "new": "1", "lengths": "518", "window": 0, "sinks": 0,
         "weights": False},
        # one very long document, one token: the cache's length is all the parallelism
        {"name": "attention_one_long", "kind": "attention", "dtype": "fp16", "heads": 28,
         "kv_heads": 4, "page": 64, "new": "1", "lengths": "131071", "window": 0, "sinks": 0,
         "weights": False},
        # a serving batch of ragged conversations, one token each, small pages
        {"name": "attention_batch", "kind": "attention", "dtype": "fp16", "heads": 28,
         "kv_heads": 4, "page": 16, "new": "1",
         "lengths": "4099,3801,77,2048,1,640,1999,8191,513,129,6007,2741,350,1201,31,4760",
         "window": 0, "sinks": 0, "weights": False},
        # drafted tokens of a batch verified in one pass: five queries a sequence
        {"name": "attention_drafts", "kind": "attention", "dtype": "bf16", "heads": 12,
         "kv_heads": 2, "page": 32, "new": "5", "lengths": "2047,1531,990,4095,261,3333,1777,642",
         "window": 0, "sinks": 0, "weights": False},
        # long streams kept to a window and their first tokens
        {"name": "attention_window", "kind": "attention", "dtype": "bf16", "heads": 28,
         "kv_heads": 4, "page": 64, "new": "1", "lengths": ",".join(["16111,9001,30003,20011"] * 8),
         "window": 4096, "sinks": 4, "weights": False},
        # a large batch whose cache is bounded by eviction: weights accumulated, one token each
        {"name": "attention_weights", "kind": "attention", "dtype": "fp16", "heads": 28,
         "kv_heads": 4, "page": 64, "new": "1",
         "lengths": ",".join(str(8191 - 37 * i) for i in range(64)), "window": 0, "sinks": 0,
         "weights": True},
        # one sequence past its budget
        {"name": "evict_one", "kind": "evict", "dtype": "fp16", "kv_heads": 2, "page": 64,
         "lengths": "1281", "budget": 1024, "sinks": 4, "recent": 256},
        # a serving batch halved at once
        {"name": "evict_batch", "kind": "evict", "dtype": "bf16", "kv_heads": 4, "page": 16,
         "lengths": ",".join(str(8191 - 201 * i) for i in range(32)), "budget": 4096, "sinks": 4,
         "recent": 1024},
        # one conversation's four drafted tokens
        {"name": "verify_one", "kind": "verify", "dtype": "fp16", "batch": 1, "drafts": 4,
         "ragged": False, "vocab": VOCAB, "temperature": 1.0, "draft": "logits"},
        # a batch's drafts, fewer where the draft model stopped early
        {"name": "verify_batch", "kind": "verify", "dtype": "fp32", "batch": 32, "drafts": 6,
         "ragged": True, "vocab": VOCAB, "temperature": 0.7, "draft": "logits"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], uniform over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _text(values):
    return ",".join(str(int(v)) for v in values)


def draw(rng):
    kind = rng.choice(("append", "attention", "attention", "attention", "evict", "verify"))
    dtype = rng.choice(("fp16", "bf16"))
    heads, kv_heads = rng.choice((SMALL, LARGE))
    page = rng.choice((16, 32, 64, 128))
    if kind == "append":
        total, new = _spread(rng, 1, 6000), []
        while sum(new) < total:
            new.append(min(_spread(rng, 1, 2048), total - sum(new)))
        return {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "page": page,
                "new": _text(new),
                "past": _text(rng.choice((0, _spread(rng, 1, 8000))) for _ in new)}
    if kind == "attention":
        new = rng.choice((1, 1, 1, 2, 5, 8, 33))     # one token, drafts, a piece of a prompt
        tokens = _spread(rng, 1, 500000 // new)      # keys of the whole batch
        batch = _spread(rng, max(1, tokens // 100000), max(1, min(64, tokens // 8)))
        mean = max(1, tokens // batch)
        lengths = [max(new, _spread(rng, max(1, mean // 4), min(131071, max(1, mean * 3 // 2))))
                   for _ in range(batch)]
        return {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "page": page,
                "new": str(new), "lengths": _text(lengths),
                "window": rng.choice((0, 0, _spread(rng, 16, 8192))),
                "sinks": rng.choice((0, 4, 16)), "weights": rng.random() < 0.25}
    if kind == "evict":
        batch = _spread(rng, 1, 32)
        top = _spread(rng, 40, 8191)
        lengths = [rng.randint(max(1, top // 3), top) for _ in range(batch)]
        budget = max(1, int(top * rng.uniform(0.3, 0.9)))
        sinks = min(rng.choice((0, 4)), budget)
        return {"kind": kind, "dtype": dtype, "kv_heads": kv_heads, "page": page,
                "lengths": _text(lengths), "budget": budget, "sinks": sinks,
                "recent": int((budget - sinks) * rng.uniform(0.0, 0.8))}
    batch = _spread(rng, 1, 32)
    return {"kind": kind, "dtype": rng.choice(("fp16", "bf16", "fp32")), "batch": batch,
            "drafts": rng.randint(1, 7 if batch <= 24 else 5), "ragged": rng.random() < 0.5,
            "vocab": rng.choice((VOCAB, VOCAB, _spread(rng, 1000, VOCAB))),
            "temperature": rng.choice((0.0, 0.7, 1.0)),
            "draft": rng.choice(("logits", "logits", "none"))}


# ------------------------------------------------------------- what is in hand

def _numbers(text):
    return [int(v) for v in text.split(",")]


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _generator(seed):
    return torch.Generator(device=_device()).manual_seed(int(seed))


def _normal(gen, shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device=gen.device).mul_(std).to(dtype)


def _pages(gen, lengths, page, extra=0):
    """(pages in all, block table [rows, most pages] int32): pages handed out in random order."""
    need = [max(1, -(-n // page)) for n in lengths]
    total = sum(need) + extra
    order = torch.randperm(total, generator=gen, device=gen.device).to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device=gen.device)
    start = 0
    for row, n in enumerate(need):
        table[row, :n] = order[start:start + n]
        start += n
    return total, table


def _cache(k, v):
    if not own:
        return SimpleNamespace(k=k, v=v)
    from soupsuck_amd.kernels.paged import PagedCache
    return PagedCache(k, v)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=_device())


def _offsets(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = _generator(seed)
    s = SimpleNamespace(case=case)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "verify":
        return _prepare_verify(case, gen, s, dtype)
    page, hk = case["page"], case["kv_heads"]
    if case["kind"] == "append":
        s.new, past = _numbers(case["new"]), _numbers(case["past"])
        s.lens = [a + b for a, b in zip(s.new, past)]
        pages, s.table = _pages(gen, s.lens, page)
        total = sum(s.new)
        s.cache = _cache(*(torch.zeros((pages, hk, page, HEAD_DIM), dtype=dtype, device=gen.device)
                           for _ in range(2)))
        # The fused projection's rows: q, k and v of a token lie side by side.
        qkv = _normal(gen, (total, case["heads"] + 2 * hk, HEAD_DIM), dtype)
        s.q, s.k, s.v = qkv.split((case["heads"], hk, hk), dim=1)
        position = torch.cat([torch.arange(b, a + b) for a, b in zip(s.new, past)]).double()
        inverse = 1e6 ** (-torch.arange(0, HEAD_DIM, 2).double() / HEAD_DIM)
        angle = (position[:, None] * inverse).repeat(1, 2)
        s.cos, s.sin = (f(angle).to(dtype).to(gen.device) for f in (torch.cos, torch.sin))
        s.lengths, s.cu = _int32(s.lens), _int32(_offsets(s.new))
        s.max_new, s.position = max(s.new), position.long().to(gen.device)
        s.row = torch.repeat_interleave(torch.arange(len(s.new)), torch.tensor(s.new)) \
            .to(gen.device)
        return s
    s.lens = _numbers(case["lengths"])
    batch = len(s.lens)
    if case["kind"] == "attention":
        pages, s.table = _pages(gen, s.lens, page)
        s.new = [int(case["new"])] * batch
        # Keys and queries with a direction in common, which the first key holds strongly (the
        # sink of trained models), over noise that leaves a few heavy keys.
        common = torch.randn((hk, 1, HEAD_DIM), generator=gen, device=gen.device)
        k = torch.randn((pages, hk, page, HEAD_DIM), generator=gen, device=gen.device) * 1.5
        first = s.table[:, 0].long()
        k[first, :, 0] = common[:, 0] * 0.6
        s.cache = _cache(k.to(dtype), _normal(gen, k.shape, dtype))
        q = torch.randn((sum(s.new), hk, case["heads"] // hk, HEAD_DIM), generator=gen,
                        device=gen.device) + common
        s.q = q.to(dtype).view(sum(s.new), case["heads"], HEAD_DIM)
        s.weights = s.out = None
        if case["weights"]:
            s.weights = torch.rand((batch, hk, s.table.shape[1] * page), generator=gen,
                                   device=gen.device)
            s.out = torch.zeros_like(s.weights)
        s.lengths, s.cu, s.max_new = _int32(s.lens), _int32(_offsets(s.new)), max(s.new)
        s.max_length = max(s.lens)
        return s
    kept = [min(n, case["budget"]) for n in s.lens]
    need = sum(-(-n // page) for n in kept)
    pages, s.table = _pages(gen, s.lens, page, extra=need)
    # The free pages are those that no row holds.
    free = torch.ones(pages, dtype=torch.bool, device=gen.device)
    for row, n in enumerate(s.lens):
        free[s.table[row, :-(-n // page)].long()] = False
    free = free.nonzero()[:, 0].to(torch.int32)
    s.out_table = torch.zeros((batch, -(-case["budget"] // page)), dtype=torch.int32,
                              device=gen.device)
    start = 0
    for row, n in enumerate(kept):
        s.out_table[row, :-(-n // page)] = free[start:start - (-n // page)]
        start += -(-n // page)
    k, v = (_normal(gen, (pages, hk, page, HEAD_DIM), dtype) for _ in range(2))
    s.cache = _cache(k, v)
    # Accumulated weights are heavy-tailed, and many small ones are equal.
    weights = torch.rand((batch, hk, s.table.shape[1] * page), generator=gen, device=gen.device)
    s.weights = (weights.pow(-0.7) * 64).round() / 64
    s.lengths, s.max_length = _int32(s.lens), max(s.lens)
    return s


def _prepare_verify(case, gen, s, dtype):
    b, g, vocab = case["batch"], case["drafts"], case["vocab"]
    s.target = _normal(gen, (b, g + 1, vocab), dtype, 2.5)
    s.draft = None
    heat = case["temperature"] or 1.0
    if case["draft"] == "logits":
        s.draft = (s.target[:, :g].float()
                   + torch.randn((b, g, vocab), generator=gen, device=gen.device)).to(dtype)
        source = s.draft.float()
    else:
        source = s.target[:, :g].float() * 3
    noise = torch.rand(source.shape, generator=gen, device=gen.device).clamp_(1e-20, 1 - 1e-7)
    if case["temperature"] == 0.0:
        # a greedy draft: mostly the target's own best, sometimes its own guess
        best = s.target[:, :g].float().argmax(-1)
        s.tokens = torch.where(noise[..., 0] < 0.8, best, source.argmax(-1))
    else:
        s.tokens = (source / heat - noise.log_().neg_().log_()).argmax(-1)
    s.uniform = torch.rand((b, g + 1), generator=gen, device=gen.device)
    s.counts = None
    if case["ragged"]:
        s.counts = torch.randint(0, g + 1, (b,), generator=gen, device=gen.device,
                                 dtype=torch.int32)
    return s


# ------------------------------------------------------------------- one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    case = s.case
    if case["kind"] == "verify":
        from soupsuck_amd.kernels.verify import verify_drafts
        accepted, tokens = verify_drafts(s.target, s.tokens, s.uniform, draft_logits=s.draft,
                                         draft_counts=s.counts, temperature=case["temperature"])
        return accepted, tokens
    from soupsuck_amd.kernels.paged import append_kv, evict_kv, cached_attention
    if case["kind"] == "append":
        q = append_kv(s.cache, s.k, s.v, s.table, s.lengths, s.cu, q=s.q, cos=s.cos, sin=s.sin)
        return q, s.cache.k, s.cache.v
    if case["kind"] == "attention":
        out = cached_attention(s.q, s.cache, s.table, s.lengths, s.cu, s.max_new, s.max_length,
                               scale=SCALE, window=case["window"] or None, sinks=case["sinks"],
                               weights=s.weights, weights_out=s.out)
        return out if s.out is None else (out, s.out)
    lengths, weights = evict_kv(s.cache, s.table, s.lengths, s.weights, s.out_table,
                                case["budget"], s.max_length, sinks=case["sinks"],
                                recent=case["recent"])
    return lengths, weights, s.cache.k, s.cache.v


def _run_plain(s):
    return {"append": _plain_append, "attention": _plain_attention, "evict": _plain_evict,
            "verify": _plain_verify}[s.case["kind"]](s)


def _rotate(x, cos, sin):
    x, cos, sin = x.float(), cos.float()[:, None], sin.float()[:, None]
    half = x.shape[-1] // 2
    low, high = x[..., :half], x[..., half:]
    return torch.cat((low * cos[..., :half] - high * sin[..., :half],
                      high * cos[..., half:] + low * sin[..., half:]), -1)


def _plain_append(s):
    page = s.cache.k.shape[2]
    slot = s.table[s.row, s.position // page].long()
    inside = s.position % page
    q = _rotate(s.q, s.cos, s.sin).to(s.q.dtype)
    s.cache.k[slot, :, inside] = _rotate(s.k, s.cos, s.sin).to(s.k.dtype)
    s.cache.v[slot, :, inside] = s.v
    return q, s.cache.k, s.cache.v


def _rows(pages, table):
    """[rows, kv heads, capacity, ...] of a paged tensor."""
    got = pages[table.long()].transpose(1, 2)
    return got.reshape(got.shape[0], got.shape[1], -1, *got.shape[4:])


def _plain_attention(s):
    case = s.case
    batch, n, hk = len(s.lens), s.new[0], case["kv_heads"]
    group = case["heads"] // hk
    k, v = _rows(s.cache.k, s.table).float(), _rows(s.cache.v, s.table).float()
    q = s.q.view(batch, n, hk, group, HEAD_DIM).permute(0, 2, 3, 1, 4).float() \
        .reshape(batch, hk, group * n, HEAD_DIM)
    score = (q @ k.transpose(2, 3)).mul_(SCALE).view(batch, hk, group, n, -1)
    key = torch.arange(k.shape[2], device=k.device)
    at = (s.lengths[:, None] - n + torch.arange(n, device=k.device))[:, :, None]
    seen = key <= at
    if case["window"]:
        seen &= (key > at - case["window"]) | (key < case["sinks"])
    seen = seen[:, None, None]
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
    out = p.view(batch, hk, group * n, -1) @ v
    out = out.view(batch, hk, group, n, HEAD_DIM).permute(0, 3, 1, 2, 4)
    out = out.reshape(batch * n, case["heads"], HEAD_DIM).to(s.q.dtype)
    if s.out is None:
        return out
    torch.add(s.weights, p.sum((2, 3)), out=s.out)
    return out, s.out


def _plain_evict(s):
    case = s.case
    budget, page = case["budget"], s.cache.k.shape[2]
    batch, hk, capacity = s.weights.shape
    key = torch.arange(capacity, device=s.weights.device)
    held = s.lengths[:, None].long()
    rank = (key < held).long()
    rank += rank * ((key < case["sinks"]) | (key >= held - case["recent"]))
    rank = rank[:, None].expand(batch, hk, capacity)
    order = torch.argsort(s.weights, dim=-1, descending=True, stable=True)
    order = order.gather(-1, torch.argsort(rank.gather(-1, order), dim=-1, descending=True,
                                           stable=True))[..., :budget]
    kept = s.lengths.clamp(max=budget)
    here = (torch.arange(order.shape[-1], device=key.device) < kept[:, None])[:, None]
    order = torch.where(here, order, capacity).sort(-1).values
    source = order.clamp(max=capacity - 1)
    full = torch.zeros((batch, hk, s.out_table.shape[1] * page), device=key.device)
    full[..., :order.shape[-1]] = torch.where(here, s.weights.gather(-1, source), 0.0)
    row, at = here[:, 0].nonzero(as_tuple=True)
    from_at = source[row, :, at]                                  # [rows kept, kv heads]
    from_page = s.table[row[:, None], from_at // page].long()
    to_page = s.out_table[row, at // page].long()[:, None]
    head = torch.arange(hk, device=key.device)
    for pages in (s.cache.k, s.cache.v):
        pages[to_page, head, (at % page)[:, None]] = pages[from_page, head, from_at % page]
    return kept, full, s.cache.k, s.cache.v


def _plain_verify(s):
    b, g, vocab = s.target.shape[0], s.tokens.shape[1], s.target.shape[2]
    counts = torch.full((b,), g, device=s.target.device) if s.counts is None else s.counts.long()
    step = torch.arange(g, device=s.target.device)
    row = torch.arange(b, device=s.target.device)
    heat = s.case["temperature"]
    if heat == 0.0:
        best = s.target.float().argmax(-1)
        good = (best[:, :g] == s.tokens) & (step < counts[:, None])
        accepted = good.long().cumprod(1).sum(1)
        last = best[row, accepted]
    else:
        p = torch.softmax(s.target.double() / heat, -1)
        px = p[:, :g].gather(-1, s.tokens[..., None])[..., 0]
        if s.draft is None:
            q, qx = None, torch.ones_like(px)
        else:
            q = torch.softmax(s.draft.double() / heat, -1)
            qx = q.gather(-1, s.tokens[..., None])[..., 0]
        good = (s.uniform[:, :g].double() * qx < px) & (step < counts[:, None])
        accepted = good.long().cumprod(1).sum(1)
        left = p[row, accepted]
        refused = (accepted < counts)[:, None]
        at = accepted.clamp(max=g - 1)
        if q is None:
            other = (torch.arange(vocab, device=p.device) == s.tokens[row, at][:, None]).double()
        else:
            other = q[row, at]
        rest = torch.where(refused, (left - other).clamp_min(0.0), left)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, left)
        mass = rest.cumsum(-1)
        last = torch.searchsorted(mass, s.uniform[:, g:].double() * mass[:, -1:],
                                  right=True)[:, 0].clamp(max=vocab - 1)
    tokens = torch.full((b, g + 1), -1, device=s.target.device)
    tokens[:, :g] = torch.where(step < accepted[:, None], s.tokens, -1)
    tokens[row, accepted] = last
    return accepted.to(torch.int32), tokens


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


def work(case):
    width = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "append":
        tokens = sum(_numbers(case["new"]))
        rows = tokens * (case["heads"] + 2 * case["kv_heads"])
        return {"bytes": (2 * rows + 2 * tokens) * HEAD_DIM * width + 4 * tokens,
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * HEAD_DIM}
    if case["kind"] == "attention":
        new, lengths = int(case["new"]), _numbers(case["lengths"])
        seen = [_visible(case, n, new) for n in lengths]
        keys, pairs = sum(a for a, _ in seen), sum(b for _, b in seen)
        tokens = new * len(lengths)
        moved = (2 * keys * case["kv_heads"] + 2 * tokens * case["heads"]) * HEAD_DIM * width
        if case["weights"]:
            moved += 2 * 4 * sum(lengths) * case["kv_heads"]
        return {"bytes": moved, "flops": 4 * HEAD_DIM * pairs * case["heads"]}
    if case["kind"] == "evict":
        lengths = _numbers(case["lengths"])
        kept = sum(min(n, case["budget"]) for n in lengths)
        return {"bytes": case["kv_heads"] * (sum(lengths) * 4 + kept * (4 * HEAD_DIM * width + 4)),
                "flops": 0}
    b, g = case["batch"], case["drafts"]
    # the rows up to each sequence's count of drafts, which averages half when ragged
    drafts = b * g / 2 if case["ragged"] else b * g
    logits = (drafts + b) * case["vocab"]
    if case["draft"] == "logits" and case["temperature"]:
        logits += drafts * case["vocab"]
    return {"bytes": logits * width + 20 * b * (g + 1), "flops": 4 * logits}


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "evict": _exact_evict,
            "verify": _exact_verify}[case["kind"]](s)


def _exact_append(s):
    k, v = s.cache.k.double(), s.cache.v.double()
    page = k.shape[2]
    half = HEAD_DIM // 2
    c, t = s.cos.double()[:, None], s.sin.double()[:, None]

    def turned(x):
        x = x.double()
        return x * c + torch.cat((-x[..., half:], x[..., :half]), -1) * t

    rotated = turned(s.k)
    start = 0
    for row, (new, length) in enumerate(zip(s.new, s.lens)):
        at = torch.arange(length - new, length, device=k.device)
        where = s.table[row].long()[torch.div(at, page, rounding_mode="floor")]
        k[where, :, at % page] = rotated[start:start + new]
        v[where, :, at % page] = s.v[start:start + new].double()
        start += new
    return turned(s.q), k, v


def _exact_attention(s):
    case = s.case
    n, hk = s.new[0], case["kv_heads"]
    outs = []
    sums = None if s.weights is None else s.weights.double()
    for row, length in enumerate(s.lens):
        pages = s.table[row].long()
        k, v = (x[pages].double().permute(1, 0, 2, 3).reshape(hk, -1, HEAD_DIM)[:, :length]
                for x in (s.cache.k, s.cache.v))
        q = s.q[row * n:(row + 1) * n].double().view(n, hk, -1, HEAD_DIM)
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
            logits = torch.matmul(q[i], k.transpose(1, 2).contiguous()) * SCALE
            p = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
            outs.append(torch.matmul(p, v).reshape(case["heads"], HEAD_DIM))
            if sums is not None:
                sums[row, :, :length] += p.sum(1)
    out = torch.stack(outs)
    return out if sums is None else (out, sums)


def _exact_evict(s):
    case = s.case
    page, hk = s.cache.k.shape[2], case["kv_heads"]
    k, v = s.cache.k.double(), s.cache.v.double()
    sums = torch.zeros((len(s.lens), hk, s.out_table.shape[1] * page), dtype=torch.float64,
                       device=k.device)
    host = s.weights.cpu().numpy()
    kept_lengths = []
    for row, length in enumerate(s.lens):
        kept = min(length, case["budget"])
        kept_lengths.append(kept)
        for head in range(hk):
            low, high = min(case["sinks"], length), max(0, length - case["recent"])
            middle = list(range(low, max(low, high)))
            ends = list(range(low)) + list(range(max(low, high), length))
            room = max(0, kept - len(ends))
            heavy = sorted(middle, key=lambda j: (-host[row, head, j], j))[:room]
            take = torch.tensor(sorted(ends + heavy), device=k.device)
            to = torch.arange(kept, device=k.device)
            a, b = s.table[row].long()[take // page], s.out_table[row].long()[to // page]
            k[b, head, to % page] = k[a, head, take % page]
            v[b, head, to % page] = v[a, head, take % page]
            sums[row, head, :kept] = s.weights[row, head, take].double()
    return torch.tensor(kept_lengths, dtype=torch.int32, device=k.device), sums, k, v


def _exact_verify(s):
    heat = s.case["temperature"]
    b, g = s.tokens.shape
    vocab = s.target.shape[2]
    counts = [g] * b if s.counts is None else s.counts.tolist()
    drafted, uniform = s.tokens.tolist(), s.uniform.double().tolist()
    accepted, tokens = [], []
    for row in range(b):
        out, last = [], None
        for i in range(counts[row]):
            x = drafted[row][i]
            logits = s.target[row, i].double()
            if heat == 0.0:
                best = int((logits == logits.max()).nonzero()[0])
                if best == x:
                    out.append(x)
                    continue
                last = best
                break
            p = torch.exp(torch.log_softmax(logits / heat, 0))
            if s.draft is None:
                q = torch.zeros(vocab, dtype=torch.float64, device=p.device)
                q[x] = 1.0
            else:
                q = torch.exp(torch.log_softmax(s.draft[row, i].double() / heat, 0))
            if uniform[row][i] * float(q[x]) < float(p[x]):
                out.append(x)
                continue
            rest = torch.relu(p - q)
            last = _inverse(rest if float(rest.sum()) > 0 else p, uniform[row][g])
            break
        if last is None:
            logits = s.target[row, counts[row]].double()
            if heat == 0.0:
                last = int((logits == logits.max()).nonzero()[0])
            else:
                last = _inverse(torch.exp(torch.log_softmax(logits / heat, 0)), uniform[row][g])
        accepted.append(len(out))
        tokens.append(out + [last] + [-1] * (g - len(out)))
    dev = s.target.device
    return (torch.tensor(accepted, dtype=torch.int32, device=dev),
            torch.tensor(tokens, dtype=torch.int64, device=dev))


def _inverse(mass, u):
    total = torch.cumsum(mass, 0)
    return min(int((total <= u * total[-1]).sum()), mass.numel() - 1)
