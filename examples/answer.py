"""Answering with a tuned model: NF4 weights with LoRA adapters, a paged cache, drafted tokens.

    python examples/answer.py [--layers 2] [--tokens 64] [--budget 256]
    python examples/answer.py --beams 4 [--bits 4]

A Qwen2.5 1.5B-shaped model (random weights here; the layers are ``soupsuck_amd.layer``'s)
answers a batch of prompts of different lengths.  Each step the next tokens are guessed from the
text so far (the tokens that followed its last two before), one forward pass gives the
logits behind every guess, and ``verify_drafts`` keeps the guesses that the model would have
made.  In that pass ``append_kv`` puts the rotated keys and the values into the sequences'
pages, ``cached_attention`` reads them and adds up every row's attention weight (again for the
tokens that stay where some were refused: a weight is a vote of the text's own tokens), and when a
sequence is well past its budget ``evict_kv`` moves each head's heaviest rows to fresh pages.

With ``--bits 4`` the cache holds its rows in 4 bits (no budget then: it gives no weights).  With
``--beams`` the best of several texts at a time is kept: ``select_beams`` chooses their
continuations and ``fork_kv`` lets the caches' sequences follow.
"""

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from soupsuck_amd.kernels.add_rmsnorm import add_rms_norm  # noqa: E402
from soupsuck_amd.kernels.attention import row_offsets  # noqa: E402
from soupsuck_amd.kernels.beams import select_beams  # noqa: E402
from soupsuck_amd.kernels.nf4_gemm import gemm_f16  # noqa: E402
from soupsuck_amd.kernels.paged import (PagedCache, PagedCache4, append_kv,  # noqa: E402
                                        cached_attention, evict_kv, fork_kv)
from soupsuck_amd.kernels.rmsnorm import rms_norm  # noqa: E402
from soupsuck_amd.kernels.swiglu import swiglu  # noqa: E402
from soupsuck_amd.kernels.verify import verify_drafts  # noqa: E402
from soupsuck_amd.layer import DecoderLayer  # noqa: E402
from soupsuck_amd.lora import qlora_projection  # noqa: E402

DIM = 128


class Model:
    """Embedding, decoder layers, final norm and the tied head."""

    def __init__(self, device, layers, vocab, hidden=1536, intermediate=8960, heads=12,
                 kv_heads=2, seed=0):
        self.heads, self.kv_heads = heads, kv_heads
        gen = torch.Generator().manual_seed(seed)
        self.embedding = (torch.randn((vocab, hidden), generator=gen) * 0.05).half().to(device)
        self.norm = torch.ones(hidden, dtype=torch.float16, device=device)
        self.layers = [DecoderLayer(device, [1], hidden, intermediate, kv_heads * DIM, heads,
                                    kv_heads, seed=seed + 1 + i) for i in range(layers)]

    def __call__(self, tokens, attend):
        """Logits of packed tokens; ``attend(layer, q, k, v)`` gives a layer's attention."""
        h = self.embedding[tokens]
        t = h.shape[0]
        for i, layer in enumerate(self.layers):
            weights = {p.name: p for p in layer.proj.projections}

            def run(name, x):
                p = weights[name]
                return qlora_projection(x, p.lora_a, p.lora_b, p.packed, p.state, p.bias,
                                        layer.proj.scaling)

            x = rms_norm(h, layer.norm_in, 1e-6)
            q, k, v = (run(n, x).view(t, -1, DIM) for n in ("q_proj", "k_proj", "v_proj"))
            o = run("o_proj", attend(i, q, k, v).view(t, -1))
            h, x = add_rms_norm(h, o, layer.norm_post, 1e-6)
            h = h + run("down_proj", swiglu(run("gate_proj", x), run("up_proj", x)))
        return gemm_f16(rms_norm(h, self.norm, 1e-6), self.embedding, b_trans=True)


def rotation(positions):
    """cos and sin [tokens, 128] of Qwen2's angles."""
    inverse = 1e6 ** (-torch.arange(0, DIM, 2, dtype=torch.float64, device=positions.device) / DIM)
    angle = (positions.double()[:, None] * inverse).repeat(1, 2)
    return angle.cos().half(), angle.sin().half()


class Session:
    """A batch of texts and their pages; one table serves the caches of all layers.

    ``beams`` texts may come to continue each row (``fork``; 0 for none); ``bits`` is 16 or 4.
    """

    def __init__(self, model, rows, longest, page=16, budget=None, sinks=4, recent=32, bits=16,
                 beams=0):
        if bits not in (4, 16):
            raise ValueError("Session: a cache has 16 or 4 bits")
        if budget and (bits == 4 or beams):
            raise ValueError("Session: a budget needs the weights of a 16-bit cache, without beams")
        device = model.embedding.device
        self.model, self.page, self.budget = model, page, budget
        self.sinks, self.recent = sinks, recent
        self.slack = budget // 4 if budget else 0   # rows past the budget before it is cut
        width = -(-longest // page)
        kept = -(-budget // page) if budget else 0
        # Beams need a page each beside those that they had.
        self.free = list(range(rows * beams * (width + 1) if beams else rows * (width + kept)))
        kind = PagedCache4 if bits == 4 else PagedCache
        self.caches = [kind.empty(len(self.free), model.kv_heads, page, device=device)
                       for _ in model.layers]
        self.pages = [[] for _ in range(rows)]        # as the table has them, on the host
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.lengths = [0] * rows                     # cache rows
        self.positions = [0] * rows                   # places in the text: eviction leaves them
        shape = (rows, model.kv_heads, width * page)
        # Every row's attention weight, and the same with the pass in hand; that pass's queries.
        self.weights, self.voted = ([torch.zeros(shape, device=device) for _ in model.layers]
                                    if budget else None for _ in range(2))
        self.counts, self.queries = [0] * rows, [None] * len(model.layers)
        self.evictions = 0

    def _int32(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.table.device)

    def _hold(self, row, length):
        """Pages for ``length`` rows of a sequence."""
        while len(self.pages[row]) * self.page < length:
            self.pages[row].append(self.free.pop())
            self.table[row, len(self.pages[row]) - 1] = self.pages[row][-1]

    def forward(self, new):
        """Logits [tokens, vocab] of each row's new tokens, which enter the cache."""
        self.counts = counts = [len(n) for n in new]
        for row, n in enumerate(counts):
            self.lengths[row] += n
            self._hold(row, self.lengths[row])
        device = self.table.device
        lengths, cu = self._int32(self.lengths), row_offsets(counts, device)
        places = [p + i for p, n in zip(self.positions, counts) for i in range(n)]
        cos, sin = rotation(torch.tensor(places, device=device))

        def attend(i, q, k, v):
            q = append_kv(self.caches[i], k, v, self.table, lengths, cu, q=q, cos=cos, sin=sin)
            self.queries[i] = q
            return self._attend(i, q, lengths, cu, max(counts))

        tokens = torch.tensor([t for n in new for t in n], device=device)
        with torch.no_grad():
            logits = self.model(tokens, attend)
        self.positions = [p + n for p, n in zip(self.positions, counts)]
        return logits

    def _attend(self, i, q, lengths, cu, max_new):
        return cached_attention(q, self.caches[i], self.table, lengths, cu, max_new,
                                max(self.lengths), DIM ** -0.5,
                                weights=self.weights[i] if self.weights else None,
                                weights_out=self.voted[i] if self.weights else None)

    def settle(self, refused):
        """The last ``refused[row]`` tokens of the pass are not in the text: their rows leave the
        cache, and the weights are those that the others' queries give."""
        self.lengths = [n - r for n, r in zip(self.lengths, refused)]
        self.positions = [n - r for n, r in zip(self.positions, refused)]
        if not self.weights:
            return
        if any(refused):
            stay = [n - r for n, r in zip(self.counts, refused)]
            device = self.table.device
            starts = [sum(self.counts[:row]) for row in range(len(stay))]
            index = torch.tensor([s + i for s, n in zip(starts, stay) for i in range(n)],
                                 device=device)
            lengths, cu = self._int32(self.lengths), row_offsets(stay, device)
            for i, q in enumerate(self.queries):
                self._attend(i, q[index], lengths, cu, max(stay))
        self.weights, self.voted = self.voted, self.weights

    def fork(self, parents):
        """Row i goes on with the text of old row ``parents[i]``."""
        spare = [self.free.pop() for _ in parents]
        held = {page for line in self.pages for page in line}
        self.table, _ = fork_kv(self.caches, self.table, self._int32(self.lengths),
                                self._int32(parents), self._int32(spare))
        # As the table has it: full pages are shared, the last one is a row's own.
        self.pages = [self.pages[p][:self.lengths[p] // self.page] + [page]
                      for p, page in zip(parents, spare)]
        self.lengths = [self.lengths[p] for p in parents]
        self.positions = [self.positions[p] for p in parents]
        self.free += sorted(held - {page for line in self.pages for page in line})

    def tidy(self):
        """Sequences well past the budget are cut to it."""
        if not self.weights or max(self.lengths) <= self.budget + self.slack:
            return
        lengths = self._int32(self.lengths)
        old = self.pages
        keep = [min(n, self.budget) for n in self.lengths]
        self.pages = [[self.free.pop() for _ in range(-(-n // self.page))] for n in keep]
        fresh = torch.full((len(keep), -(-self.budget // self.page)), -1, dtype=torch.int32)
        for row, pages in enumerate(self.pages):
            fresh[row, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        fresh = fresh.to(lengths.device)
        for i, cache in enumerate(self.caches):
            _, sums = evict_kv(cache, self.table, lengths, self.weights[i], fresh, self.budget,
                               max(self.lengths), sinks=self.sinks, recent=self.recent)
            self.weights[i].zero_()
            self.weights[i][:, :, :sums.shape[2]] = sums
        self.table.fill_(-1)
        self.table[:, :fresh.shape[1]] = fresh
        self.lengths = keep
        for pages in old:
            self.free += pages
        self.evictions += 1


def guess(text, most):
    """The tokens that followed the text's last two before, at most ``most``."""
    for at in range(len(text) - 3, -1, -1):
        if text[at:at + 2] == text[-2:]:
            return text[at + 2:at + 2 + most]
    return []


def answer(model, prompts, tokens, drafts=4, temperature=0.0, budget=None, page=16, seed=0,
           bits=16):
    """(texts, forward passes, evictions): each prompt with ``tokens`` more tokens."""
    if not prompts or not all(prompts):
        raise ValueError("answer: needs prompts of at least one token")
    device = model.embedding.device
    gen = torch.Generator(device=device).manual_seed(seed)
    longest = max(len(p) for p in prompts) + tokens + 2 * drafts + 2
    session = Session(model, len(prompts), longest, page, budget, bits=bits)
    texts = [list(p) for p in prompts]
    pending = [list(p) for p in prompts]      # tokens that the cache does not hold yet
    passes = 0
    while True:
        # A row that has its tokens brings no more: the table has room for those alone.
        going = [len(t) - len(p) < tokens for t, p in zip(texts, prompts)]
        if not any(going):
            break
        drafted = [guess(t, drafts) if go else [] for t, go in zip(texts, going)]
        new = [p + d if go else [] for p, d, go in zip(pending, drafted, going)]
        logits = session.forward(new)
        passes += 1
        # Row i of a sequence's logits follows its first i guesses.
        rows = []
        end = 0
        for d, n in zip(drafted, new):
            end += len(n)
            first = max(end - len(d) - 1, 0)
            rows.append([max(min(first + i, end - 1), 0) for i in range(drafts + 1)])
        target = logits[torch.tensor(rows, device=device)]
        guesses = torch.tensor([d + [0] * (drafts - len(d)) for d in drafted],
                               dtype=torch.int64, device=device)
        uniform = torch.rand((len(texts), drafts + 1), generator=gen, device=device)
        accepted, out = verify_drafts(
            target, guesses, uniform, temperature=temperature,
            draft_counts=torch.tensor([len(d) for d in drafted], dtype=torch.int32, device=device))
        accepted, out = accepted.tolist(), out.tolist()
        session.settle([len(d) - n if go else 0 for d, n, go in zip(drafted, accepted, going)])
        for row, n in enumerate(accepted):
            if not going[row]:
                continue
            texts[row] += out[row][:n + 1]
            pending[row] = [out[row][n]]
        session.tidy()
    return [t[:len(p) + tokens] for t, p in zip(texts, prompts)], passes, session.evictions


def beam_answer(model, prompts, tokens, beams=4, bits=16, page=16, session=None):
    """(texts, scores): each prompt with the ``tokens`` more tokens that are the best of ``beams``
    texts kept at a time, and the sum of their log-probabilities."""
    if not prompts or not all(prompts):
        raise ValueError("beam_answer: needs prompts of at least one token")
    if tokens < 1 or beams < 1:
        raise ValueError("beam_answer: needs at least one token and one beam")
    rows = len(prompts)
    device = model.embedding.device
    longest = max(len(p) for p in prompts) + tokens + 1
    session = session or Session(model, rows, longest, page, bits=bits, beams=beams)
    logits = session.forward(prompts)
    ends = torch.tensor([sum(session.counts[:row + 1]) - 1 for row in range(rows)], device=device)
    # The first step: one text a row, and as many continuations of it as there are beams.
    scores, parents, chosen = select_beams(logits[ends][:, None],
                                           torch.zeros((rows, 1), device=device), beams)
    texts = [list(p) for p in prompts for _ in range(beams)]
    before = list(range(rows))                       # the session's row of each row's first text
    for step in range(tokens):
        follows = [before[row] + p for row, line in enumerate(parents.tolist()) for p in line]
        if step:
            texts = [list(texts[p]) for p in follows]
        for text, token in zip(texts, chosen.flatten().tolist()):
            text.append(token)
        if step == tokens - 1:
            break
        session.fork(follows)
        before = list(range(0, rows * beams, beams))
        logits = session.forward([text[-1:] for text in texts])
        scores, parents, chosen = select_beams(logits.view(rows, beams, -1), scores, beams)
    return texts[::beams], scores[:, 0].tolist()


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--layers", type=int, default=2)
    parser.add_argument("--tokens", type=int, default=64)
    parser.add_argument("--budget", type=int, default=256)
    parser.add_argument("--temperature", type=float, default=0.0)
    parser.add_argument("--vocab", type=int, default=32000)
    parser.add_argument("--bits", type=int, default=16, choices=(4, 16))
    parser.add_argument("--beams", type=int, default=1)
    args = parser.parse_args()
    device = torch.device("cuda", torch.cuda.current_device())
    model = Model(device, args.layers, args.vocab)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, args.vocab, (n,), generator=gen).tolist() for n in (300, 37, 180)]
    if args.beams > 1:
        texts, scores = beam_answer(model, prompts, args.tokens, args.beams, args.bits)
        for prompt, text, score in zip(prompts, texts, scores):
            print(f"{len(prompt)} tokens, then {text[len(prompt):][:12]} ... ({score:.2f})")
        return
    texts, passes, evictions = answer(model, prompts, args.tokens, temperature=args.temperature,
                                      budget=args.budget if args.bits == 16 else None,
                                      bits=args.bits)
    for prompt, text in zip(prompts, texts):
        print(f"{len(prompt)} tokens, then {text[len(prompt):][:12]} ...")
    print(f"{args.tokens} tokens each in {passes} passes, {evictions} evictions")


if __name__ == "__main__":
    main()
