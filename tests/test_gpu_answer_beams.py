"""The example over a 4-bit cache and with beams: append, attention, selection and forks together.

A row's attention does not depend on the pages that hold it, so sessions whose forks copy whole
sequences to pages of their own in plain torch have to give the very same texts and scores.
"""

import pytest
import torch

from examples.answer import Model, Session, answer, beam_answer
from soupsuck_amd.kernels.paged import PagedCache4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(device):
    return Model(device, 2, 2048, hidden=512, intermediate=1024, heads=4, kv_heads=2)


def _prompts(vocab, lengths):
    gen = torch.Generator().manual_seed(5)
    return [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in lengths]


class Copying(Session):
    """Forks by copies: no page is shared."""

    def fork(self, parents):
        old = self.pages
        need = [-(-(self.lengths[p] + 1) // self.page) for p in parents]
        fresh = [[self.free.pop() for _ in range(n)] for n in need]
        for cache in self.caches:
            tensors = (cache.data,) if isinstance(cache, PagedCache4) else (cache.k, cache.v)
            for t in tensors:
                moved = [t[old[p]].clone() for p in parents]
                for pages, rows in zip(fresh, moved):
                    t[pages[:len(rows)]] = rows[:len(pages)]
        table = torch.full((len(parents), self.table.shape[1]), -1, dtype=torch.int32)
        for row, pages in enumerate(fresh):
            table[row, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        self.table = table.to(self.table.device)
        self.pages = fresh
        self.lengths = [self.lengths[p] for p in parents]
        self.positions = [self.positions[p] for p in parents]
        self.free += [page for line in old for page in line]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("beams,page", [(1, 16), (3, 16), (4, 32)])
def test_forks_share_pages_and_change_nothing(model, bits, beams, page):
    prompts, tokens = _prompts(2048, (40, 3, 32)), 21
    texts, scores = beam_answer(model, prompts, tokens, beams, bits, page)
    # room for the copies beside what they are taken from
    copying = Copying(model, 3, 40 + tokens + 1, page, bits=bits, beams=2 * beams + 2)
    want, want_scores = beam_answer(model, prompts, tokens, beams, bits, page, session=copying)
    assert texts == want and scores == want_scores
    for prompt, text in zip(prompts, texts):
        assert text[:len(prompt)] == prompt and len(text) == len(prompt) + tokens


@pytest.mark.parametrize("bits", [16, 4])
def test_one_beam_is_the_greedy_answer(model, bits):
    prompts = _prompts(2048, (33, 7))
    greedy, _, _ = answer(model, prompts, 20, drafts=0, bits=bits)
    texts, scores = beam_answer(model, prompts, 20, 1, bits)
    assert texts == greedy and all(s < 0 for s in scores)


def test_pages_come_back(model):
    """After every fork no page is lost, and none has two uses."""
    session = Session(model, 2, 60, 16, bits=4, beams=3)
    every = sorted(session.free)
    session.forward(_prompts(2048, (15, 20)))
    session.fork([0, 0, 0, 1, 1, 1])
    for step in range(30):
        session.forward([[step]] * 6)
        parents = [(step * 7 + i * i) % 3 + 3 * (i // 3) for i in range(6)]
        session.fork(parents)
        used = {page for line in session.pages for page in line}
        assert sorted(session.free + list(used)) == every
        table = session.table.tolist()
        for line, pages in zip(table, session.pages):
            assert line[:len(pages)] == pages
        last = [pages[-1] for pages in session.pages]
        assert len(set(last)) == 6


@pytest.mark.parametrize("bits", [16, 4])
def test_drafted_answers_over_either_cache(model, bits):
    prompts = _prompts(2048, (50, 4))
    texts, passes, _ = answer(model, prompts, 30, drafts=3, bits=bits)
    assert passes <= 31
    for prompt, text in zip(prompts, texts):
        assert text[:len(prompt)] == prompt and len(text) == len(prompt) + 30


def test_refusals(model):
    with pytest.raises(ValueError, match="16 or 4"):
        Session(model, 1, 10, bits=8)
    with pytest.raises(ValueError, match="budget"):
        answer(model, [[1]], 2, budget=64, bits=4)
    with pytest.raises(ValueError, match="at least one token"):
        beam_answer(model, [[]], 2)
    with pytest.raises(ValueError, match="one beam"):
        beam_answer(model, [[1]], 2, beams=0)
