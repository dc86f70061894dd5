"""The weights by which the example's bounded cache is ranked: votes of the text's own tokens."""

import pytest
import torch

import examples.answer as example

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drafts", [0, 4])
def test_only_the_texts_own_tokens_vote(device, monkeypatch, drafts):
    """Every token's probabilities sum to 1 for each q head, so that a kv head's weights sum to
    the cached tokens times its q heads, whatever was drafted and refused in between.

    A sum of n probabilities: n additions of its denominator and of its own, and exponents of at
    most 100 whose rounding the two have apart (1 step each): 2^-23 (n + 100) of the whole.
    """
    model = example.Model(device, 2, 2048, hidden=512, intermediate=1024, heads=4, kv_heads=2)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 2048, (n,), generator=gen).tolist() for n in (40, 3, 17)]
    tidy, refusals = example.Session.tidy, []

    def checked(session):
        tidy(session)
        lengths = torch.tensor(session.lengths, device=device).double()[:, None]
        behind = torch.arange(session.weights[0].shape[2], device=device) >= lengths[..., None]
        for sums in session.weights:
            total, want = sums.double().sum(-1), 2 * lengths.expand(-1, 2)
            assert ((total - want).abs() <= 2.0 ** -23 * (lengths + 100) * want).all()
            assert (sums.masked_select(behind.expand_as(sums)) == 0).all()
        refusals.append(sum(session.lengths))

    monkeypatch.setattr(example.Session, "tidy", checked)
    # guesses of which hardly one is right
    monkeypatch.setattr(example, "guess", lambda text, most: [(text[-1] * 7 + 3) % 2048] * most)
    texts, passes, evictions = example.answer(model, prompts, 12, drafts=drafts, budget=2000)
    assert evictions == 0 and passes == len(refusals)
    assert [len(t) - len(p) for t, p in zip(texts, prompts)] == [12] * 3


def test_a_bounded_cache_keeps_its_budget_and_its_pages(device, monkeypatch):
    """After every pass each page is held once or free, what the table names is what is held, and
    no sequence is past its budget by more than the slack; the heaviest rows stay."""
    model = example.Model(device, 2, 2048, hidden=512, intermediate=1024, heads=4, kv_heads=2)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 2048, (n,), generator=gen).tolist() for n in (90, 20, 61)]
    tidy, evictions = example.Session.tidy, []

    def checked(session):
        lengths, before = list(session.lengths), [w.clone() for w in session.weights]
        count = session.evictions
        tidy(session)
        held = [p for pages in session.pages for p in pages]
        assert sorted(held + session.free) == list(range(session.caches[0].k.shape[0]))
        for row, pages in enumerate(session.pages):
            assert session.table[row, :len(pages)].tolist() == pages
            assert session.lengths[row] <= len(pages) * session.page
        assert max(session.lengths) <= session.budget + session.slack
        if session.evictions > count:
            evictions.append(lengths)
            ends = session.sinks + session.recent
            for old, new in zip(before, session.weights):
                for row, n in enumerate(lengths):
                    if n <= session.budget:
                        assert torch.equal(new[row, :, :n], old[row, :, :n])
                        continue
                    middle = old[row, :, session.sinks:n - session.recent]
                    best = middle.topk(session.budget - ends).values.sort().values
                    got = new[row, :, session.sinks:session.budget - session.recent]
                    assert torch.equal(got.sort().values, best)
                    assert (new[row, :, session.budget:] == 0).all()

    monkeypatch.setattr(example.Session, "tidy", checked)
    texts, _, count = example.answer(model, prompts, 50, budget=64, temperature=0.8)
    assert count == len(evictions) > 0
    for prompt, text in zip(prompts, texts):
        assert text[:len(prompt)] == prompt and len(text) == len(prompt) + 50
