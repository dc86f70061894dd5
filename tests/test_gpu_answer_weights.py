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
