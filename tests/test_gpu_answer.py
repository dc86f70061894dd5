"""The example that answers with a tuned model: append, attention, eviction and verification
together, against the same text in one pass."""

import pytest
import torch

from examples.answer import Model, Session, answer, guess

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(device):
    return Model(device, 2, 2048, hidden=512, intermediate=1024, heads=4, kv_heads=2)


def _prompts(vocab, lengths):
    gen = torch.Generator().manual_seed(3)
    return [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in lengths]


def test_guess():
    assert guess([1, 2, 3, 4, 1, 2], 2) == [3, 4]
    assert guess([1, 2, 3], 4) == [] and guess([5], 4) == [] and guess([], 4) == []


@pytest.mark.parametrize("drafts", [0, 4])
def test_greedy_answers_are_the_models_own(model, drafts):
    """Every token is the best of the whole text's logits in one pass, up to the fp16 rounding
    of two ways through the model (2e-2 of the logits' largest)."""
    prompts = _prompts(2048, (40, 3, 17))
    texts, passes, evictions = answer(model, prompts, 24, drafts=drafts)
    assert evictions == 0 and passes <= 24 + 1
    session = Session(model, 3, 80)
    logits = session.forward(texts).float()
    start = 0
    for prompt, text in zip(prompts, texts):
        assert text[:len(prompt)] == prompt and len(text) == len(prompt) + 24
        rows = logits[start + len(prompt) - 1:start + len(text) - 1]
        got = rows.gather(1, torch.tensor(text[len(prompt):], device=rows.device)[:, None])[:, 0]
        assert (rows.amax(1) - got <= 2e-2 * rows.abs().amax(1)).all()
        start += len(text)


def test_drafts_save_passes_and_change_nothing_drawn(model):
    """With guesses that are always right there are fewer passes; the first token is the same."""
    prompts = _prompts(2048, (12, 9))
    one, passes, _ = answer(model, prompts, 40, drafts=0)
    many, fewer, _ = answer(model, prompts, 40, drafts=4)
    assert fewer <= passes
    assert [t[len(p)] for t, p in zip(one, prompts)] == [t[len(p)] for t, p in zip(many, prompts)]


def test_a_bounded_cache(model):
    prompts = _prompts(2048, (90, 20, 61))
    texts, _, evictions = answer(model, prompts, 50, budget=64, temperature=0.8)
    assert evictions > 0
    for prompt, text in zip(prompts, texts):
        assert len(text) == len(prompt) + 50 and all(0 <= t < 2048 for t in text)
