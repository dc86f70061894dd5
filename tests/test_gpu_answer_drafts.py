"""Drafted answers of the example's model with guesses that are known to be right or wrong."""

import pytest
import torch

import examples.answer as example

pytestmark = pytest.mark.gpu
TOKENS, DRAFTS = 40, 4


@pytest.fixture(scope="module")
def told(device):
    """(model, prompts, texts without drafts)."""
    model = example.Model(device, 2, 2048, hidden=512, intermediate=1024, heads=4, kv_heads=2)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 2048, (n,), generator=gen).tolist() for n in (12, 9, 30)]
    texts, passes, _ = example.answer(model, prompts, TOKENS, drafts=0)
    assert passes == TOKENS
    _are_its_own(model, prompts, texts)
    return model, prompts, texts


def _are_its_own(model, prompts, texts):
    """Every token is the best of the whole text's logits in one pass, up to the fp16 rounding
    of two ways through the model (2e-2 of the logits' largest)."""
    logits = example.Session(model, len(texts), 100).forward(texts).float()
    start = 0
    for prompt, text in zip(prompts, texts):
        assert text[:len(prompt)] == prompt and len(text) == len(prompt) + TOKENS
        rows = logits[start + len(prompt) - 1:start + len(text) - 1]
        got = rows.gather(1, torch.tensor(text[len(prompt):], device=rows.device)[:, None])[:, 0]
        assert (rows.amax(1) - got <= 2e-2 * rows.abs().amax(1)).all()
        start += len(text)


def _guesses(told, change):
    """The tokens that follow where the text so far is one that was told, changed."""
    def guess(text, most):
        for full in told:
            if full[:len(text)] == text:
                return [change(t) for t in full[len(text):len(text) + most]]
        return []
    return guess


@pytest.mark.parametrize("budget", [None, 200])
def test_right_guesses_save_passes(told, monkeypatch, budget):
    model, prompts, texts = told
    monkeypatch.setattr(example, "guess", _guesses(texts, lambda t: t))
    got, passes, evictions = example.answer(model, prompts, TOKENS, drafts=DRAFTS, budget=budget)
    assert passes < TOKENS and evictions == 0
    _are_its_own(model, prompts, got)


@pytest.mark.parametrize("budget", [None, 200])
def test_wrong_guesses_change_nothing(told, monkeypatch, budget):
    model, prompts, texts = told
    monkeypatch.setattr(example, "guess", _guesses(texts, lambda t: (t + 1) % 2048))
    got, passes, evictions = example.answer(model, prompts, TOKENS, drafts=DRAFTS, budget=budget)
    assert passes <= TOKENS and evictions == 0
    _are_its_own(model, prompts, got)


def test_a_wrong_token_is_seen(told):
    """The check itself: one token changed is outside it."""
    model, prompts, texts = told
    bad = [list(t) for t in texts]
    bad[1][len(prompts[1]) + 20] = (bad[1][len(prompts[1]) + 20] + 1) % 2048
    with pytest.raises(AssertionError):
        _are_its_own(model, prompts, bad)
