"""The loop of examples/answer.py on the CPU: a model of one rule (the next token follows from the
last one), no layers, and the oracle in place of the draft check."""

import pytest
import torch

import examples.answer as example
from oracle import cache as ocache
from tests.cache_util import offsets

VOCAB = 512


def _next(token):
    """1, 2, 3 in a circle, which the text so far tells; the others count up."""
    return token % 3 + 1 if token <= 3 else token + 1


class Rule:
    embedding, kv_heads, layers = torch.zeros((VOCAB, 1)), 2, []

    def __call__(self, tokens, attend):
        return torch.nn.functional.one_hot(torch.tensor([_next(t) for t in tokens.tolist()]),
                                           VOCAB).float()


@pytest.fixture(autouse=True)
def checked(monkeypatch):
    def verify(target, tokens, uniform, draft_counts, temperature):
        got = [ocache.verify(target[b].double().numpy(), tokens[b].tolist(), uniform[b].tolist(),
                             None, int(draft_counts[b]), temperature)
               for b in range(target.shape[0])]
        return torch.tensor([n for n, _ in got]), torch.tensor([t for _, t in got])

    monkeypatch.setattr(example, "verify_drafts", verify)
    monkeypatch.setattr(example, "row_offsets", offsets)       # the package's is in pinned memory


def _expected(prompt, tokens):
    text = list(prompt)
    for _ in range(tokens):
        text.append(_next(text[-1]))
    return text


@pytest.mark.parametrize("drafts", [0, 1, 4])
@pytest.mark.parametrize("tokens", [1, 7, 40])
def test_rows_that_go_on_at_different_rates(tokens, drafts):
    """One row's guesses are always right, the others have none: the first has its tokens long
    before them."""
    prompts = [[1, 2, 3, 1, 2], [10, 11, 12], [100], list(range(200, 260))]
    texts, passes, evictions = example.answer(Rule(), prompts, tokens, drafts=drafts)
    assert texts == [_expected(p, tokens) for p in prompts]
    assert passes == tokens and evictions == 0


def test_right_guesses_save_passes():
    prompts = [[1, 2, 3, 1, 2], [3, 1, 2, 3]]
    texts, passes, _ = example.answer(Rule(), prompts, 40, drafts=4)
    assert texts == [_expected(p, 40) for p in prompts]
    assert passes < 40


@pytest.mark.parametrize("prompts", [[], [[]], [[1, 2], []], [[], [5]]])
def test_prompts_without_a_token_are_refused(prompts):
    """There is no row of logits behind them; another sequence's must not answer for them."""
    with pytest.raises(ValueError, match="at least one token"):
        example.answer(Rule(), prompts, 3)
