"""Drafted tokens checked against the target model's logits (speculative decoding).

No counterpart in the reference, which trains only.  The random numbers are inputs, so a
call is a function of its arguments; probabilities and running sums are fp64
(csrc/verify.hip says why), logits fp16, bf16 or fp32.
"""

import torch

from .. import _lib, native
from ..contract import Rule, enforce, finite_real

_CODES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _logits(t, dtype, shape):
    return (isinstance(t, torch.Tensor) and t.dtype == dtype and t.shape == shape
            and (t.stride(-1) == 1 or t.shape[-1] == 1))


VERIFY_RULES = (
    Rule("verify_drafts: target_logits must be fp16, bf16 or fp32 [rows, drafts + 1, vocab] with "
         "a unit last stride",
         lambda a: isinstance(a.target, torch.Tensor) and a.target.ndim == 3
         and a.target.dtype in _CODES and a.target.shape[1] > 0 and 0 < a.target.shape[2] < 2 ** 31
         - 8192 and _logits(a.target, a.target.dtype, a.target.shape)),
    Rule("verify_drafts: draft_tokens must be a contiguous int64 [rows, drafts]",
         lambda a: isinstance(a.tokens, torch.Tensor) and a.tokens.dtype == torch.int64
         and a.tokens.shape == (a.target.shape[0], a.target.shape[1] - 1)
         and a.tokens.is_contiguous()),
    Rule("verify_drafts: temperature must be a finite number from 0 up",
         lambda a: finite_real(a.temperature, 0.0)),
    Rule("verify_drafts: uniform must be a contiguous fp32 [rows, drafts + 1] (None only at "
         "temperature 0)",
         lambda a: (a.uniform is None and a.temperature == 0)
         or (isinstance(a.uniform, torch.Tensor) and a.uniform.dtype == torch.float32
             and a.uniform.shape == a.target.shape[:2] and a.uniform.is_contiguous())),
    Rule("verify_drafts: draft_logits must be [rows, drafts, vocab] of the target's type with a "
         "unit last stride",
         lambda a: a.draft is None or _logits(
             a.draft, a.target.dtype, (*a.tokens.shape, a.target.shape[2]))),
    Rule("verify_drafts: draft_counts must be a contiguous int32 [rows]",
         lambda a: a.counts is None or (
             isinstance(a.counts, torch.Tensor) and a.counts.dtype == torch.int32
             and a.counts.shape == a.target.shape[:1] and a.counts.is_contiguous())),
    Rule("verify_drafts: at most 65535 rows of logits in one call",
         lambda a: a.target.shape[0] * (2 * a.target.shape[1] - 1) <= 65535),
    Rule("verify_drafts: all tensors must be CUDA tensors on one device",
         lambda a: a.target.is_cuda and all(t is None or t.device == a.target.device
                                            for t in (a.tokens, a.uniform, a.draft, a.counts))),
)


def verify_drafts(target_logits, draft_tokens, uniform=None, draft_logits=None, draft_counts=None,
                  temperature=1.0):
    """Accept drafted tokens and draw the next one; returns (accepted int32 [rows], tokens int64
    [rows, drafts + 1]: the accepted drafts, the next token, then -1).

    ``target_logits`` [rows, drafts + 1, vocab]: row i follows the first i drafted tokens.
    ``draft_logits`` [rows, drafts, vocab] are those the drafts were drawn from; None means that
    drafts were not drawn (looked up, or the draft model's best): q is 1 on the drafted token.
    ``uniform`` [rows, drafts + 1] in [0, 1): one number for each draft and the last one for the
    next token.  ``draft_counts`` [rows] says how many of the drafts a row has (None: all).
    Draft i is accepted while u_i q(x_i) < p(x_i); the next token is drawn from max(p - q, 0) at
    the first refusal, else from p behind the last draft.  ``temperature`` divides both logits;
    0 compares with the target's largest logit (the lowest token of equal ones).
    """
    nodes = native.nodes()
    if nodes is not None:
        got = nodes.verify_drafts(target_logits, draft_tokens, uniform, draft_logits, draft_counts,
                                  temperature)
        if got is not None:
            return got
    enforce(VERIFY_RULES, target=target_logits, tokens=draft_tokens, uniform=uniform,
            draft=draft_logits, counts=draft_counts, temperature=temperature)
    rows, length, vocab = target_logits.shape
    device = target_logits.device
    accepted = torch.empty(rows, dtype=torch.int32, device=device)
    out = torch.empty((rows, length), dtype=torch.int64, device=device)
    if rows == 0:
        return accepted, out
    drafted = draft_logits is not None and length > 1
    size = _lib.load().ss_verify_drafts_workspace_size(rows, length - 1, vocab, drafted)
    with torch.cuda.device(device):
        scratch = torch.empty(size, dtype=torch.uint8, device=device)
        _lib.call("ss_verify_drafts", target_logits.data_ptr(), target_logits.stride(0),
                  target_logits.stride(1),
                  *((draft_logits.data_ptr(), draft_logits.stride(0), draft_logits.stride(1))
                    if drafted else (None, 0, 0)),
                  _CODES[target_logits.dtype], draft_tokens.data_ptr(), _lib.ptr(draft_counts),
                  _lib.ptr(uniform), rows, length - 1, vocab, float(temperature),
                  accepted.data_ptr(), out.data_ptr(), scratch.data_ptr(), size,
                  _lib.stream(device))
    return accepted, out
