"""The best continuations of beams, from logits and running scores (beam search).

No counterpart in the reference, which trains only.  ``kernels.paged.fork_kv`` moves the
cache's sequences along.  Scores are fp64 from the logits' sum on (csrc/beam_select.hip says
why), logits fp16, bf16 or fp32.
"""

import torch

from .. import _lib, native
from ..contract import Rule, enforce

_CODES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}

SELECT_RULES = (
    Rule("select_beams: logits must be fp16, bf16 or fp32 [rows, beams, vocab] with a unit last "
         "stride, without gradients",
         lambda a: isinstance(a.logits, torch.Tensor) and a.logits.ndim == 3
         and a.logits.dtype in _CODES and 0 < a.logits.shape[2] < 2 ** 31 - 65536
         and (a.logits.stride(2) == 1 or a.logits.shape[2] == 1) and not a.logits.requires_grad),
    Rule("select_beams: at most 64 beams and 65535 rows",
         lambda a: 0 < a.logits.shape[1] <= 64 and a.logits.shape[0] <= 65535),
    Rule("select_beams: scores must be a contiguous fp32 [rows, beams]",
         lambda a: isinstance(a.scores, torch.Tensor) and a.scores.dtype == torch.float32
         and a.scores.shape == a.logits.shape[:2] and a.scores.is_contiguous()),
    Rule("select_beams: count must be a whole number from 1 to 64, at most beams * vocab, and "
         "beams * count at most 2048",
         lambda a: isinstance(a.count, int) and not isinstance(a.count, bool)
         and 0 < a.count <= min(64, a.logits.shape[1] * a.logits.shape[2])
         and a.logits.shape[1] * a.count <= 2048),
    Rule("select_beams: logits and scores must be CUDA tensors on one device",
         lambda a: a.logits.is_cuda and a.scores.device == a.logits.device),
)


def select_beams(logits, scores, count):
    """The ``count`` best of every row's beams x vocabulary: (scores fp32, parents int32, tokens
    int64), each [rows, count], best first.

    ``logits`` [rows, beams, vocab] follow the beams' texts, ``scores`` [rows, beams] are the sums
    of their tokens' log-probabilities so far (-inf for a beam that is not there: all but one at the
    first step).  A candidate's score is its beam's plus the token's log-probability, NaN counting as -inf.
    Of equal ones the lower beam comes first, then the greater logit, then the lower token.
    """
    nodes = native.nodes()
    if nodes is not None:
        got = nodes.select_beams(logits, scores, count)
        if got is not None:
            return got
    enforce(SELECT_RULES, logits=logits, scores=scores, count=count)
    rows, beams, vocab = logits.shape
    device = logits.device
    out = torch.empty((rows, count), dtype=torch.float32, device=device)
    parents = torch.empty((rows, count), dtype=torch.int32, device=device)
    tokens = torch.empty((rows, count), dtype=torch.int64, device=device)
    if rows == 0:
        return out, parents, tokens
    code = _CODES[logits.dtype]
    size = _lib.load().ss_select_beams_workspace_size(rows, beams, vocab, count, code)
    with torch.cuda.device(device):
        scratch = torch.empty(size, dtype=torch.uint8, device=device)
        _lib.call("ss_select_beams", logits.data_ptr(), logits.stride(0), logits.stride(1), code,
                  scores.data_ptr(), rows, beams, vocab, count, out.data_ptr(),
                  parents.data_ptr(), tokens.data_ptr(), scratch.data_ptr(), size,
                  _lib.stream(device))
    return out, parents, tokens
