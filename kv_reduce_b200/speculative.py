"""Verification of drafted tokens against the target model's probabilities.

A round of speculative decoding ends here: the target model has scored the
drafted tokens in one forward, and the longest accepted run of them and one
more token are taken over.  (The reference compares the target's argmax on
the host, kv_reduce/experiments/packed_review.py:101-137; sampling with the
acceptance rule min(1, p/q) is an addition.)
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

_verify_op = None


class VerifyResult(NamedTuple):
    tokens: torch.Tensor        # int64 [batch, draft + 1]: accepted tokens, the new one, then -1
    accepted: torch.Tensor      # int32 [batch]: drafted tokens accepted
    accept_prob: torch.Tensor   # fp32 [batch, draft]: min(1, p / q), 0 behind the first refusal


def verify_draft_tokens(
    target_logits: torch.Tensor,
    draft_logits: Optional[torch.Tensor],
    draft_tokens: torch.Tensor,
    uniforms: Optional[torch.Tensor] = None,
    noise: Optional[torch.Tensor] = None,
    *,
    temperature: float = 1.0,
    draft_lengths: Optional[torch.Tensor] = None,
) -> VerifyResult:
    """Accept drafted tokens and draw the next one.

    With ``p = softmax(target_logits / temperature)`` and ``q`` likewise from
    the draft's, token ``x_k`` is accepted while ``uniforms[k] < min(1,
    p_k(x_k) / q_k(x_k))``.  At the first refusal j the next token is the
    argmax of ``max(p_j - q_j, 0) / noise``, after a full acceptance that of
    ``p_K / noise``: with ``noise`` exponentially distributed that is a draw
    from the distribution (ties: the lowest index), and the tokens are
    distributed as the target's own samples.  Logits of -inf (top-k or top-p
    filters) are tokens of no weight.

    ``temperature=0`` accepts a token while it is the target's argmax; the
    draft's logits, uniforms and noise are not used then (None).

    target_logits [batch, draft + 1, vocab] and draft_logits [batch, draft,
    vocab]: bf16, fp16 or fp32; draft_tokens [batch, draft] int64 or int32;
    uniforms fp32 [batch, draft] in [0, 1); noise fp32 [batch, vocab] > 0;
    draft_lengths int32 [batch]: how many positions each sequence drafted
    (default: all).  A row without any weight gives the token -1.
    """
    global _verify_op
    if _verify_op is None:
        _lib.load_torch_ops()
        _verify_op = torch.ops.kvr.verify_draft.default
    return VerifyResult(*_verify_op(target_logits, draft_logits, draft_tokens, uniforms, noise, temperature,
                                    draft_lengths))
