"""The target model's key-value cache in pages, and attention over it.

The packed draft cache of this package serves the draft model; a round of
speculative decoding ends at the target model, whose sequences accept
different numbers of drafted tokens.  Their keys and values live in pages of
a few tokens that a block table assigns to the sequences, so every sequence
has a length of its own.  (The reference has no counterpart: it leaves the
target's cache to transformers, one sequence at a time,
kv_reduce/experiments/packed_review.py:101-137.)

    key_pages, value_pages  [num_pages, kv_heads, page_size, head_dim]  bf16 or fp16, any order in memory
    block_table             int32 [batch, max_pages], token j of sequence b in page block_table[b, j // page_size]
    lengths                 int32 [batch], on the device; the new tokens of a step are already counted

All compute runs in libkvr.so through the C++ operators
torch.ops.kvr.paged_*; the host never reads the lengths, so the calls can be
captured in a CUDA graph.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

_append_op = None
_attention_op = None
_evict_op = None


def _bind_ops() -> None:
    global _append_op, _attention_op, _evict_op
    _lib.load_torch_ops()
    _append_op = torch.ops.kvr.paged_append.default
    _attention_op = torch.ops.kvr.paged_attention.default
    _evict_op = torch.ops.kvr.paged_evict.default


def paged_append(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                 block_table: torch.Tensor, lengths: torch.Tensor) -> None:
    """Write the newest T tokens' key and value [batch, kv_heads, T, head_dim]
    into their pages, at positions ``lengths - T .. lengths - 1`` (the lengths
    already count them).  Positions below 0, and rows whose page number is not
    in the pool, are skipped."""
    if _append_op is None:
        _bind_ops()
    _append_op(key, value, key_pages, value_pages, block_table, lengths)


def paged_decode_attention(
    query: torch.Tensor,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: Optional[float] = None,
    window: int = 0,
    sinks: int = 0,
    token_weights: Optional[torch.Tensor] = None,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of the newest T tokens of every sequence over its pages.

    ``query`` is [batch, query_heads, T, head_dim]: one token in a plain
    decode step, the last accepted and the drafted tokens in a verification.
    Query t stands at ``i = lengths - T + t`` and sees the tokens ``j <= i``;
    with ``window > 0`` only those with ``j > i - window``, and the first
    ``sinks`` tokens.  ``scale`` defaults to ``head_dim ** -0.5``.

    ``token_weights`` (fp32 [batch, >= max_pages * page_size]): the weight
    that each cached token got, summed over heads and queries, is added to it.

    Returns the output like ``query`` (contiguous), and with ``return_lse``
    the natural log of the softmax sums, fp32 [batch, query_heads, T].  A
    query that sees no token gives zeros and -inf.  A sequence longer than
    its block table, or with a page number outside the pool among the tokens
    it sees, gives NaN.
    """
    if _attention_op is None:
        _bind_ops()
    out, lse = _attention_op(query, key_pages, value_pages, block_table, lengths, scale, window, sinks, token_weights,
                             return_lse)
    return (out, lse) if return_lse else out


def paged_evict(
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    token_weights: torch.Tensor,
    new_block_table: torch.Tensor,
    *,
    keep: int,
    recent: int = 0,
    first: int = 0,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Bring every sequence down to ``keep`` tokens by accumulated weight.

    A sequence longer than ``keep`` keeps its first ``first`` tokens, its last
    ``recent`` ones and the heaviest of those between by ``token_weights``
    (ties: the lowest position; NaN counts as heaviest); a shorter one keeps
    all.  The kept rows are copied, in order, into the pages of
    ``new_block_table`` (int32 [batch, pages]), which must be free: not pages
    that a block table still uses.  Pages that sequences share stay whole.

    Returns ``kept`` (int32 [batch, keep], old positions, -1 behind the last),
    the new lengths (int32 [batch]) and the kept tokens' weights (fp32
    [batch, keep], 0 behind the last).  The keys keep the rotary positions
    they were written with.
    """
    if _evict_op is None:
        _bind_ops()
    return _evict_op(key_pages, value_pages, block_table, lengths, token_weights, new_block_table, keep, recent, first)
