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

from typing import List, Optional, Sequence, Tuple, Union

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
                 block_table: torch.Tensor, lengths: torch.Tensor, new_counts: Optional[torch.Tensor] = None) -> None:
    """Write the newest T tokens' key and value [batch, kv_heads, T, head_dim]
    into their pages, at positions ``lengths - T .. lengths - 1`` (the lengths
    already count them).  Positions below 0, and rows whose page number is not
    in the pool, are skipped.

    ``new_counts`` (int32 [batch]): sequences with fewer new tokens than T.
    Theirs are the last ``new_counts[b]`` of the T; the rows before are padding
    and are not written."""
    if _append_op is None:
        _bind_ops()
    _append_op(key, value, key_pages, value_pages, block_table, lengths, new_counts)


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
    new_counts: Optional[torch.Tensor] = None,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of the newest T tokens of every sequence over its pages.

    ``query`` is [batch, query_heads, T, head_dim]: one token in a plain
    decode step, the last accepted and the drafted tokens in a verification.
    Query t stands at ``i = lengths - T + t`` and sees the tokens ``j <= i``;
    with ``window > 0`` only those with ``j > i - window``, and the first
    ``sinks`` tokens.  ``scale`` defaults to ``head_dim ** -0.5``.

    ``token_weights`` (fp32 [batch, >= max_pages * page_size]): the weight
    that each cached token got, summed over heads and queries, is added to it.

    ``new_counts`` (int32 [batch]): sequences with fewer new tokens than T.
    Their queries are the last ``new_counts[b]`` of the T; those before are
    padding, see nothing and add no weight.

    Returns the output like ``query`` (contiguous), and with ``return_lse``
    the natural log of the softmax sums, fp32 [batch, query_heads, T].  A
    query that sees no token gives zeros and -inf.  A sequence longer than
    its block table, or with a page number outside the pool among the tokens
    it sees, gives NaN.
    """
    if _attention_op is None:
        _bind_ops()
    out, lse = _attention_op(query, key_pages, value_pages, block_table, lengths, scale, window, sinks, token_weights,
                             return_lse, new_counts)
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


class PagedKVCache:
    """A model's key-value cache in pages: pools for every layer, one block
    table and one set of lengths for all of them.

    The host keeps the lengths too, to hand out and take back pages; a step is

        cache.advance(T)                      # once: pages and lengths for T more tokens
        cache.append(layer, k, v)             # every layer: [batch, kv_heads, T, head_dim]
        out = cache.attention(layer, q)       # [batch, query_heads, T, head_dim]
        cache.crop(lengths)                   # after a verification: each sequence to its own length

    With ``track_weights`` the attention adds up what weight every token got
    (per layer), and ``evict`` brings the sequences down to a budget by it.
    The totals are those of all queries that ``attention`` was called with:
    ``crop`` forgets the removed tokens' own totals, but what their queries
    added to the tokens before them stays (drafted tokens that a verification
    refused have voted), and an attention that did not run here, a prompt's
    say, has not been counted.

    ``max_pages``: pages a sequence may come to, the table's width (default:
    the whole pool).  The table and the weights take batch * max_pages entries
    and are kept on the host too, so in a large pool give it.
    """

    def __init__(self, num_layers: int, batch: int, kv_heads: int, head_dim: int, *, num_pages: int,
                 page_size: int = 16, max_pages: Optional[int] = None, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda", track_weights: bool = False) -> None:
        if min(num_layers, batch, kv_heads, head_dim, num_pages, page_size) <= 0:
            raise ValueError("num_layers, batch, kv_heads, head_dim, num_pages and page_size must be positive.")
        self.batch, self.page_size, self.num_pages = int(batch), int(page_size), int(num_pages)
        # a sequence's share of the block table (default: all pages could be one sequence's)
        self.max_pages = int(max_pages or num_pages)
        self.device = torch.device(device)
        shape = (self.num_pages, kv_heads, self.page_size, head_dim)
        self.key_pages = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(num_layers)]
        self.value_pages = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(num_layers)]
        self.block_table = torch.full((self.batch, self.max_pages), -1, dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(self.batch, dtype=torch.int32, device=self.device)
        self.token_weights: Optional[List[torch.Tensor]] = None
        if track_weights:
            self.token_weights = [torch.zeros(self.batch, self.max_pages * self.page_size, device=self.device)
                                  for _ in range(num_layers)]
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(self.batch)]
        self._lengths = [0] * self.batch
        self._width = 0      # pages of the longest sequence
        # what advance gave each sequence, whether that differed, whether a step has used it, and the counts that the
        # device has
        self._new, self._ragged, self._used = [0] * self.batch, False, True
        self.new_counts = torch.zeros(self.batch, dtype=torch.int32, device=self.device)
        self._counts_of = list(self._new)

    # ------------------------------------------------------------- lengths
    def get_seq_length(self) -> int:
        """Tokens of the longest sequence."""
        return max(self._lengths)

    def seq_lengths(self) -> List[int]:
        return list(self._lengths)

    def free_pages(self) -> int:
        return len(self._free)

    def _upload(self, table: bool) -> None:
        if table:
            rows = [p + [-1] * (self.max_pages - len(p)) for p in self._pages]
            self.block_table.copy_(torch.tensor(rows, dtype=torch.int32))
        self.lengths.copy_(torch.tensor(self._lengths, dtype=torch.int32))
        self._width = max(len(p) for p in self._pages)

    def advance(self, tokens: Union[int, Sequence[int]]) -> None:
        """Lengthen the sequences (by one number, or one each) and give them
        pages; the rows are written by ``append``.  Where the numbers differ,
        ``append`` and ``attention`` take the largest as T and each sequence's
        new tokens as the last of the T.  Numbers given before the rows were
        written add up."""
        more = [int(tokens)] * self.batch if isinstance(tokens, int) else [int(t) for t in tokens]
        if len(more) != self.batch or min(more) < 0:
            raise ValueError(f"advance needs a number of tokens >= 0 for each of {self.batch} sequences.")
        need = [-(-(n + m) // self.page_size) - len(p) for n, m, p in zip(self._lengths, more, self._pages)]
        if sum(max(n, 0) for n in need) > len(self._free):
            raise ValueError("not enough free pages: crop, evict or make the cache with more.")
        if any(len(p) + n > self.max_pages for p, n in zip(self._pages, need)):
            raise ValueError("a sequence needs more than max_pages pages.")
        for pages, n in zip(self._pages, need):
            pages.extend(self._free.pop() for _ in range(n))
        self._lengths = [n + m for n, m in zip(self._lengths, more)]
        if not self._used:       # rows made room for earlier and not written yet
            more = [n + m for n, m in zip(self._new, more)]
        self._new, self._ragged, self._used = more, min(more) != max(more), False
        self._upload(any(n > 0 for n in need))

    def crop(self, lengths: Union[int, Sequence[int]]) -> None:
        """Roll every sequence back to its length; pages behind it are free again."""
        to = [min(int(lengths), n) for n in self._lengths] if isinstance(lengths, int) else [int(n) for n in lengths]
        if len(to) != self.batch or any(not 0 <= t <= n for t, n in zip(to, self._lengths)):
            raise ValueError(f"crop needs a length within each of the {self.batch} sequences.")
        freed = False
        for b, t in enumerate(to):
            keep = -(-t // self.page_size)
            freed |= keep < len(self._pages[b])
            self._free.extend(reversed(self._pages[b][keep:]))
            del self._pages[b][keep:]
            if self.token_weights is not None and t < self._lengths[b]:
                for w in self.token_weights:
                    w[b, t:self._lengths[b]] = 0
        self._new = [max(0, m - (n - t)) for m, n, t in zip(self._new, self._lengths, to)]
        self._lengths = to
        self._upload(freed)

    # ---------------------------------------------------------- operations
    def _counts(self) -> torch.Tensor:
        """``_new`` on the device."""
        if self._counts_of != self._new:
            self.new_counts.copy_(torch.tensor(self._new, dtype=torch.int32))
            self._counts_of = list(self._new)
        return self.new_counts

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Write the tokens that ``advance`` made room for: key and value
        [batch, kv_heads, T, head_dim], T the most that a sequence was given,
        each sequence's own the last of them."""
        if key.shape[2] > max(self._new):
            raise ValueError(f"append takes the {max(self._new)} tokens that advance made room for, not {key.shape[2]}.")
        self._used = True
        paged_append(key, value, self.key_pages[layer], self.value_pages[layer], self.block_table, self.lengths,
                     self._counts() if min(self._new) < key.shape[2] else None)

    def attention(self, layer: int, query: torch.Tensor, *, scale: Optional[float] = None, window: int = 0,
                  sinks: int = 0) -> torch.Tensor:
        """Attention of the newest T tokens, query [batch, query_heads, T,
        head_dim].  After an ``advance`` by different numbers the queries of a
        sequence are its new tokens' only, the last of the T; the outputs
        before them are zeros."""
        self._used = True
        weights, table = None, self.block_table
        if self.token_weights is not None:
            weights = self.token_weights[layer]
            # the scores' memory goes by the table's width: the columns in use.  (A captured step keeps all of them:
            # its sequences may be longer when it is replayed.)
            if not (self.device.type == "cuda" and torch.cuda.is_current_stream_capturing()):
                table = table[:, :self._width]
        return paged_decode_attention(query, self.key_pages[layer], self.value_pages[layer], table, self.lengths,
                                      scale=scale, window=window, sinks=sinks, token_weights=weights,
                                      new_counts=self._counts() if self._ragged else None)

    def evict(self, keep: int, *, recent: int = 0, first: int = 0) -> bool:
        """Bring every sequence down to ``keep`` tokens (see ``paged_evict``),
        each layer by its own weights; the rows move to fresh pages.  False,
        and nothing done, while no sequence is longer.  Tokens that no counted
        query has seen weigh 0, and of equal weights the first are kept: call
        it once a few steps have run over a prompt, or with ``recent``."""
        if self.token_weights is None:
            raise ValueError("evict needs a cache made with track_weights=True.")
        if keep <= 0 or recent < 0 or first < 0 or first + recent > keep:
            raise ValueError("keep must be positive and hold first + recent tokens.")
        if max(self._lengths) <= keep:
            return False
        left = [min(n, keep) for n in self._lengths]
        need = [-(-n // self.page_size) for n in left]
        if sum(need) > len(self._free):
            raise ValueError("not enough free pages to evict into.")
        # (the pages leave the free list, and the weights change, once every layer's call has been accepted)
        spare = iter(self._free[:-sum(need) - 1:-1])
        fresh = [[next(spare) for _ in range(n)] for n in need]
        width = -(-keep // self.page_size)
        rows = [p + [-1] * (width - len(p)) for p in fresh]
        new_table = torch.tensor(rows, dtype=torch.int32).to(self.device)
        # the columns in use: the operator's limit is on the table's width, and a pool may be far wider than a sequence
        table = self.block_table[:, :self._width]
        kept = [paged_evict(self.key_pages[layer], self.value_pages[layer], table, self.lengths, weights, new_table,
                            keep=keep, recent=recent, first=first)[2]
                for layer, weights in enumerate(self.token_weights)]
        for weights, w in zip(self.token_weights, kept):
            n = min(keep, weights.shape[1])
            weights.zero_()
            weights[:, :n].copy_(w[:, :n])
        del self._free[-sum(need):]
        for pages in self._pages:
            self._free.extend(reversed(pages))
        self._pages, self._lengths = fresh, left
        self._new, self._ragged, self._used = [0] * self.batch, False, True
        self._upload(True)
        return True
