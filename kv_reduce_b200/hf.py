"""Integration with transformers: a packed Cache for the draft model, a
paged one for the target model, their attention hooks, and a generation
loop that runs both.

Mirrors kv_reduce/experiments/packed_review.py:17-80:

* ``PackedDraftCache`` plays the role of the reference's ``PackedCache``
  (a ``DynamicCache`` whose layers hold the packed K/V; :56-63), built from a
  prefilled cache, with ``commit()`` (promote full key groups out of the
  BF16 residual window, :32-41, :61-62) and ``breakdown()`` (:50-54, :63).
  Its layers are the preallocated streaming layers of
  ``kv_reduce_b200.streaming``, so a decode step appends one token in place
  instead of the reference's ``torch.cat`` of the whole payload.
* ``PackedDraftCache.empty(num_layers, residual)`` packs each layer during
  the prompt forward itself (streaming prefill): the full BF16 cache the
  reference builds first and packs afterwards never exists.
* ``install(model)`` patches every decoder layer's attention (:65-80): with
  a ``PackedDraftCache`` and a one-token step, it projects q/k/v, applies the
  rotary embedding and runs ``decode_step`` on the packed layer (append
  in place + fused decode, two library calls from device-side lengths); any
  other call goes to the original forward.

The target's side has no counterpart in the reference (it runs the target
on transformers' own cache, packed_review.py:101-137):

* ``PagedTargetCache`` holds the target's K/V in pages
  (``kv_reduce_b200.paged``); ``install_target(model)`` routes the attention
  of steps over it through ``paged_decode_attention``, the last accepted and
  the drafted tokens at once.
* ``speculative_generate`` drafts with the packed cache, scores with the
  paged one and verifies with ``verify_draft_tokens``.

Written against the Qwen2 attention module of transformers 5.x (q/k/v/o
projections, ``head_dim``, ``layer_idx``, rotary ``position_embeddings``).
"""
from __future__ import annotations

import types
from typing import Dict, Iterable, List, Optional, Tuple

import torch
from transformers.cache_utils import DynamicCache, DynamicLayer
from transformers.models.qwen2.modeling_qwen2 import apply_rotary_pos_emb

from .paged import PagedKVCache
from .speculative import verify_draft_tokens
from .streaming import PackedKVCacheLayer, PackedLayer


class PackedDraftLayer(DynamicLayer):
    """A transformers cache layer over one streaming packed layer.

    Built over an already packed layer, or empty: then the prompt forward's
    ``update`` packs the layer's K/V as soon as they are produced (streaming
    prefill) and passes the BF16 tensors on to that layer's attention only,
    so the model never holds a BF16 copy of more than one layer's cache.
    """

    def __init__(self, packed: PackedKVCacheLayer | None = None, *, residual: int = 128,
                 spare_capacity: int = 2048, **kw) -> None:
        super().__init__()
        self.packed = packed
        self._residual, self._spare, self._kw = int(residual), int(spare_capacity), kw
        self.is_initialized = True

    def get_seq_length(self) -> int:
        return 0 if self.packed is None else self.packed.get_seq_length()

    def get_mask_sizes(self, query_length: int) -> Tuple[int, int]:
        return self.get_seq_length() + int(query_length), 0

    def crop(self, max_length: int) -> None:
        # transformers semantics: a negative length removes tokens from the end
        n = self.get_seq_length()
        self.packed.crop(n + max_length if max_length < 0 else min(max_length, n))

    def update(self, key_states, value_states, *args, **kwargs):
        if self.get_seq_length() == 0:
            # streaming prefill: pack this layer now (pack_kivi_kv semantics)
            B, H, S, D = (int(x) for x in key_states.shape)
            if self.packed is None:
                self.packed = PackedKVCacheLayer(B, H, D, residual_length=self._residual,
                                                 capacity=S + self._spare, device=key_states.device, **self._kw)
            self.packed.prefill(key_states, value_states)
            return key_states, value_states
        raise RuntimeError("a packed draft cache is extended by the installed attention hook, one token per step "
                           "(call kv_reduce_b200.hf.install(model) first)")


def _legacy_pairs(cache) -> Iterable[Tuple[torch.Tensor, torch.Tensor]]:
    if isinstance(cache, DynamicCache):
        return [(layer.keys, layer.values) for layer in cache.layers]
    return list(cache)


class PackedDraftCache(DynamicCache):
    """Packed draft cache built from a prefilled cache (a ``DynamicCache`` or
    (k, v) pairs of [B, H, S, D] bf16 per layer)."""

    def __init__(self, cache, residual: int, **kw) -> None:
        super().__init__()
        self.layers = [PackedDraftLayer(PackedLayer(k, v, residual, **kw)) for k, v in _legacy_pairs(cache)]

    @classmethod
    def empty(cls, num_layers: int, residual: int, *, spare_capacity: int = 2048, **kw) -> "PackedDraftCache":
        """A cache to run the prompt forward into: each layer is packed as the
        forward produces it (streaming prefill), then decoded through the hook.
        ``kw`` are PackedKVCacheLayer options (k_bits, v_bits, group_size)."""
        self = cls([], residual)
        self.layers = [PackedDraftLayer(None, residual=residual, spare_capacity=spare_capacity, **kw)
                       for _ in range(int(num_layers))]
        return self

    def commit(self) -> None:
        for layer in self.layers:
            if layer.packed is not None:
                layer.packed.commit()

    def breakdown(self) -> Dict[str, int]:
        parts = [layer.packed.breakdown() for layer in self.layers if layer.packed is not None]
        return {key: sum(p[key] for p in parts) for key in parts[0]}


def install(model, *, split_tokens: int = 0) -> None:
    """Route one-token attention steps over a ``PackedDraftCache`` through the
    packed decode kernel (packed_review.py:65-80).  ``split_tokens`` is
    passed to the kernel (0: the library's split plan; the reference used
    512)."""
    for layer in model.model.layers:
        attn = layer.self_attn
        original = attn.forward

        def forward(self, hidden_states, position_embeddings, attention_mask, past_key_values=None,
                    _original=original, **kwargs):
            if (not isinstance(past_key_values, PackedDraftCache)
                    or past_key_values.layers[self.layer_idx].get_seq_length() == 0):
                # other caches, and the prompt forward of an empty packed cache
                # (its update() packs the layer: streaming prefill)
                return _original(hidden_states, position_embeddings, attention_mask, past_key_values, **kwargs)
            if hidden_states.shape[1] != 1:
                raise ValueError("the packed draft cache decodes one token per step")
            shape = hidden_states.shape[:-1]
            view = (*shape, -1, self.head_dim)
            q = self.q_proj(hidden_states).view(view).transpose(1, 2)
            k = self.k_proj(hidden_states).view(view).transpose(1, 2)
            v = self.v_proj(hidden_states).view(view).transpose(1, 2)
            q, k = apply_rotary_pos_emb(q, k, *position_embeddings)
            packed = past_key_values.layers[self.layer_idx].packed
            out = packed.decode_step(q, k, v, split_tokens=split_tokens)
            return self.o_proj(out.transpose(1, 2).reshape(*shape, -1).contiguous()), None

        attn.forward = types.MethodType(forward, attn)


class PagedTargetLayer(DynamicLayer):
    """One layer's view of a ``PagedTargetCache``."""

    def __init__(self, cache: "PagedTargetCache", index: int) -> None:
        super().__init__()
        self._cache, self._index = cache, index
        self.is_initialized = True

    def get_seq_length(self) -> int:
        return self._cache.pages.get_seq_length()

    def get_mask_sizes(self, query_length: int) -> Tuple[int, int]:
        return self.get_seq_length() + int(query_length), 0

    def crop(self, max_length: int) -> None:
        raise RuntimeError("crop the PagedTargetCache: its layers share their lengths")

    def update(self, key_states, value_states, *args, **kwargs):
        # the prompt: its keys and values go to the pages, its attention is the model's own
        if self._index == 0:
            if self._cache.pages.get_seq_length() > 0:
                raise RuntimeError("a paged target cache is extended by the installed attention hook "
                                   "(call kv_reduce_b200.hf.install_target(model) first)")
            self._cache.pages.advance(int(key_states.shape[2]))
        self._cache.pages.append(self._index, key_states, value_states)
        return key_states, value_states


class PagedTargetCache(DynamicCache):
    """The target model's cache in pages.  ``max_tokens``: what each sequence
    may hold; with ``keep`` the cache is brought back to that many tokens, the
    ``first`` ones, the ``recent`` ones and the heaviest of the others, by
    ``evict()``.  ``window`` and ``sinks`` restrict the attention of the steps
    after the prompt.

    A token's weight is what the steps' queries gave it, those of refused
    drafts among them.  The prompt's own attention runs in the model and is
    not counted: an eviction right after the first step ranks the prompt by
    that step's few queries alone, so leave ``recent`` room, or evict after
    some steps."""

    def __init__(self, num_layers: int, batch: int, kv_heads: int, head_dim: int, *, max_tokens: int,
                 page_size: int = 16, dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda",
                 window: int = 0, sinks: int = 0, keep: int = 0, recent: int = 0, first: int = 0) -> None:
        super().__init__()
        per_seq = -(-int(max_tokens) // page_size)
        spare = -(-int(keep) // page_size) if keep else 0      # an eviction's fresh pages
        self.pages = PagedKVCache(num_layers, batch, kv_heads, head_dim, num_pages=batch * (per_seq + spare),
                                  page_size=page_size, max_pages=per_seq, dtype=dtype, device=device,
                                  track_weights=keep > 0)
        self.window, self.sinks = int(window), int(sinks)
        self.keep, self.recent, self.first = int(keep), int(recent), int(first)
        self.layers = [PagedTargetLayer(self, i) for i in range(num_layers)]
        self.prompt = True      # the running forward is the prompt's

    @classmethod
    def for_model(cls, model, batch: int, **kw) -> "PagedTargetCache":
        c = model.config
        head_dim = getattr(c, "head_dim", None) or c.hidden_size // c.num_attention_heads
        return cls(c.num_hidden_layers, batch, c.num_key_value_heads, head_dim, device=model.device, dtype=model.dtype,
                   **kw)

    def crop(self, lengths) -> None:
        self.pages.crop(lengths)

    def evict(self) -> bool:
        """Back to ``keep`` tokens, if a sequence is longer."""
        return bool(self.keep) and self.pages.evict(self.keep, recent=self.recent, first=self.first)


def _pads_left(mask: Optional[torch.Tensor]) -> bool:
    """Whether a prompt's attention mask ([batch, tokens], or [batch, 1,
    queries, keys] of truth values or of what is added to the scores) hides the
    first token of a sequence from itself."""
    if mask is None:
        return False
    first = mask[:, 0] if mask.dim() == 2 else mask[:, 0, 0, 0]
    return not bool((first == 0 if first.is_floating_point() else first != 0).all())


def install_target(model) -> None:
    """Route attention steps over a ``PagedTargetCache`` through the paged
    kernels: any number of new tokens, every sequence at its own length.  The
    prompt's forward (an empty cache) stays the model's own.  Positions come
    from ``position_ids``; pass them where sequences differ in length or
    tokens have been evicted.

    Prompts of different lengths are padded on the right and the cache then
    cropped to each one's own (``cache.crop(lengths)``); left padding would
    stay in the cache and is refused.  A sliding layer's own window holds where
    the cache's is not tighter.  After the prompt the attention mask is
    not read: a token sees its sequence's tokens up to itself."""
    for layer in model.model.layers:
        attn = layer.self_attn
        original = attn.forward

        def forward(self, hidden_states, position_embeddings, attention_mask, past_key_values=None,
                    _original=original, **kwargs):
            cache = past_key_values
            tokens = hidden_states.shape[1]
            if not isinstance(cache, PagedTargetCache) or (
                    cache.pages.get_seq_length() == 0 if self.layer_idx == 0 else cache.prompt):
                if isinstance(cache, PagedTargetCache):
                    if self.layer_idx == 0 and _pads_left(attention_mask):
                        raise ValueError("a paged target cache takes prompts padded on the right: "
                                         "crop it to each prompt's length afterwards.")
                    cache.prompt = True
                return _original(hidden_states, position_embeddings, attention_mask, past_key_values, **kwargs)
            if self.layer_idx == 0:
                cache.prompt = False
                cache.pages.advance(int(tokens))
            shape = hidden_states.shape[:-1]
            view = (*shape, -1, self.head_dim)
            q = self.q_proj(hidden_states).view(view).transpose(1, 2)
            k = self.k_proj(hidden_states).view(view).transpose(1, 2)
            v = self.v_proj(hidden_states).view(view).transpose(1, 2)
            q, k = apply_rotary_pos_emb(q, k, *position_embeddings)
            cache.pages.append(self.layer_idx, k, v)
            window, sinks = cache.window, cache.sinks
            own = getattr(self, "sliding_window", None) or 0
            if own and not 0 < window <= own:        # a sliding layer's own window, unless the cache's is tighter
                window, sinks = own, 0
            out = cache.pages.attention(self.layer_idx, q, scale=self.scaling, window=window, sinks=sinks)
            return self.o_proj(out.transpose(1, 2).reshape(*shape, -1).contiguous()), None

        attn.forward = types.MethodType(forward, attn)


@torch.inference_mode()
def speculative_generate(target, draft, input_ids: torch.Tensor, *, max_new_tokens: int, draft_tokens: int = 4,
                         temperature: float = 0.0, residual: int = 128, page_size: int = 16,
                         generator: Optional[torch.Generator] = None, window: int = 0, sinks: int = 0, keep: int = 0,
                         recent: int = 0, first: int = 0, **draft_kw) -> Tuple[torch.Tensor, List[int]]:
    """Speculative decoding of one sequence: ``draft`` proposes
    ``draft_tokens`` tokens a round over its packed cache, ``target`` scores
    them in one forward over its paged cache, ``verify_draft_tokens`` takes
    the accepted ones and one more (``temperature=0``: the target's greedy
    tokens; else its samples).  Both models need the hooks (``install(draft)``,
    ``install_target(target)``).

    Returns the ids with the new tokens, and how many drafted tokens each
    round accepted.  ``window``, ``sinks``, ``keep``, ``recent``, ``first``
    are the target cache's (``PagedTargetCache``, which says what an early
    eviction goes by); ``draft_kw`` the draft cache's (k_bits, v_bits,
    group_size).  Raises RuntimeError where the target's logits leave no token.
    """
    if input_ids.shape[0] != 1:
        raise ValueError("the packed draft cache serves one sequence length: generate one sequence at a time.")
    if draft_tokens < 1 or max_new_tokens < 1:
        raise ValueError("draft_tokens and max_new_tokens must be positive.")
    dev, K = input_ids.device, int(draft_tokens)
    length = int(input_ids.shape[1])
    room = length + max_new_tokens + K + 1
    cache = PagedTargetCache.for_model(target, 1, max_tokens=room, page_size=page_size, window=window, sinks=sinks,
                                       keep=keep, recent=recent, first=first)
    packed = PackedDraftCache.empty(len(draft.model.layers), residual, spare_capacity=room - length, **draft_kw)

    def pick(logits: torch.Tensor) -> torch.Tensor:
        if temperature == 0:
            return logits.argmax(-1, keepdim=True)
        p = torch.softmax(logits.float() / temperature, -1)
        return torch.multinomial(p, 1, generator=generator)

    def positions(n: int) -> torch.Tensor:
        return torch.arange(length, length + n, device=dev)[None]

    token = pick(target(input_ids, past_key_values=cache, use_cache=True).logits[:, -1])
    draft(input_ids, past_key_values=packed, use_cache=True)
    out, rounds = [token], []
    while len(out) < max_new_tokens:
        start = packed.get_seq_length()
        fed, drafted, scores = token, [], []
        for i in range(K + 1):          # the last step only brings the draft's cache up to the last drafted token
            logits = draft(fed, past_key_values=packed, use_cache=True,
                           position_ids=torch.full((1, 1), length + i, device=dev)).logits[:, -1]
            if i < K:
                fed = pick(logits)
                drafted.append(fed)
                scores.append(logits)
        proposal = torch.cat(drafted, 1)
        held = cache.pages.get_seq_length()
        logits = target(torch.cat([token, proposal], 1), past_key_values=cache, use_cache=True,
                        position_ids=positions(K + 1)).logits
        uniforms = noise = q_logits = None
        if temperature > 0:
            uniforms = torch.rand(1, K, device=dev, generator=generator)
            noise = torch.empty(1, logits.shape[-1], device=dev).exponential_(generator=generator)
            q_logits = torch.stack(scores, 1)
        r = verify_draft_tokens(logits, q_logits, proposal, uniforms, noise, temperature=temperature)
        accepted = int(r.accepted[0])
        new = r.tokens[0, :accepted + 1]
        if int(new[-1]) < 0:     # not an id: an embedding would read out of range
            raise RuntimeError("no token can follow: the target's logits are NaN or -inf throughout.")
        packed.crop(start + 1 + accepted)
        packed.commit()
        cache.crop([held + 1 + accepted])
        cache.evict()
        length += 1 + accepted
        rounds.append(accepted)
        out.extend(t.view(1, 1) for t in new)
        token = new[-1:].view(1, 1)
    return torch.cat([input_ids, *out[:max_new_tokens]], 1), rounds
