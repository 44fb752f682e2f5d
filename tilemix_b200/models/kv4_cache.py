"""Key/value cache in 4 bits for the HF models: pass a ``Kv4Cache`` as ``past_key_values``.

    cache = Kv4Cache(max_cache_len=8192)
    model(prompt, past_key_values=cache, use_cache=True)          # prefill, then
    model(next_ids, past_key_values=cache, use_cache=True)        # steps of one or more tokens
    model.generate(prompt, past_key_values=cache, ...)

(no counterpart in the reference). A model with TileMix attention (``inject_tilemix_into_llama`` /
``_qwen``) prefills with the routed attention, stores its keys and values in 4 bits and attends
over the cache itself (``kv4_attention``) in every later step, whatever its length (made for a few
tokens: hundreds over a long cache are slow); the prompt's first pass uses the unrounded keys and values, except for prompts under 16 tokens. Any other
attention gets the cached keys and values read back as fp16 from ``update``. Of an attention mask
the steps after the prompt use the keys that its last row allows: a batch's padding, not a pattern
of its own for each new token.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from transformers.cache_utils import Cache, CacheLayerMixin

from tilemix_b200.attention.kv4 import build_block_tables, kv4_append, kv4_attention, kv4_pool, kv4_read

__all__ = ["Kv4Cache"]


class _Kv4Layer(CacheLayerMixin):
    """One layer's pool; pages, lengths and slots belong to the cache and are the same for every layer."""

    is_sliding = False

    def __init__(self, cache: "Kv4Cache"):
        super().__init__()
        self.cache = cache
        self.pool: Optional[Tensor] = None
        self.seen = 0  # tokens a request in this layer's pool

    def lazy_initialization(self, key_states: Tensor, value_states: Tensor) -> None:
        self.pool = self.cache._new_pool(key_states)
        self.is_initialized = True

    def append(self, key_states: Tensor, value_states: Tensor) -> None:
        """Store [B, H, T, D] keys and values of the next T tokens of every request."""
        if key_states.dtype != torch.float16 or value_states.dtype != torch.float16:
            raise TypeError("Kv4Cache holds fp16 keys and values; run the model in torch.float16")
        b, h, t, d = key_states.shape
        if self.seen == self.cache.seen:
            self.cache._plan(b, t, key_states.device)
        elif self.seen + t != self.cache.seen or b != self.cache.batch:
            raise ValueError("the layers of a Kv4Cache must be given the same tokens")
        if self.pool is None:
            self.lazy_initialization(key_states, value_states)
        rows = lambda x: x.transpose(1, 2).reshape(b * t, h, d)  # noqa: E731  (a view of token-major storage)
        kv4_append(rows(key_states), rows(value_states), self.pool, self.cache.step.slots)
        self.seen += t

    def update(self, key_states: Tensor, value_states: Tensor, *args, **kwargs) -> tuple[Tensor, Tensor]:
        b, h, _, d = key_states.shape
        self.append(key_states, value_states)
        k, v = kv4_read(self.pool, self.cache._all_slots(), d)
        return tuple(x.view(b, self.seen, h, d).transpose(1, 2) for x in (k, v))

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        return self.seen + query_length, 0

    def get_seq_length(self) -> int:
        return self.seen

    def get_max_cache_shape(self) -> int:
        return self.cache.max_cache_len

    def reset(self) -> None:
        self.seen = 0

    def offload(self) -> None:
        raise NotImplementedError("Kv4Cache stays on its device")

    prefetch = offload

    def reorder_cache(self, beam_idx) -> None:
        raise NotImplementedError("Kv4Cache does not reorder its requests (beam search)")

    def crop(self, max_length: int) -> None:
        raise NotImplementedError("Kv4Cache does not give tokens back one by one; reset() it")

    def batch_repeat_interleave(self, repeats: int) -> None:
        raise NotImplementedError("Kv4Cache does not copy requests")

    def batch_select_indices(self, indices) -> None:
        raise NotImplementedError("Kv4Cache does not select requests")


class Kv4Cache(Cache):
    """4-bit paged cache of up to ``max_cache_len`` tokens for each request of a batch.

    ``page_size`` tokens a page (a multiple of 16); ``num_pages`` pages a layer (default: enough for
    ``max_cache_len`` tokens of every request). The batch size is that of the first call; ``reset``
    empties the cache for a new batch of the same size.
    """

    def __init__(self, max_cache_len: int, page_size: int = 64, num_pages: Optional[int] = None):
        if max_cache_len <= 0:
            raise ValueError("max_cache_len must be positive")
        if page_size < 16 or page_size % 16:
            raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")
        super().__init__(layers=[])
        self.page_size, self.num_pages = page_size, num_pages
        self._max_len = max_cache_len
        self.batch = 0
        self.seen = 0     # tokens a request, host-known: every request of an HF batch has as many
        self.pages = 0    # pages taken
        self.step = None  # block tables of the current step (slots of its tokens, lengths after it)

    @property
    def max_cache_len(self) -> int:
        return self._max_len

    @property
    def max_batch_size(self) -> int:
        return self.batch

    def _layer(self, layer_idx: int) -> _Kv4Layer:
        while len(self.layers) <= layer_idx:
            self.layers.append(_Kv4Layer(self))
        return self.layers[layer_idx]

    def update(self, key_states: Tensor, value_states: Tensor, layer_idx: int, *args, **kwargs):
        return self._layer(layer_idx).update(key_states, value_states)

    def append(self, key_states: Tensor, value_states: Tensor, layer_idx: int) -> None:
        """:meth:`update` without reading the cache back."""
        self._layer(layer_idx).append(key_states, value_states)

    def attend(self, q: Tensor, layer_idx: int, sm_scale: float, key_mask: Optional[Tensor] = None) -> Tensor:
        """Causal attention of the T tokens just appended, q [B, H, T, D] -> [B, T, H, D]."""
        b, h, t, d = q.shape
        rows = q.transpose(1, 2).reshape(b * t, h, d)
        out = kv4_attention(rows, self._layer(layer_idx).pool, self.table, self.step.kv_lens, self.step.cu_seqlens_q, t,
                            sm_scale=sm_scale, key_mask=key_mask, max_kv_len=self.seen)
        return out.view(b, t, h, d)

    def reset(self) -> None:
        super().reset()
        self.seen = self.pages = 0
        self.step = None
        if self.batch:
            self._free_all()

    # -- pages
    @torch.inference_mode()  # where tensors that were made in it, by a step, may be changed in place
    def _free_all(self) -> None:
        self.table.fill_(-1)
        self.lens.zero_()
        torch.arange(self.ring.numel(), dtype=torch.int32, out=self.ring)
        self.span.copy_(torch.tensor([0, self.ring.numel()]))

    def _plan(self, batch: int, tokens: int, device: torch.device) -> None:
        """Pages and slots of the next ``tokens`` tokens of every request."""
        per = (self._max_len + self.page_size - 1) // self.page_size
        if not self.batch:
            self.batch = batch
            n = batch * per if self.num_pages is None else self.num_pages
            self.table = torch.empty((batch, per), dtype=torch.int32, device=device)
            self.lens = torch.empty(batch, dtype=torch.int32, device=device)
            self.ring = torch.empty(n, dtype=torch.int32, device=device)
            self.span = torch.empty(2, dtype=torch.int64, device=device)
            self._free_all()
        if batch != self.batch:
            raise ValueError(f"the cache holds {self.batch} requests, got {batch}")
        if self.seen + tokens > self._max_len:
            raise ValueError(f"{self.seen} + {tokens} tokens exceed max_cache_len {self._max_len}")
        pages = batch * ((self.seen + tokens + self.page_size - 1) // self.page_size)
        if pages > self.ring.numel():
            raise ValueError(f"{pages} pages are needed, the cache has {self.ring.numel()}")
        new = torch.full((batch,), tokens, dtype=torch.int32, device=device)
        self.step = build_block_tables(self.lens, new, self.table, self.ring, self.span, page_size=self.page_size,
                                       max_new_tokens=batch * tokens)
        self.lens, self.span = self.step.kv_lens, self.step.free_span
        self.seen += tokens
        self.pages = pages

    def _new_pool(self, key_states: Tensor) -> Tensor:
        return kv4_pool(self.ring.numel(), self.page_size, key_states.shape[1], key_states.shape[3],
                        key_states.device)

    def _all_slots(self) -> Tensor:
        pos = torch.arange(self.seen, device=self.table.device)
        return (self.table[:, pos // self.page_size].long() * self.page_size + pos % self.page_size).flatten()
