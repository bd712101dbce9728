"""Caches for `transformers` that keep no dense copy: `PackedCacheLayer` over the packed store, and (not in the reference in any form)
`PagedCache` over the paged 8-bit cache.

`PackedCacheLayer` is a cache layer whose tokens live only in the packed store.

The reference keeps a dense fp16 copy of every layer's keys and values in the model's
`DynamicCache` next to its quantised banks (kvquant/adaptive_backend_press.py:131-149 writes the
dequantised rows back into it) and `DynamicLayer.update` re-concatenates that copy at every decode
step.  With the fused decode kernel nothing reads the copy any more, so a press built with
``release_dense_cache=True`` swaps each layer of the cache for a `PackedCacheLayer` once the
prefill has been packed:

* ``keys`` / ``values`` keep the shape ``[B, H, T, D]`` the model and the mask code look at, but
  are stride-0 views of the newest token: no memory, no concatenation;
* a single-token ``update`` re-aliases the views; the attention function takes the token from
  them and everything older from the store;
* an ``update`` with several tokens (prompt text after the prefill) returns the new tokens alone, tagged
  with the store's length: the attention patch runs the block through the fused kernel as well;
* ``crop`` truncates the store; a harness that rewinds the cache the reference's way
  (benchmark/core/pipeline.py:211-228: ``layer._tq_backend_state.truncate`` and a slice of
  ``layer.keys``) works on it unchanged.

The dense attention path cannot run on the aliased views; the attention patch refuses them.
"""
from __future__ import annotations

from typing import Optional

import torch
from transformers.cache_utils import Cache, CacheLayerMixin, DynamicLayer
from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

from kvquant._lib import HEAD_DIM, _native
from kvquant.attention_patch import patch_attention_functions
from kvquant.paged_cache import KINDS, OutOfPages, PagedKVCache

alias = _native.alias             # stride-0 views of the last token (two views in one call)


class PackedCacheLayer(DynamicLayer):
    def __init__(self, state, keys: torch.Tensor, values: torch.Tensor):
        """`state` holds every token of `keys`/`values` ([B, H, T, D], the layer's dense cache so
        far); only their last token is kept."""
        super().__init__()
        if state.seq_len != keys.shape[-2]:
            raise ValueError(f"the packed store holds {state.seq_len} tokens, the cache layer {keys.shape[-2]}")
        self.dtype, self.device = keys.dtype, keys.device
        self.is_initialized = True
        self.state = state
        self._tq_backend_state = state
        self.recent = (keys[:, :, -1:, :].clone(), values[:, :, -1:, :].clone())
        self._alias(keys.shape[-2])

    def _alias(self, length: int) -> None:
        self.keys, self.values = alias(*self.recent, length)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        q_len = key_states.shape[-2]
        before = self.keys.shape[-2]
        if q_len == 1:
            self.recent = (key_states, value_states)
            self._alias(before + 1)
            return self.keys, self.values
        if self.state.seq_len != before:
            raise RuntimeError(f"the packed store holds {self.state.seq_len} tokens, the cache layer {before}: "
                               "a multi-token step needs the two in step")
        # the new tokens alone, tagged with the number of tokens the store holds: the attention patch takes the
        # stored part from the fused kernel and the block's own attention from these (nothing is dequantised)
        key_states._odmkv_store_len = before
        value_states._odmkv_store_len = before
        self.recent = (key_states, value_states)
        self._alias(before + q_len)
        return key_states, value_states

    def crop(self, tokens_to_remove: int) -> None:
        current = self.keys.shape[-2]
        if tokens_to_remove > 0:                      # legacy meaning: the length to keep
            if tokens_to_remove >= current:
                return
            tokens_to_remove = current - tokens_to_remove
        if tokens_to_remove == 0:
            return
        length = max(current - abs(tokens_to_remove), 0)
        self.state.truncate(length)
        self._alias(length)

    # the dense-tensor operations of the base class have no meaning on aliased views
    def reset(self) -> None:
        raise NotImplementedError("PackedCacheLayer cannot be reset in place: start a new cache")

    def reorder_cache(self, beam_idx) -> None:
        raise NotImplementedError("PackedCacheLayer does not support beam reordering")

    def batch_repeat_interleave(self, repeats: int) -> None:
        raise NotImplementedError("PackedCacheLayer does not support batch expansion")

    def batch_select_indices(self, indices) -> None:
        raise NotImplementedError("PackedCacheLayer does not support batch selection")

    def offload(self) -> None:
        return

    def prefetch(self) -> None:
        return


def is_aliased(t: torch.Tensor) -> bool:
    """True for the stride-0 token views a `PackedCacheLayer` hands out."""
    return t.dim() == 4 and t.shape[2] > 1 and t.stride(2) == 0


class PagedTokens(torch.Tensor):
    """New tokens' keys or values as a `PagedCache` hands them out: a mark for the patched attention functions, which read everything from the pages.  They are not
    all the keys that there are, so that whoever would compute with them (attention inside a model, an attention function that is not patched, a cast
    or copy that leaves the mark behind) is told instead of being given the attention over the newest tokens alone."""

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        name = getattr(func, "__name__", "")
        with torch._C.DisableTorchFunctionSubclass():
            if name in _LOOKS or func in _FIELDS:
                return func(*args, **(kwargs or {}))
            if name in _KEEPS:                            # where nothing is to be done they hand the tensor itself on
                out = func(*args, **(kwargs or {}))
                if out is args[0]:
                    return out
        raise RuntimeError(f"{name}() of a PagedCache's keys or values: they are the newest tokens alone, the others lie in pages, which the attention functions that transformers "
                           "registers read (attn_implementation=\"sdpa\"); casts, copies and attention inside the model cannot be answered")


# what a look at a tensor is, and what may be a look
_LOOKS = ("dim", "size", "stride", "numel", "is_contiguous", "is_floating_point", "is_complex", "data_ptr", "get_device", "element_size", "storage_offset", "__len__", "__hash__", "__repr__")
_FIELDS = tuple(getattr(torch.Tensor, field).__get__ for field in ("shape", "dtype", "device", "ndim", "layout", "is_cuda", "is_cpu", "requires_grad", "grad_fn", "is_leaf", "grad"))
_KEEPS = ("contiguous", "to", "type_as", "half", "bfloat16", "float", "cuda")


def paged_tokens(keys: torch.Tensor, values: torch.Tensor, paged):
    """Keys and values as `PagedTokens`, the keys with what the attention patch needs: (pool, layer, tokens of a row)."""
    keys, values = keys.as_subclass(PagedTokens), values.as_subclass(PagedTokens)
    keys._odmkv_paged = paged
    return keys, values


class PagedCacheLayer(CacheLayerMixin):
    """A model layer's part of a `PagedCache`."""
    is_sliding = False

    def __init__(self, owner: "PagedCache", index: int):
        super().__init__()
        self.owner, self.index, self.length = owner, index, 0

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        self.owner._make(key_states)
        self.dtype, self.device = key_states.dtype, key_states.device
        self.is_initialized = True

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        """Stores the new tokens.  With `native_prompt` the first ones of a row (the prompt) go back as `PagedTokens` that carry themselves, for the attention patch to hand to
        `prompt_attention`.  Otherwise they go back as they are, for the model's own attention in full precision, unless that caps scores, which
        the registered functions that a model would use here leave out in silence (a call with `softcap` finds its way by the mark); these and all later ones go
        back as `PagedTokens`, for the attention patch, which reads everything from the pages."""
        owner, T = self.owner, key_states.shape[-2]
        if self.length == 0:
            self.lazy_initialization(key_states, value_states)
        owner._room(self.length + T)
        owner.pool.write(self.index, key_states, value_states)
        before, self.length = self.length, self.length + T
        paged = (owner.pool, self.index, self.length)
        if before == 0 and owner.native_prompt:
            tokens = paged_tokens(key_states, value_states, paged)
            tokens[0]._odmkv_prompt_rows = (key_states, value_states)
            return tokens
        if before == 0 and not owner.capped:
            key_states._odmkv_prompt = paged
            return key_states, value_states
        return paged_tokens(key_states, value_states, paged)

    def get_seq_length(self) -> int:
        return self.length

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        return self.length + query_length, 0

    def get_max_length(self) -> int:
        return self.owner.max_tokens

    @property
    def batch_size(self) -> int:
        return -1 if self.owner.pool is None else self.owner.pool.batch

    # rows and lengths are all layers' together: see the cache's own methods
    def _all_layers(self, *args):
        raise NotImplementedError("the layers of a PagedCache share their rows: call the cache's own method")

    reset = crop = reorder_cache = batch_repeat_interleave = batch_select_indices = _all_layers

    def offload(self) -> None:
        return

    def prefetch(self) -> None:
        return


class PagedCache(Cache):
    """A `transformers` cache of 8 bits a value (``kvquant.PagedKVCache``: int8 or e4m3 codes, one scale for 64 tokens of a head): pass it as
    ``past_key_values``.  The prompt is attended in the model's own precision and stored; every later token attends over the pages, soft caps and sliding
    windows included.  Where scores are capped, the prompt attends over the pages as well: one cap from the first token on.  Beams and samples share the pages of what they have in common: ``reorder_cache``, ``batch_repeat_interleave`` and
    ``batch_select_indices`` copy 16-bit tails and count holders.  The pool starts at the prompt's size and is grown as rows do.

    `config`: the model's; its attention must be one of the registered functions (not "eager", which cannot be told to read the pages).

    `shared`: steps read the pages that rows have in common once for all of them (``PagedKVCache.attend(shared=True)``): for beams and samples of long prompts,
    not for windows much shorter than those, nor for samples of several prompts behind one system prompt.
    `native_prompt`: the prompt is attended by ``kvquant.prompt_attention``, padding in front, windows and soft caps included, in the model's own precision where scores
    are capped too; the model's own attention is not called then."""

    def __init__(self, config, max_tokens: Optional[int] = None, kind: str = "int8", *, shared: bool = False, native_prompt: bool = False):
        text = config.get_text_config(decoder=True)
        head_dim = getattr(text, "head_dim", None) or text.hidden_size // text.num_attention_heads
        kinds = set(getattr(text, "layer_types", None) or ()) - {"full_attention", "sliding_attention"}
        implementation = getattr(text, "_attn_implementation", None) or getattr(config, "_attn_implementation", None)
        if head_dim != HEAD_DIM:
            raise ValueError(f"head_dim {head_dim} is not supported (the kernels are written for {HEAD_DIM})")
        if kinds:
            raise ValueError(f"layers of type {sorted(kinds)} keep no keys and values a token")
        if implementation not in ALL_ATTENTION_FUNCTIONS.keys():
            raise ValueError(f"attn_implementation={implementation!r} is not a registered attention function: set \"sdpa\"")
        if kind not in KINDS:
            raise ValueError(f"kind must be one of {sorted(KINDS)}, got {kind!r}")
        patch_attention_functions()
        self.capped = getattr(text, "attn_logit_softcapping", None) is not None
        self.max_tokens = int(text.max_position_embeddings if max_tokens is None else max_tokens)
        self.kind, self.pool, self._extended = kind, None, 0
        self.shared, self.native_prompt = bool(shared), bool(native_prompt)
        super().__init__(layers=[PagedCacheLayer(self, i) for i in range(text.num_hidden_layers)])

    def _make(self, keys: torch.Tensor) -> None:
        B, H, T, _ = keys.shape
        if self.pool is None or (self._extended == 0 and self.pool.batch != B):
            self.pool = PagedKVCache(B, H, self.max_tokens, layers=len(self.layers), pages=B * (T // 64 + 4), kind=self.kind, dtype=keys.dtype,
                                     device=keys.device, head_dim=keys.shape[-1])
            self.pool.shares = self.shared

    def _room(self, length: int) -> None:
        """The rows hold `length` tokens from here on: the first layer that comes by with new ones sees to it for all."""
        if length <= self._extended:
            return
        try:
            self.pool.extend(length - self._extended)
        except OutOfPages:
            # half as much again as there is, and what this call needs
            need = self.pool.batch * ((length - self._extended) // 64 + 1)
            self.pool = self.pool.compacted(pages=self.pool.pages + max(self.pool.pages // 2, need))
            self.pool.extend(length - self._extended)
        self._extended = length

    def _set_length(self, length: int) -> None:
        self._extended = length
        for layer in self.layers:
            layer.length = length

    def reset(self) -> None:
        if self.pool is not None:
            self.pool.free()
        self._set_length(0)

    def crop(self, tokens_to_remove: int) -> None:
        current = self._extended
        keep = min(tokens_to_remove, current) if tokens_to_remove > 0 else max(current + tokens_to_remove, 0)      # (positive: the length to keep)
        if keep < current:
            self.pool.truncate(keep)
            self._set_length(keep)

    def reorder_cache(self, beam_idx) -> None:
        if self.pool is not None:
            self.pool.reorder(beam_idx.to(self.pool.device) if isinstance(beam_idx, torch.Tensor) else beam_idx)

    def batch_select_indices(self, indices) -> None:
        if self.pool is None:
            return
        old = self.pool
        if isinstance(indices, torch.Tensor) and indices.dtype == torch.bool:
            indices = indices.nonzero().view(-1)
        self.pool = old.select(indices.to(old.device) if isinstance(indices, torch.Tensor) else indices)
        old.release()

    def batch_repeat_interleave(self, repeats: int) -> None:
        if self.pool is not None:
            self.batch_select_indices([b for b in range(self.pool.batch) for _ in range(repeats)])
