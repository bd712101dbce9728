"""Attention of whole prompts in 16 bits: what stands in front of the paged 8-bit cache, whose own attention takes every later token.

    turned, keys = cache.write_rotated(layer, query, keys, values, cosine, sine, offsets=offsets, return_keys=True)
    out = prompt_attention(turned, keys, values, offsets=offsets)
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from ._lib import HEAD_DIM, lib
from .paged_cache import _device, _FAR, _LEAST_CAP, _SCALING, _as, _recorded, PagedKVCache

_ATTEND, _ATTEND_BYTES = _lib.PROMPT_ENTRIES
_native = _lib._native


def prompt_attention(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, *, offsets: Optional[torch.Tensor] = None,
                     key_offsets: Optional[torch.Tensor] = None, causal: bool = True, starts: Optional[torch.Tensor] = None, scaling: Optional[float] = None,
                     softcap: Optional[float] = None, window: Optional[int] = None, return_lse: bool = False):
    """query [B, Hq, L, 128] over keys, values [B, Hkv, T, 128] of the same 16-bit type -> [B, L, Hq, 128] of that type, and on request lse fp32 [B, Hq, L].

    Query l stands at position i = T - L + l (a prompt: L = T; a later chunk over all keys so far: L < T; where there are more queries than keys, the first ones see nothing) and sees keys
    lo <= j < hi: lo is its row's start (`starts`, int32 [B]: where the text behind padding begins; default 0), and not before i - window + 1; hi is i + 1, or T where
    `causal` is False.  Scores are scaling * q.k (default 128 ** -0.5), then softcap * tanh(x / softcap) (a softcap past 2 ** 100 counts as that).  Queries that see nothing get 0, and -inf for lse; what a query
    does not see has no part in its result, infinities and NaN included.

    Packed: with `offsets` (int32 [S + 1] on the device, ascending) query is [1, Hq, N, 128], sequence s's queries those from offsets[s] to before offsets[s + 1], its keys and values in [1, Hkv,
    M, 128] by `key_offsets`, or by the same offsets; `starts` is [S] then.  Queries that no sequence has get 0 and -inf.  Nothing is read back.

    The same call gives the same bits; a query's last bits may differ where its neighbours do (32 queries make their weights together).

    Grouped heads: Hq a multiple of Hkv.  For inference: tensors that require gradients are refused while gradients are recorded, and so are dual numbers."""
    if isinstance(query, torch.Tensor) and query.is_cuda and query.device.index == _device() and (softcap is None or _LEAST_CAP <= softcap < math.inf) and (
            window is None or (window >= 1 and causal)):
        # (everything as the kernel takes it: one native call)
        done = _native.prompt_attend(_ATTEND, _ATTEND_BYTES, query.device.index, query, keys, values, offsets, key_offsets, starts, causal,
                                     0 if window is None else min(window, _FAR), _SCALING if scaling is None else scaling, 0.0 if softcap is None else softcap,
                                     return_lse, _lib.stream_ptr(query.device))
        if done is not None:
            return done
    for t, what in ((query, "queries"), (keys, "keys"), (values, "values")):
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape[3] != HEAD_DIM:
            raise ValueError(f"{what} must be [B, heads, tokens, {HEAD_DIM}], got {tuple(getattr(t, 'shape', ())) or type(t).__name__}")
        _lib.require_gpu(t, what)
        if t.dtype not in (torch.float16, torch.bfloat16) or t.dtype != query.dtype:
            raise ValueError(f"{what} must be float16 or bfloat16, all of one type, got {t.dtype}")
        if t.device != query.device:
            raise ValueError(f"{what} lie on {t.device}, queries on {query.device}")
    if _recorded(query, keys, values):
        raise RuntimeError("prompt_attention records no gradients and carries no tangents: call it under torch.no_grad(), outside of dual numbers")
    B, Hq, L, _ = query.shape
    Hkv, T = keys.shape[1], keys.shape[2]
    if keys.shape != values.shape:
        raise ValueError(f"keys are {tuple(keys.shape)}, values {tuple(values.shape)}")
    if keys.shape[0] != B or B == 0 or (offsets is not None and B != 1):
        raise ValueError(f"{B} rows of queries, {keys.shape[0]} of keys{'' if offsets is None else ': packed tensors have one'}")
    if Hq == 0 or Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads over {Hkv} kv heads")
    if softcap is not None and not _LEAST_CAP <= softcap < math.inf:
        raise ValueError(f"softcap must be positive, at least 2 ** -100, got {softcap}")
    if window is not None and (window < 1 or not causal):
        raise ValueError(f"window must be positive, and the attention causal, got {window}")
    if key_offsets is not None and offsets is None:
        raise ValueError("key_offsets say where packed rows' keys begin: offsets are wanted beside them")
    if offsets is not None and (not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 2):
        raise ValueError(f"offsets must be [sequences + 1], got {tuple(getattr(offsets, 'shape', ())) or type(offsets).__name__}")
    if offsets is not None and key_offsets is None and L != T:
        raise ValueError(f"{L} packed queries and {T} keys: key_offsets say where the keys begin")
    device, rows = query.device, B if offsets is None else offsets.shape[0] - 1

    def small(t, n, what):
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.shape != (n,):
            raise ValueError(f"{what} must be [{n}], got {tuple(getattr(t, 'shape', ())) or type(t).__name__}")
        if t.device != device:
            raise ValueError(f"{what} lie on {t.device}, queries on {device}")
        if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
            raise ValueError(f"{what} must be whole numbers, got {t.dtype}")
        return _as(t, torch.int32).contiguous()

    offsets, key_offsets, starts = small(offsets, rows + 1, "offsets"), small(key_offsets, rows + 1, "key_offsets"), small(starts, rows, "starts")
    query, keys, values = (PagedKVCache._rows_ok(t) for t in (query, keys, values))
    keys, values = (t.contiguous() if t.stride(2) >= 1 << 24 else t for t in (keys, values))
    out = torch.empty(B, L, Hq, HEAD_DIM, dtype=query.dtype, device=device)
    lse = torch.empty(B, Hq, L, dtype=torch.float32, device=device) if return_lse else None
    if L:
        nbytes = lib.odmkv_prompt_attend_workspace_bytes(offsets is not None, rows, Hq, Hkv, L, T, bool(causal), min(window or 0, _FAR), 0.0 if softcap is None else softcap)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None          # (of its own for every call: a graph's is the graph's)
        a = _lib.PromptAttend(*(x for t in (query, keys, values) for x in (t.data_ptr(), *t.stride()[:3])), out.data_ptr(), _lib.ptr(lse), _lib.ptr(offsets),
                              _lib.ptr(key_offsets), _lib.ptr(starts), _lib.ptr(ws), nbytes, _lib._DT[query.dtype], rows, L, T, Hq, Hkv, causal, min(window or 0, _FAR),
                              _SCALING if scaling is None else float(scaling), 0.0 if softcap is None else float(softcap))
        with torch.cuda.device(device):
            _lib.check(lib.odmkv_prompt_attend(C.byref(a), _lib.stream_ptr(device)))
    return (out, lse) if return_lse else out
