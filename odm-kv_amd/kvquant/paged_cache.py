"""A paged KV cache of 8 bits a value, with the attention that reads it and the operations that move its rows.

``PagedKVCache`` holds the rows (sequences) of a batch.  Tokens 64 j .. 64 j + 63 of a row are its block j: a full block lies in a page, as
int8 or e4m3 codes with one scale per kv-head for keys and one for values; the newest tokens, fewer than 64, stay in the model's 16 bits in the row's
tail.  Pages are shared between rows (``reorder``, ``select``) and between the layers' bookkeeping: one ``extend`` a step makes room in all
layers, one ``write`` a layer stores its tokens, one ``attend`` a layer reads them.

    cache = PagedKVCache(batch, kv_heads, max_tokens, layers=n_layers, dtype=torch.bfloat16)
    cache.extend(q_len)                                   # once a forward
    cache.write(layer, keys, values)                      # [B, Hkv, q_len, 128], once a layer
    out = cache.attend(layer, query)                      # [B, Hq, q_len, 128] -> [B, q_len, Hq, 128]

Lengths, tables and the count of every page's holders live on the device, so that a step can be captured into a graph and goes on from where
the rows are at each replay.  The host keeps an upper bound of every row's length and of the pages in use, checks every call against them
before anything is launched, and reads the device's only where those bounds do not settle it.  After replays of a captured ``extend`` the bounds are out
of date: ``refresh`` reads them back (and raises if a replay found no room).  The cache is for inference: nothing records gradients.
"""
from __future__ import annotations

import ctypes as C
import math
import weakref
from typing import Optional, Sequence, Union

import torch

from . import _lib
from ._lib import HEAD_DIM, lib

BLOCK = 64                                    # tokens of a page
MAX_ROWS = 1024                               # the bookkeeping runs in one workgroup, a thread a row
HOST_ROWS = 512                               # batches up to here have a row's number each travel in the launch's arguments
MAX_GROUP = 8
KINDS = {"int8": (0, torch.int8), "e4m3": (1, torch.float8_e4m3fn)}

_SCALING = HEAD_DIM ** -0.5
_FAR = 2 ** 30                                # a window past everything
_LEAST_CAP = 2.0 ** -100                      # (what 32 bits make 0 of would be no cap)
_WRITE, _ATTEND, _ATTEND_BYTES = _lib.PAGES_ENTRIES
_native = _lib._native
_device = torch.cuda.current_device
_capturing = torch.cuda.is_current_stream_capturing

Counts = Union[int, Sequence[int], torch.Tensor]


class OutOfPages(ValueError):
    """The pool has too few free pages for a call: `compacted` gives a larger one."""


def _blocks(tokens: int) -> int:
    return (tokens + BLOCK - 1) // BLOCK


def _as(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Whole numbers as another type; those that 32 bits do not hold stop at their end."""
    return t.clamp(-2 ** 31, 2 ** 31 - 1).to(dtype) if dtype == torch.int32 and t.dtype == torch.int64 else t.to(dtype)


class PagedKVCache:
    """`batch` rows of at most `max_tokens` tokens, `layers` layers of `kv_heads` heads of 128; `pages`: full blocks that there is room for in each layer
    (default: every row's longest).  `kind`: "int8" or "e4m3".  The tensors are attributes, laid out as include/odmkv.h says (struct odmkv_pages)."""

    def __init__(self, batch: int, kv_heads: int, max_tokens: int, *, layers: int = 1, pages: Optional[int] = None, kind: str = "int8",
                 dtype: torch.dtype = torch.float16, device="cuda", head_dim: int = HEAD_DIM):
        if head_dim != HEAD_DIM:
            raise ValueError(f"head_dim {head_dim} is not supported (the kernels are written for {HEAD_DIM})")
        if kind not in KINDS:
            raise ValueError(f"kind must be one of {sorted(KINDS)}, got {kind!r}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
        if not 1 <= batch <= MAX_ROWS:
            raise ValueError(f"batch must be 1 to {MAX_ROWS}, got {batch}")
        if kv_heads < 1 or layers < 1 or max_tokens < 1 or layers * kv_heads > 65534:
            raise ValueError(f"bad shape: {layers} layers of {kv_heads} heads, {max_tokens} tokens")
        pages = batch * (max_tokens // BLOCK) if pages is None else int(pages)
        if pages < 0:
            raise ValueError(f"pages must not be negative, got {pages}")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("the cache must live on the GPU: the ODM-KV kernels have no CPU path")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device, self.dtype, self.kind = device, dtype, kind
        self.layers, self.batch, self.kv_heads, self.max_tokens = layers, batch, kv_heads, int(max_tokens)
        self._make_pool(max(pages, 1))
        for t in (self.k_codes, self.v_codes, self.k_scale, self.v_scale):
            t.view(torch.uint8).zero_()                      # (never read before they are written: so that equal histories are equal bytes)
        self._make_rows()
        self._struct()
        with torch.cuda.device(device):
            _lib.check(lib.odmkv_pages_init(C.byref(self._p), _lib.stream_ptr(device)))

    # ------------------------------------------------------------------ memory
    def _make_pool(self, pages: int) -> None:
        codes, empty = KINDS[self.kind][1], dict(device=self.device)
        self.pages = pages
        self.k_codes = torch.empty(self.layers, pages, self.kv_heads, BLOCK, HEAD_DIM, dtype=codes, **empty)
        self.v_codes = torch.empty(self.layers, pages, self.kv_heads, HEAD_DIM, BLOCK, dtype=codes, **empty)
        self.k_scale = torch.empty(self.layers, pages, self.kv_heads, dtype=torch.float32, **empty)
        self.v_scale = torch.empty(self.layers, pages, self.kv_heads, dtype=torch.float32, **empty)
        self.refs = torch.empty(pages, dtype=torch.int32, **empty)
        self.status = torch.empty(4, dtype=torch.int32, **empty)
        # what the batches over this pool share: an upper bound of the pages in use, every batch's bounds (its own list, changed in place), and the rows of
        # batches that were dropped without `release`, whose pages the next call on the pool takes back
        self._shared = {"used": 0, "bounds": [], "left": []}

    def _make_rows(self) -> None:
        B, H, empty = self.batch, self.kv_heads, dict(device=self.device)
        self.k_tail = torch.empty(self.layers, B, H, BLOCK, HEAD_DIM, dtype=self.dtype, **empty)
        self.v_tail = torch.empty(self.layers, B, H, HEAD_DIM, BLOCK, dtype=self.dtype, **empty)
        self.table = torch.empty(B, _blocks(self.max_tokens), dtype=torch.int32, **empty)
        self.length = torch.empty(B, dtype=torch.int32, **empty)
        self.start = torch.empty(B, dtype=torch.int32, **empty)
        self.slot = torch.empty(B, dtype=torch.int32, **empty)
        self._bounds = [0] * B                               # no row is longer
        self._grown, self._written = 0, set()                # tokens a row at most of the last extend, and the layers that have stored them
        self._shared["bounds"].append(self._bounds)
        self._looked: dict = {}                              # what the attention patch has found masks to say (kvquant/attention_patch.py)

    def _nothing_to_write(self) -> None:
        self._grown, self._written = 0, range(self.layers)   # (rows have moved: what was to be stored is not there any more)

    def _struct(self) -> None:
        self._p = _lib.Pages(self.layers, self.batch, self.kv_heads, self.pages, self.table.shape[1], _lib._DT[self.dtype], KINDS[self.kind][0],
                             *(t.data_ptr() for t in (self.k_codes, self.v_codes, self.k_scale, self.v_scale, self.k_tail, self.v_tail, self.table,
                                                      self.length, self.start, self.slot, self.refs, self.status)), self.max_tokens)
        self._at = C.addressof(self._p)
        rows = (self.k_tail, self.v_tail, self.table, self.length, self.start, self.slot)
        self._dropped = weakref.finalize(self, self._shared["left"].append, (self._bounds, self._p, rows))
        self._dropped.atexit = False

    def _sibling(self, batch: int) -> "PagedKVCache":
        new = object.__new__(PagedKVCache)
        for name in ("device", "dtype", "kind", "layers", "kv_heads", "max_tokens"):
            setattr(new, name, getattr(self, name))
        new.batch = batch
        return new

    def _call(self, fn, *args) -> None:
        """One library call on the current stream of the cache's device."""
        index = self.device.index
        if torch.cuda.current_device() != index:
            with torch.cuda.device(index):
                _lib.check(fn(*args, _lib.stream_ptr(self.device)))
        else:
            _lib.check(fn(*args, _lib.stream_ptr(self.device)))

    def _ints(self, values, n: int, dtype, what: str):
        """One whole number a row: (device tensor or None, host int32 array or None, the same as a list where the host knows it)."""
        if isinstance(values, torch.Tensor) and values.is_cuda:
            if values.is_floating_point() or values.is_complex() or values.dtype == torch.bool:
                raise ValueError(f"{what} must be whole numbers, got {values.dtype}")
            if values.device != self.device:
                raise ValueError(f"{what} lie on {values.device}, the cache on {self.device}")
            if values.shape != (n,):
                raise ValueError(f"{what} must be one number a row, [{n}], got {list(values.shape)}")
            return _as(values, dtype).contiguous(), None, None
        if isinstance(values, torch.Tensor) and (values.is_floating_point() or values.is_complex() or values.dtype == torch.bool):
            raise ValueError(f"{what} must be whole numbers, got {values.dtype}")
        known = [int(v) for v in values]
        if len(known) != n:
            raise ValueError(f"{len(known)} {what} for {n} rows")
        if known and not -2 ** 31 <= min(known) <= max(known) < 2 ** 31:
            raise ValueError(f"{what} must fit 32 bits")
        if n <= HOST_ROWS:
            return None, (C.c_int32 * n)(*known), known
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} of more than {HOST_ROWS} rows must lie on the device while a graph is captured: every replay would read the host's memory again")
        return torch.tensor(known, dtype=dtype, pin_memory=True).to(self.device, non_blocking=True), None, known

    # ------------------------------------------------------------------ what the host knows
    @property
    def max_length(self) -> int:
        """No row is longer."""
        return max(self._bounds)

    def refresh(self) -> list:
        """Reads the rows' lengths and the pool's state back (this waits for the stream), and returns the lengths.  Raises RuntimeError if a
        call since the last refresh was refused on the device (a replayed graph that found no room, a bad index on the device)."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the cache's bounds do not settle this call, and its lengths cannot be read while a graph is captured")
        self._take_back()
        status, lengths = self.status.tolist(), self.length.tolist()
        self._bounds[:] = lengths
        self._shared["used"] = self.pages - status[0]
        if status[2]:
            self.status[2] = 0
            raise RuntimeError("a call on the paged cache was refused on the device: no free page, a row beyond max_tokens, or an index out of range")
        return lengths

    def _take_back(self) -> None:
        """The pages of batches over this pool that were dropped: freed on the current stream, as the pool's other calls."""
        if not self._shared["left"] or torch.cuda.is_current_stream_capturing():         # (a graph would free them at every replay)
            return
        while self._shared["left"]:
            bounds, p, rows = self._shared["left"].pop()
            self._call(lib.odmkv_pages_truncate, C.byref(p), None, None, 0, None)
            for t in rows:
                t.record_stream(torch.cuda.current_stream(self.device))
            self._shared["bounds"] = [b for b in self._shared["bounds"] if b is not bounds]
        self._used_at_most()

    def _make_room(self, counts) -> None:
        """Raises unless rows that grow by `counts` fit; afterwards the bounds include them."""
        self._take_back()
        for attempt in (0, 1):
            after = [n + c for n, c in zip(self._bounds, counts)]
            need = sum((c + BLOCK - 1) // BLOCK if self._loose else a // BLOCK - n // BLOCK for n, a, c in zip(self._bounds, after, counts))
            if max(after) <= self.max_tokens and self._shared["used"] + need <= self.pages:
                break
            if attempt:
                if max(after) > self.max_tokens:
                    raise ValueError(f"a row of {max(after)} tokens does not fit max_tokens={self.max_tokens}")
                raise OutOfPages(f"out of pages: {self._shared['used']} of {self.pages} in use, {need} more wanted")
            self.refresh()
            self._loose = False
        self._bounds[:] = after
        self._shared["used"] += need

    _loose = False                                           # the bounds may be above the lengths
    _replayed = False                                        # a write has been captured: replays store what the host does not know of

    # ------------------------------------------------------------------ tokens in
    def extend(self, counts: Counts, *, bound: Optional[int] = None) -> None:
        """Every row grows by its count of tokens (one number for all, a list, or an int32 tensor on the device with `bound`: no count is larger).
        Every layer's ``write`` then stores them."""
        if isinstance(counts, int):
            if counts < 0:
                raise ValueError(f"counts must not be negative, got {counts}")
            self._make_room([counts] * self.batch)
            self._grown, self._written = counts, set()
            self._call(lib.odmkv_pages_extend, C.byref(self._p), None, None, counts, counts)
            return
        on_device, host, known = self._ints(counts, self.batch, torch.int32, "counts")
        if known is None:
            if bound is None or bound < 0:
                raise ValueError("counts on the device need a bound that none of them is above")
            try:
                self._make_room([int(bound)] * self.batch)
            except ValueError:                               # not if every row grew by the bound: what they do grow by decides
                read = on_device.tolist()
                if min(read) < 0 or max(read) > bound:
                    raise ValueError(f"counts must be 0 to bound={bound}, got {min(read)} to {max(read)}") from None
                self._make_room(read)
            self._loose = True
        else:
            if min(known) < 0:
                raise ValueError(f"counts must not be negative, got {min(known)}")
            if bound is not None and max(known) > bound:
                raise ValueError(f"a count of {max(known)} is above bound={bound}")
            bound = max(known)
            self._make_room(known)
        bound = min(int(bound), self.max_tokens)
        self._grown, self._written = bound, set()
        self._call(lib.odmkv_pages_extend, C.byref(self._p), _lib.ptr(on_device), host, 0, bound)

    def write(self, layer: int, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Stores the tokens of the last ``extend`` in one layer, once and before rows are moved or cut: keys, values [B, Hkv, T, 128] of the cache's dtype, row b's at t < its count, T at least the
        largest count (or its bound)."""
        if layer in self._written:                           # (the new tail would be taken for the old one)
            raise ValueError(f"layer {layer} has no tokens to store: it has stored those of the last extend already, or rows have been moved or cut since")
        if not self._replayed and _capturing():
            self._replayed = True
        if (isinstance(keys, torch.Tensor) and isinstance(values, torch.Tensor) and keys.dim() == 4 and keys.shape[2] >= self._grown
                and _device() == self.device.index and _native.paged_write(_WRITE, self._at, self.device.index, layer, keys, values,
                                                                           _lib.stream_ptr(self.device))):
            self._written.add(layer)
            return
        self._check_layer(layer)
        for t, what in ((keys, "keys"), (values, "values")):
            if t.dim() != 4 or t.shape[0] != self.batch or t.shape[1] != self.kv_heads or t.shape[3] != HEAD_DIM:
                raise ValueError(f"{what} must be [{self.batch}, {self.kv_heads}, T, {HEAD_DIM}], got {tuple(t.shape)}")
            self._check_tensor(t, what)
        if keys.shape[2] != values.shape[2]:
            raise ValueError(f"{keys.shape[2]} keys and {values.shape[2]} values a row")
        if keys.shape[2] < self._grown:
            raise ValueError(f"{keys.shape[2]} tokens a row, but rows have grown by up to {self._grown}")
        keys, values = self._rows_ok(keys), self._rows_ok(values)
        self._call(lib.odmkv_pages_write, C.byref(self._p), layer, keys.data_ptr(), *keys.stride()[:3], values.data_ptr(), *values.stride()[:3],
                   keys.shape[2])
        self._written.add(layer)

    def append(self, keys: torch.Tensor, values: torch.Tensor, counts: Optional[Counts] = None) -> None:
        """``extend`` and ``write`` of a cache of one layer."""
        if self.layers != 1:
            raise ValueError("append is for caches of one layer: extend once, then write every layer")
        T = keys.shape[2] if keys.dim() == 4 else 0
        self.extend(T if counts is None else counts, bound=None if counts is None else T)
        self.write(0, keys, values)

    def _check_layer(self, layer: int) -> None:
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")

    def _check_stored(self, layer: int) -> None:
        """Raises where a layer has not stored the tokens of the last `extend`: its rows would be read with what lay in their places before."""
        if self._grown and layer not in self._written and not self._replayed:
            self._check_layer(layer)
            raise ValueError(f"layer {layer} has not stored the tokens of the last extend: write them first")

    def _check_tensor(self, t: torch.Tensor, what: str) -> None:
        _lib.require_gpu(t, what)
        if t.device != self.device:
            raise ValueError(f"{what} lie on {t.device}, the cache on {self.device}")
        if t.dtype != self.dtype:
            raise ValueError(f"{what} must be {self.dtype}, got {t.dtype}")

    @staticmethod
    def _rows_ok(t: torch.Tensor) -> torch.Tensor:
        """Rows of 128 that start on 16 bytes, copied where they do not.  (The stride of a dimension of one means nothing, and may be any number.)"""
        strides = [s if n > 1 else 0 for n, s in zip(t.shape, t.stride())]
        if t.stride(3) != 1 or any(s % 8 for s in strides[:3]) or t.data_ptr() % 16:
            return t.clone(memory_format=torch.contiguous_format)
        return t.as_strided(t.shape, (*strides[:3], 1)) if any(s % 8 for s in t.stride()[:3]) else t

    # ------------------------------------------------------------------ tokens out
    def read(self, layer: int = 0, tokens: Optional[int] = None, dtype: Optional[torch.dtype] = None):
        """Dense keys and values of one layer, [B, Hkv, tokens, 128] (default: the longest row's bound), 0 behind a row's length."""
        self._check_layer(layer)
        self._check_stored(layer)
        tokens = self.max_length if tokens is None else int(tokens)
        if tokens < 0:
            raise ValueError(f"tokens must not be negative, got {tokens}")
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _lib._DT:
            raise ValueError(f"unsupported dtype {dtype}; expected float16, bfloat16 or float32")
        keys, values = (torch.empty(self.batch, self.kv_heads, tokens, HEAD_DIM, dtype=dtype, device=self.device) for _ in range(2))
        if tokens:
            self._call(lib.odmkv_pages_read, C.byref(self._p), layer, keys.data_ptr(), values.data_ptr(), _lib._DT[dtype], tokens)
        return keys, values

    def attend(self, layer: int, query: torch.Tensor, *, scaling: Optional[float] = None, softcap: Optional[float] = None,
               slopes: Optional[torch.Tensor] = None, window: Optional[int] = None, prefix: Optional[torch.Tensor] = None,
               starts: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None, return_lse: bool = False,
               longest: Optional[int] = None):
        """Attention of the newest tokens' queries, query [B, Hq, L, 128], over one layer, which holds those tokens already -> [B, L, Hq, 128] of
        the same type, and on request lse fp32 [B, Hq, L].

        Row b's query l of its n (`counts`, int32 [B]; default L, what lies behind n is neither read nor written) stands at position i = length - n + l and sees
        tokens lo <= j < hi: lo is its start (`starts`, int32 [B] or [B, L]: where a document or the text behind padding begins; default 0), and not before
        i - window + 1; hi is i + 1, or `prefix` (int32 [B]: tokens that everybody sees) where that is more, within the row; a query in front of
        the row (i < 0: more queries than tokens) sees nothing.  Scores are scaling * q.k
        (default 128 ** -0.5), then softcap * tanh(x / softcap), then less slope * |i - j| (`slopes`, fp32 [Hq]).  Queries that see nothing
        get 0, and -inf for lse.

        `longest`: about how long the longest row is, which decides how the work is cut and nothing else (default: the host's bound, and while a graph is captured
        max_tokens, since the rows may be that long at a replay)."""
        self._check_stored(layer)
        if longest is None:
            longest = self.max_tokens if _capturing() else max(self._bounds)
        elif longest < 0:
            raise ValueError(f"longest must not be negative, got {longest}")
        longest = min(longest, self.max_tokens)
        if _device() == self.device.index and isinstance(query, torch.Tensor) and (softcap is None or _LEAST_CAP <= softcap < math.inf) and (window is None or window >= 1):
            # (everything as the kernels take it: one native call)
            done = _native.paged_attend(_ATTEND, _ATTEND_BYTES, self._at, self.device.index, layer, query, _SCALING if scaling is None else scaling,
                                        0.0 if softcap is None else softcap, 0 if window is None else min(window, _FAR), longest, return_lse,
                                        counts, slopes, prefix, starts, _lib.stream_ptr(self.device))
            if done is not None:
                return done
        self._check_layer(layer)
        if query.dim() != 4 or query.shape[0] != self.batch or query.shape[3] != HEAD_DIM:
            raise ValueError(f"query must be [{self.batch}, Hq, L, {HEAD_DIM}], got {tuple(query.shape)}")
        self._check_tensor(query, "queries")
        B, Hq, L, _ = query.shape
        if Hq == 0 or Hq % self.kv_heads or Hq // self.kv_heads > MAX_GROUP:
            raise ValueError(f"{Hq} query heads over {self.kv_heads} kv heads: groups of 1 to {MAX_GROUP} are built")
        if softcap is not None and not _LEAST_CAP <= softcap < math.inf:
            raise ValueError(f"softcap must be positive, at least 2 ** -100, got {softcap}")
        if window is not None and window < 1:
            raise ValueError(f"window must be positive, got {window}")
        scaling = _SCALING if scaling is None else float(scaling)
        query = self._rows_ok(query)
        slopes = self._small(slopes, "slopes", torch.float32, ((Hq,),))
        prefix = self._small(prefix, "prefix", torch.int32, ((B,),))
        counts = self._small(counts, "counts", torch.int32, ((B,),))
        starts = self._small(starts, "starts", torch.int32, ((B,), (B, L)))
        make = torch.empty if counts is None else torch.zeros
        out = make(B, L, Hq, HEAD_DIM, dtype=query.dtype, device=self.device)
        lse = make(B, Hq, L, dtype=torch.float32, device=self.device) if return_lse else None
        if L:
            nbytes = lib.odmkv_pages_attend_workspace_bytes(C.byref(self._p), Hq, L, longest)
            # (of its own for every call: two graphs that share one would race, and a graph's is the graph's)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
            a = _lib.Attend(C.pointer(self._p), query.data_ptr(), *query.stride()[:3], out.data_ptr(), _lib.ptr(lse), _lib.ptr(counts), _lib.ptr(slopes),
                            _lib.ptr(prefix), _lib.ptr(starts), 0 if starts is None else starts.stride(0),
                            0 if starts is None or starts.dim() == 1 else starts.stride(1), _lib.ptr(ws), nbytes, layer, L, Hq, min(window or 0, _FAR), longest,
                            scaling, 0.0 if softcap is None else float(softcap))
            self._call(lib.odmkv_pages_attend, C.byref(a))
        return (out, lse) if return_lse else out

    def _small(self, t, what: str, dtype: torch.dtype, shapes):
        """A small operand on the cache's device, of its type and contiguous."""
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or tuple(t.shape) not in shapes:
            raise ValueError(f"{what} must be {' or '.join(str(list(s)) for s in shapes)}, got {tuple(getattr(t, 'shape', ())) or type(t).__name__}")
        if t.device != self.device:
            raise ValueError(f"{what} lie on {t.device}, the cache on {self.device}")
        if dtype == torch.int32 and (t.is_floating_point() or t.is_complex() or t.dtype == torch.bool):
            raise ValueError(f"{what} must be whole numbers, got {t.dtype}")
        return (_as(t, dtype) if dtype == torch.int32 else t.to(dtype)).contiguous()

    # ------------------------------------------------------------------ rows
    def reorder(self, parents) -> None:
        """Row b becomes a copy of row parents[b], all at once (beam search, samples of one prompt): full blocks are shared, tails copied.
        `parents`: a list, or whole numbers on the device (an index out of range is then refused there: see ``refresh``)."""
        on_device, host, known = self._parents(parents, self.batch)
        if known is None:                                    # indices that only the device knows
            if min(self._bounds) < self.max_length:          # (rows of one length stay that)
                self._bounds[:] = [self.max_length] * self.batch
                self._loose = True
        else:
            self._bounds[:] = [self._bounds[b] for b in known]
        self._used_at_most()
        self._nothing_to_write()
        nbytes = lib.odmkv_pages_reorder_workspace_bytes(self.batch)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self._call(lib.odmkv_pages_reorder, C.byref(self._p), _lib.ptr(on_device), host, ws.data_ptr(), nbytes)

    def select(self, parents) -> "PagedKVCache":
        """A batch of its own over the same pages, whose row b is a copy of this one's row parents[b]; this one's rows stay (``release`` it where it is
        not needed; the pages of a batch that is dropped come back with the next ``extend``, ``refresh`` or ``compacted`` over the pool).  Both batches draw on the one pool."""
        if _capturing():
            raise RuntimeError("select makes a new batch, whose pages every replay of a captured one would take again: call it outside, and capture what the batch goes on with")
        n = int(parents.shape[0]) if isinstance(parents, torch.Tensor) and parents.dim() == 1 else len(parents)
        if not 1 <= n <= MAX_ROWS:
            raise ValueError(f"a batch must be 1 to {MAX_ROWS} rows, got {n}")
        on_device, host, known = self._parents(parents, n)
        if on_device is None:
            on_device = torch.tensor(known, dtype=torch.int64).to(self.device)
        new = self._sibling(n)
        for name in ("pages", "k_codes", "v_codes", "k_scale", "v_scale", "refs", "status", "_shared"):
            setattr(new, name, getattr(self, name))
        new._make_rows()
        for t in (new.table, new.length, new.start):
            t.zero_()
        new.slot.copy_(torch.arange(n, dtype=torch.int32, device=self.device))
        new._struct()
        new._nothing_to_write()
        new._bounds[:] = [self.max_length] * n if known is None else [self._bounds[b] for b in known]
        new._loose = self._loose or known is None
        nbytes = lib.odmkv_pages_reorder_workspace_bytes(n)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self._call(lib.odmkv_pages_select, C.byref(self._p), C.byref(new._p), on_device.data_ptr(), ws.data_ptr(), nbytes)
        return new

    def _parents(self, parents, n: int):
        on_device, host, known = self._ints(parents, n, torch.int64, "parents")
        if known is not None and not (0 <= min(known) and max(known) < self.batch):
            raise ValueError(f"parents must be rows 0 to {self.batch - 1}, got {min(known)} to {max(known)}")
        return on_device, host, known

    def truncate(self, lengths: Counts, rows: Optional[Sequence[int]] = None) -> None:
        """Rows shrink to a length (one for all, a list of one a row, or int32 on the device); rows that are not longer stay as they are.  A full block that is
        cut becomes the tail, as the values its codes stand for.  `rows`: the rows meant (default all)."""
        mask = None
        if rows is not None:
            mask = (C.c_uint32 * (MAX_ROWS // 32))()
            for b in rows:
                if not 0 <= b < self.batch:
                    raise ValueError(f"row {b} of {self.batch}")
                mask[b >> 5] |= 1 << (b & 31)
        meant = range(self.batch) if rows is None else set(rows)
        if isinstance(lengths, int):
            on_device, host, known = None, None, [lengths] * self.batch
        else:
            on_device, host, known = self._ints(lengths, self.batch, torch.int32, "lengths")
        if known is not None and min(known) < 0:
            raise ValueError(f"a length must not be negative, got {min(known)}")
        self._call(lib.odmkv_pages_truncate, C.byref(self._p), _lib.ptr(on_device), host, min(lengths, self.max_tokens) if isinstance(lengths, int) else 0, mask)
        self._nothing_to_write()
        if known is not None:
            for b in meant:
                self._bounds[b] = min(self._bounds[b], known[b])
        else:
            self._loose = True
        if not any(self._bounds):
            self._loose = False
        self._used_at_most()

    def free(self, rows: Optional[Sequence[int]] = None) -> None:
        """Rows (default all) hold nothing any more."""
        self.truncate(0, rows)

    def release(self) -> None:
        """Frees all rows and leaves the pool to the batches that share it: this one is not used any more."""
        self.free()
        self._dropped.detach()
        self._shared["bounds"] = [bounds for bounds in self._shared["bounds"] if bounds is not self._bounds]

    def _used_at_most(self) -> None:
        self._shared["used"] = min(self._shared["used"], sum(n // BLOCK for bounds in self._shared["bounds"] for n in bounds))

    # ------------------------------------------------------------------ the pool
    def compacted(self, pages: Optional[int] = None) -> "PagedKVCache":
        """A copy with a pool of its own of `pages` pages (default: those in use, read back from the device), in which the pages in use lie one behind the other:
        to give memory back, or to have more of it.  This cache stays as it is until it is dropped."""
        self._take_back()
        if any(any(bounds) for bounds in self._shared["bounds"] if bounds is not self._bounds):
            raise ValueError("the pool is shared with another batch (select): its pages cannot be renumbered for this one alone")
        if pages is None or self._shared["used"] > pages:
            self.refresh()
        pages = max(self._shared["used"], 1) if pages is None else int(pages)
        if pages < max(self._shared["used"], 1):
            raise ValueError(f"{self._shared['used']} pages are in use, a pool of {pages} does not hold them")
        new = self._sibling(self.batch)
        new._make_pool(pages)
        new._make_rows()
        new._struct()
        new._bounds[:], new._loose = self._bounds, self._loose
        new._grown, new._written = self._grown, set(self._written)       # (what is still to be stored can be stored there)
        new._shared["used"] = self._shared["used"]
        nbytes = lib.odmkv_pages_compact_workspace_bytes(self.pages)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self._call(lib.odmkv_pages_compact, C.byref(self._p), C.byref(new._p), ws.data_ptr(), nbytes)
        return new
