"""A paged key/value cache held in breccia's recipes, and attention over it
(extension: breccia casts tensors and has no cache).

* :class:`QuantizedKVCache` -- keys and values quantised as they are written
  (``write``), read back as dense tensors (``read``). A cached row (one token,
  one head) holds exactly the codes and scales that ``cast`` gives for it
  (``Float8BlockScaling`` with ``block_k`` = the head dimension,
  ``MXFP8BlockScaling``, ``NVFP4BlockScaling``; jvoltci/breccia v0.1.3,
  ``src/breccia/kernels/reference/cast.py:384-404, 420-446, 468-496``).
* :func:`cache_attention` -- attention of the newest token of every sequence,
  or of a tree of drafted tokens, straight from the codes.

Slots, page tables and lengths live on the device and are not read by the
host, so every call can be captured in a CUDA graph.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .api import _IN_DT, _require_cuda

__all__ = ["QuantizedKVCache", "cache_attention"]

_FMT = {"E4M3": _lib.FP8_E4M3, "E5M2": _lib.FP8_E5M2}
_HEAD_DIMS = (64, 128, 256)
# elements in 16 bytes
_VEC = {torch.float32: 4, torch.bfloat16: 8, torch.float16: 8}
# Single-token calls are bound by the host: these read the current device and
# its stream without the wrappers around them (0.2 us against 1 to 2 us).
_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream
_CONTIGUOUS = torch.contiguous_format


class _Entry:
    """A C entry point, called on a device's current stream with that device
    current: ``entry(index, *arguments without the stream)``."""

    __slots__ = ("name", "fn")

    def __init__(self, name: str):
        self.name, self.fn = name, None

    def __call__(self, index: int, *args) -> None:
        fn = self.fn
        if fn is None:
            fn = self.fn = getattr(_lib.lib(), self.name)
        if index == _current_device():
            rc = fn(*args, _current_stream(index))
        else:
            with torch.cuda.device(index):
                rc = fn(*args, _current_stream(index))
        if rc:
            _lib.check(self.name, rc)


_kv_write, _kv_read, _kv_attention = (_Entry(n) for n in
                                      ("brc_kv_write", "brc_kv_read", "brc_kv_attention"))


def _like(x: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor like ``x`` (the cheapest allocation
    there is from Python)."""
    return torch.empty_like(x, memory_format=_CONTIGUOUS)


def _no_grad(what: str, *tensors) -> None:
    """A serving call has no derivatives: it refuses rather than cut a graph, or drop a
    forward-mode tangent, silently."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
    if _in_dual_level():
        for t in tensors:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward-mode derivative")


def _in_dual_level() -> bool:
    """Whether forward-mode tangents are carried here (under torch.no_grad() they are)."""
    return forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()


def _on(t: torch.Tensor, what: str, dev) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _require_cuda(t, what)
    if t.device != dev:
        raise ValueError(f"{what} is on {t.device}, expected {dev}")


def _heads(x: torch.Tensor, what: str, dev=None) -> torch.Tensor:
    """``(..., heads, d)`` as ``(tokens, heads, d)`` with the last axis
    contiguous and every row 16-byte aligned; a copy only where it is not."""
    if dev is None:
        _require_cuda(x, what)
    else:
        _on(x, what, dev)
    n = _VEC.get(x.dtype)
    if n is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {x.dtype}")
    if x.ndim != 3:
        if x.ndim < 2:
            raise ValueError(f"{what} must be (..., heads, head_dim), got shape {tuple(x.shape)}")
        x = x.reshape(math.prod(x.shape[:-2]), x.shape[-2], x.shape[-1])
    st, sh, sd = x.stride()
    if sd != 1 or (st | sh) % n:
        x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone(memory_format=_CONTIGUOUS)
    return x


def _index(t: torch.Tensor, what: str, n: int, dev) -> Tuple[torch.Tensor, int]:
    """A device index tensor of ``n`` elements, and whether it is int64."""
    _on(t, what, dev)
    dt = t.dtype
    if dt is not torch.int64 and dt is not torch.int32:
        raise TypeError(f"{what} must be int32 or int64, got {dt}")
    if t.numel() != n:
        raise ValueError(f"{what} must have one entry per token ({n}), got {t.numel()}")
    return t.contiguous(), 1 if dt is torch.int64 else 0


def _lengths(t: torch.Tensor, what: str, batch: int, dev) -> torch.Tensor:
    _on(t, what, dev)
    if t.dtype is not torch.int32:
        raise TypeError(f"{what} must be int32, got {t.dtype}")
    if t.shape != (batch,):
        raise ValueError(f"{what} must have shape ({batch},), got {tuple(t.shape)}")
    return t.contiguous()


def _table(t: torch.Tensor, batch: Optional[int], dev) -> torch.Tensor:
    _on(t, "page_table", dev)
    if t.dtype is not torch.int32:
        raise TypeError(f"page_table must be int32, got {t.dtype}")
    if t.ndim != 2 or (batch is not None and t.shape[0] != batch):
        want = "(batch, pages)" if batch is None else f"({batch}, pages)"
        raise ValueError(f"page_table must have shape {want}, got {tuple(t.shape)}")
    return t if t.stride(1) == 1 else t.contiguous()


def _recipe_kind(recipe: Any, head_dim: int):
    """(kind, fmt, code bytes per row, scales per row, scale dtype)."""
    name = getattr(recipe, "name", None)
    if name == "block":
        if recipe.block_k != head_dim:
            raise ValueError(f"a cached row has one scale: block_k={recipe.block_k} must equal "
                             f"head_dim={head_dim}")
        return _lib.STE_BLOCK_FP8, _FMT[recipe.fp8_format], head_dim, 1, torch.float32
    if name == "mxfp8":
        return _lib.STE_MXFP8, _FMT[recipe.fp8_format], head_dim, head_dim // 32, torch.uint8
    if name == "nvfp4":
        return _lib.STE_NVFP4, _lib.FP8_E4M3, head_dim // 2, head_dim // 16, torch.uint8
    raise TypeError(f"unsupported cache recipe: {type(recipe).__name__}")


class QuantizedKVCache:
    """``num_pages`` pages of ``page_size`` tokens for ``num_heads`` key/value
    heads of ``head_dim`` (64, 128 or 256), held in ``recipe``.

    Buffers, in the order (page, head, place in page): ``k_data`` / ``v_data``
    uint8 codes (``head_dim`` bytes per row; NVFP4 ``head_dim / 2``, element
    2i in the low nibble of byte i) and ``k_scale`` / ``v_scale`` (block FP8:
    one float32; MXFP8: ``head_dim / 32`` E8M0 bytes; NVFP4: ``head_dim / 16``
    E4M3 bytes). A token's slot is ``page * page_size + place``.
    ``page_size`` is a power of two of at least 16."""

    def __init__(self, num_pages: int, page_size: int, num_heads: int, head_dim: int, recipe: Any,
                 device: Any = None):
        if num_pages <= 0 or num_heads <= 0:
            raise ValueError(f"num_pages and num_heads must be > 0, got {num_pages}, {num_heads}")
        _, _, row, scales, sdt = self._check(page_size, head_dim, recipe)
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise TypeError(f"breccia_b200 operates on CUDA devices, got {dev}")
        data, scale = ((num_pages, num_heads, page_size, n) for n in (row, scales))
        self._bind(*(torch.zeros(s, dtype=t, device=dev) for s, t in
                     ((data, torch.uint8), (scale, sdt), (data, torch.uint8), (scale, sdt))),
                   recipe, head_dim)

    @classmethod
    def from_buffers(cls, k_data, k_scale, v_data, v_scale, recipe) -> "QuantizedKVCache":
        """A cache over existing buffers (no copy), in the layout above."""
        for t, what in ((k_data, "k_data"), (k_scale, "k_scale"), (v_data, "v_data"),
                        (v_scale, "v_scale")):
            _require_cuda(t, what)
            if t.ndim != 4 or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{what} must be a contiguous, 16-byte aligned 4-D tensor")
            if t.device != k_data.device:
                raise ValueError(f"{what} is on {t.device}, expected {k_data.device}")
        pages, heads, page_size, row = k_data.shape
        if pages <= 0 or heads <= 0:
            raise ValueError(f"k_data has no pages or heads: {tuple(k_data.shape)}")
        d = 2 * row if getattr(recipe, "name", None) == "nvfp4" else row
        _, _, row, scales, sdt = cls._check(page_size, d, recipe)
        for t, what, n, dt in ((k_data, "k_data", row, torch.uint8), (k_scale, "k_scale", scales, sdt),
                               (v_data, "v_data", row, torch.uint8), (v_scale, "v_scale", scales, sdt)):
            if t.dtype != dt:
                raise TypeError(f"{what} must be {dt}, got {t.dtype}")
            if tuple(t.shape) != (pages, heads, page_size, n):
                raise ValueError(f"{what} must have shape {(pages, heads, page_size, n)}, "
                                 f"got {tuple(t.shape)}")
        self = cls.__new__(cls)
        self._bind(k_data, k_scale, v_data, v_scale, recipe, d)
        return self

    @staticmethod
    def _check(page_size, head_dim, recipe):
        if head_dim not in _HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {head_dim}")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two >= 16, got {page_size}")
        return _recipe_kind(recipe, head_dim)

    def _bind(self, k_data, k_scale, v_data, v_scale, recipe, head_dim):
        self._buffers = (k_data, k_scale, v_data, v_scale)
        self.recipe = recipe
        self.num_pages, self.num_heads, self.page_size = k_data.shape[:3]
        self.head_dim = head_dim
        self.device = k_data.device
        self._device_index = self.device.index
        self._workspaces = {}  # (draft, heads): bytes, and what to allocate like
        kind, fmt = _recipe_kind(recipe, head_dim)[:2]
        self._struct = _lib.KvCache(k_data.data_ptr(), k_scale.data_ptr(), v_data.data_ptr(),
                                    v_scale.data_ptr(), self.num_pages, self.num_heads,
                                    self.page_size, head_dim, kind, fmt)
        self._desc = ctypes.addressof(self._struct)

    @property
    def k_data(self) -> torch.Tensor:
        return self._buffers[0]

    @property
    def k_scale(self) -> torch.Tensor:
        return self._buffers[1]

    @property
    def v_data(self) -> torch.Tensor:
        return self._buffers[2]

    @property
    def v_scale(self) -> torch.Tensor:
        return self._buffers[3]

    def __repr__(self) -> str:
        return (f"QuantizedKVCache(pages={self.num_pages}, page_size={self.page_size}, "
                f"heads={self.num_heads}, head_dim={self.head_dim}, "
                f"recipe={type(self.recipe).__name__})")

    def _rows(self, x, what):
        x = _heads(x, what, self.device)
        if x.shape[1] != self.num_heads or x.shape[2] != self.head_dim:
            raise ValueError(f"{what} must be (..., {self.num_heads}, {self.head_dim}), "
                             f"got {tuple(x.shape)}")
        return x

    def _workspace(self, draft: int, hq: int):
        """Scratch of one attention call, allocated anew on the current
        stream: calls of other streams, and of captured graphs, have their own."""
        ent = self._workspaces.get((draft, hq))
        if ent is None:
            # per device too: its size follows the number of multiprocessors
            with torch.cuda.device(self._device_index):
                nbytes = _lib.lib().brc_kv_attention_workspace(self._desc, 1, draft, hq)
            like = torch.empty(1, dtype=torch.uint8, device=self.device).expand(max(nbytes, 16))
            ent = self._workspaces[draft, hq] = (nbytes, like)
        return ent[0], _like(ent[1])

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise ``k`` and ``v`` ``(..., num_heads, head_dim)`` into the
        rows ``slots`` (one int32 or int64 slot per token). A slot outside the
        cache is not written: pad with -1. Slots of one call are distinct."""
        k, v = self._rows(k, "k"), self._rows(v, "v")
        _no_grad("QuantizedKVCache.write", k, v)
        if k.shape[0] != v.shape[0] or k.dtype != v.dtype:
            raise ValueError(f"k and v differ: {tuple(k.shape)} {k.dtype}, "
                             f"{tuple(v.shape)} {v.dtype}")
        slots, is64 = _index(slots, "slots", k.shape[0], self.device)
        ks, vs = k.stride(), v.stride()
        _kv_write(self._device_index, self._desc, k.data_ptr(), v.data_ptr(), _IN_DT[k.dtype],
                  k.shape[0], ks[0], ks[1], vs[0], vs[1], slots.data_ptr(), is64)

    def read(self, page_table: torch.Tensor, lengths: torch.Tensor, max_length: int,
             out_dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of a batch as dense ``(batch, max_length,
        num_heads, head_dim)`` tensors, ``decode(code) * scale`` rounded once.
        ``page_table``: int32 ``(batch, pages)``; ``lengths``: int32
        ``(batch,)``. Tokens past a sequence's length, past its table row or in
        a page outside the cache read as zero."""
        if out_dtype not in _IN_DT:
            raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
        if max_length < 0:
            raise ValueError(f"max_length must be >= 0, got {max_length}")
        table = _table(page_table, None, self.device)
        batch = table.shape[0]
        lengths = _lengths(lengths, "lengths", batch, self.device)
        shape = (batch, max_length, self.num_heads, self.head_dim)
        k = torch.empty(shape, dtype=out_dtype, device=self.device)
        v = _like(k)
        _kv_read(self._device_index, self._desc, table.data_ptr(), table.stride(0), table.shape[1],
                 lengths.data_ptr(), batch, max_length, k.data_ptr(), v.data_ptr(),
                 _IN_DT[out_dtype])
        return k, v


def cache_attention(q: torch.Tensor, cache: QuantizedKVCache, page_table: torch.Tensor,
                    context_lens: torch.Tensor, *, draft_lens: Optional[torch.Tensor] = None,
                    tree_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    return_lse: bool = False):
    """Attention of the newest tokens of every sequence over the cache.

    ``q``: ``(batch, heads, head_dim)`` for one token per sequence, or
    ``(batch, draft, heads, head_dim)`` for drafted tokens; bfloat16 or
    float16; ``heads`` a multiple of the cache's (query head ``i`` reads cache
    head ``i // (heads // num_heads)``). Sequence ``b`` holds
    ``context_lens[b]`` tokens before the drafted ones (for one token: before
    that token), whose own rows are already written behind them. ``page_table``
    is int32 ``(batch, pages)``.

    Every query sees the whole context. Drafted token ``i`` sees drafted token
    ``j`` where ``tree_mask[i, j]`` (bool, ``(draft, draft)`` or ``(batch,
    draft, draft)``; default ``j <= i``). ``draft_lens`` (int32, default all):
    how many of ``draft`` exist in each sequence; rows past it give 0.

    Returns ``softmax(scale q k^T) v`` in ``q``'s dtype and shape (``scale``
    defaults to ``head_dim ** -0.5``), and with ``return_lse`` also the
    float32 log-sum-exp of every row. A row that sees nothing gives 0 and
    ``-inf``; what it does not see, NaN included, does not reach it. Values more
    than ``2**60`` below the largest that a row sees (MXFP8: in the same 32
    elements) may vanish beside it, and values as small as the casts hold zeros
    (E4M3: below 6e-8; block FP8: 1e-10) count as zero beside larger ones.

    Many rows of a cache head run with bounded waits: if one runs out (2 s), rows
    stay unwritten and ``brc_gemm_status`` tells, as for the GEMMs. Scratch is
    allocated per call on the current stream, up to 40 MB."""
    if not isinstance(cache, QuantizedKVCache):
        raise TypeError(f"cache must be a QuantizedKVCache, got {type(cache).__name__}")
    dev = cache.device
    _on(q, "q", dev)
    _no_grad("cache_attention", q)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    shape = q.shape
    if len(shape) not in (3, 4) or shape[-1] != cache.head_dim or shape[-2] == 0 or \
            shape[-2] % cache.num_heads:
        raise ValueError(f"q must be (batch, [draft,] heads, {cache.head_dim}) with heads a "
                         f"multiple of {cache.num_heads}, got {tuple(shape)}")
    batch, hq = shape[0], shape[-2]
    draft = shape[1] if len(shape) == 4 else 1
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    table = _table(page_table, batch, dev)
    context = _lengths(context_lens, "context_lens", batch, dev)
    drafts = None if draft_lens is None else _lengths(draft_lens, "draft_lens", batch, dev)
    tree, tree_stride = None, 0
    if tree_mask is not None:
        _on(tree_mask, "tree_mask", dev)
        if tree_mask.dtype is not torch.bool:
            raise TypeError(f"tree_mask must be bool, got {tree_mask.dtype}")
        if tuple(tree_mask.shape) not in ((draft, draft), (batch, draft, draft)):
            raise ValueError(f"tree_mask must be ({draft}, {draft}) or ({batch}, {draft}, "
                             f"{draft}), got {tuple(tree_mask.shape)}")
        tree = tree_mask.contiguous()
        tree_stride = draft * draft if tree.ndim == 3 else 0
    out = _like(q)
    lse = torch.empty(shape[:-1], dtype=torch.float32, device=dev) if return_lse else None
    if out.numel():
        nbytes, ws = cache._workspace(draft, hq)
        _kv_attention(cache._device_index, cache._desc, q.data_ptr(), _IN_DT[q.dtype], batch,
                      draft, hq, table.data_ptr(), table.stride(0), table.shape[1],
                      context.data_ptr(), None if drafts is None else drafts.data_ptr(),
                      None if tree is None else tree.data_ptr(), tree_stride,
                      cache.head_dim ** -0.5 if scale is None else float(scale), out.data_ptr(),
                      None if lse is None else lse.data_ptr(), ws.data_ptr(), nbytes)
    return (out, lse) if return_lse else out
