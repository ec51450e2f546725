"""Norm of every query and key head and position rotation in one pass, with
its gradients, and fused with the quantised cache write of a serving step
(extension: breccia has no operator of the attention block).

For a head ``x`` of ``d`` elements: ``r = (mean(x^2) + eps)^-1/2``, ``z = x r
w``, and the first ``2 * cos.shape[1]`` elements of ``z`` are rotated by the
token's angles, pairs ``(i, i + half)`` or, interleaved, ``(2i, 2i + 1)``.
Arithmetic is float32 with one rounding into the result.
"""

from __future__ import annotations

import ctypes
from typing import Tuple

import torch

from . import _lib
from .api import _IN_DT, _require_cuda
from .kvcache import QuantizedKVCache, _call, _heads, _index, _no_grad

__all__ = ["qk_norm_rope", "qk_norm_rope_write"]


def _vector(w, what, d, dev):
    _require_cuda(w, what)
    if w.dtype not in _IN_DT:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {w.dtype}")
    if tuple(w.shape) != (d,):
        raise ValueError(f"{what} must have shape ({d},), got {tuple(w.shape)}")
    if w.device != dev:
        raise ValueError(f"{what} is on {w.device}, expected {dev}")
    w = w.contiguous()
    return w.clone() if w.data_ptr() % 16 else w


def _angles(t, what, dev):
    _require_cuda(t, what)
    if t.dtype != torch.float32:
        raise TypeError(f"{what} must be float32, got {t.dtype}")
    if t.ndim != 2 or t.shape[0] == 0:
        raise ValueError(f"{what} must be (positions, rotated / 2), got {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"{what} is on {t.device}, expected {dev}")
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _arguments(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    """The C ABI's argument record, and what it points to (kept alive by the
    caller until the launch)."""
    q = _heads(q, "q")
    dev = q.device
    k = _heads(k, "k", dev)
    tokens, hq, d = q.shape
    if k.shape[0] != tokens or k.shape[2] != d or k.dtype != q.dtype:
        raise ValueError(f"q and k differ: {tuple(q.shape)} {q.dtype}, {tuple(k.shape)} {k.dtype}")
    if d % 16 or not 16 <= d <= 256:
        raise ValueError(f"head_dim must be a multiple of 16 up to 256, got {d}")
    wq, wk = _vector(q_weight, "q_weight", d, dev), _vector(k_weight, "k_weight", d, dev)
    if wq.dtype != wk.dtype:
        raise TypeError(f"q_weight and k_weight differ: {wq.dtype}, {wk.dtype}")
    cos, sin = _angles(cos, "cos", dev), _angles(sin, "sin", dev)
    rot = 2 * cos.shape[1]
    if cos.shape != sin.shape:
        raise ValueError(f"cos and sin differ: {tuple(cos.shape)}, {tuple(sin.shape)}")
    if rot % 16 or not 16 <= rot <= d:
        raise ValueError(f"the rotated width must be a multiple of 16 up to head_dim={d}, got {rot}")
    positions, is64 = _index(positions, "positions", tokens, dev)
    a = _lib.NormRope(q.data_ptr(), k.data_ptr(), q.stride(0), q.stride(1), k.stride(0),
                      k.stride(1), wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                      positions.data_ptr(), tokens, cos.shape[0], hq, k.shape[1], d, rot,
                      _IN_DT[q.dtype], _IN_DT[wq.dtype], is64, int(bool(interleaved)), eps)
    return a, (q, k, wq, wk, cos, sin, positions)


def _forward(a, keep):
    q, k = keep[0], keep[1]
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=q.device)
    _call(q.device, "brc_qk_norm_rope", ctypes.addressof(a), q_out.data_ptr(), k_out.data_ptr())
    return q_out, k_out


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        a, keep = _arguments(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
        ctx.save_for_backward(*keep)
        ctx.shapes = q.shape, k.shape
        ctx.eps, ctx.interleaved = eps, interleaved
        q_out, k_out = _forward(a, keep)
        return q_out.view(q.shape), k_out.view(k.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        a, keep = _arguments(q, k, wq, wk, cos, sin, positions, ctx.eps, ctx.interleaved)
        gq, gk = _heads(gq.to(q.dtype), "gradient"), _heads(gk.to(k.dtype), "gradient")
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=q.device)
        dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
        nbytes = _lib.lib().brc_qk_norm_rope_bwd_workspace(q.shape[2])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        _call(q.device, "brc_qk_norm_rope_bwd", ctypes.addressof(a), gq.data_ptr(), gk.data_ptr(),
              gq.stride(0), gq.stride(1), gk.stride(0), gk.stride(1), dq.data_ptr(), dk.data_ptr(),
              dwq.data_ptr(), dwk.data_ptr(), ws.data_ptr(), nbytes)
        return (dq.view(ctx.shapes[0]), dk.view(ctx.shapes[1]), dwq, dwk, None, None, None, None,
                None)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
                 eps: float = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Norm and rotate the heads of ``q (..., heads, d)`` and ``k (...,
    kv_heads, d)`` (views with strides, such as slices of a packed projection,
    are read in place), differentiable in ``q``, ``k`` and the weights.

    ``q_weight``, ``k_weight``: ``(d,)``, of one dtype. ``cos``, ``sin``:
    float32 ``(table, rotated / 2)`` with ``rotated`` at most ``d``.
    ``positions``: one int32 or int64 per token; a position outside the table
    gives a row of NaN. ``d`` and ``rotated`` are multiples of 16, ``d`` at
    most 256. Returns new ``q`` and ``k`` of the inputs' dtype and shape."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad or
                                    k_weight.requires_grad):
        return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    a, keep = _arguments(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    q_out, k_out = _forward(a, keep)
    return q_out.view(q.shape), k_out.view(k.shape)


def qk_norm_rope_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor,
                       k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                       positions: torch.Tensor, cache: QuantizedKVCache, slots: torch.Tensor, *,
                       eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """A serving step's ``qk_norm_rope`` and ``cache.write`` in one launch:
    returns the new ``q`` and leaves the cache as ``cache.write(k', v, slots)``
    of the normed and rotated ``k'`` (rounded to its dtype) leaves it.
    bfloat16 or float16; no gradient."""
    if not isinstance(cache, QuantizedKVCache):
        raise TypeError(f"cache must be a QuantizedKVCache, got {type(cache).__name__}")
    _no_grad("qk_norm_rope_write", q, k, v, q_weight, k_weight)
    a, keep = _arguments(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    q2, k2 = keep[0], keep[1]
    if q2.dtype == torch.float32:
        raise TypeError("qk_norm_rope_write takes bfloat16 or float16")
    if k2.device != cache.device:
        raise ValueError(f"k is on {k2.device}, expected {cache.device}")
    cache._rows(k2, "k")
    v2 = cache._rows(v, "v")
    if v2.shape[0] != k2.shape[0] or v2.dtype != k2.dtype:
        raise ValueError(f"k and v differ: {tuple(k2.shape)} {k2.dtype}, "
                         f"{tuple(v2.shape)} {v2.dtype}")
    slots, is64 = _index(slots, "slots", k2.shape[0], cache.device)
    q_out = torch.empty(q2.shape, dtype=q2.dtype, device=q2.device)
    _call(q2.device, "brc_qk_norm_rope_write", ctypes.addressof(a), v2.data_ptr(), v2.stride(0),
          v2.stride(1), q_out.data_ptr(), cache._desc, slots.data_ptr(), is64)
    return q_out.view(q.shape)
