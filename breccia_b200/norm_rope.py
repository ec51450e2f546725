"""Norm of every query and key head and position rotation in one pass, with
its gradients, and fused with the quantised cache write of a serving step
(extension: breccia has no operator of the attention block).

For a head ``x`` of ``d`` elements: ``r = (mean(x^2) + eps)^-1/2``, ``z = x r
w``, and the first ``2 * cos.shape[1]`` elements of ``z`` are rotated by the
token's angles, pairs ``(i, i + half)`` or, interleaved, ``(2i, 2i + 1)``.
Arithmetic is float32 with one rounding into the result.
"""

from __future__ import annotations

from ctypes import addressof
from typing import Tuple

import torch

from . import _lib
from .api import _IN_DT
from .kvcache import (QuantizedKVCache, _Entry, _heads, _in_dual_level, _index, _like, _no_grad,
                      _on)

__all__ = ["qk_norm_rope", "qk_norm_rope_write"]

_norm_rope, _norm_rope_bwd, _norm_rope_write = (_Entry(n) for n in (
    "brc_qk_norm_rope", "brc_qk_norm_rope_bwd", "brc_qk_norm_rope_write"))


def _plain(t):
    """Contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _check_parameters(wq, wk, cos, sin, d, dev):
    """The parameters' checks, message by message."""
    for w, what in ((wq, "q_weight"), (wk, "k_weight")):
        _on(w, what, dev)
        if w.dtype not in _IN_DT:
            raise TypeError(f"{what} must be float32, bfloat16 or float16, got {w.dtype}")
        if w.shape != (d,):
            raise ValueError(f"{what} must have shape ({d},), got {tuple(w.shape)}")
    if wq.dtype is not wk.dtype:
        raise TypeError(f"q_weight and k_weight differ: {wq.dtype}, {wk.dtype}")
    for t, what in ((cos, "cos"), (sin, "sin")):
        _on(t, what, dev)
        if t.dtype is not torch.float32:
            raise TypeError(f"{what} must be float32, got {t.dtype}")
    if cos.shape != sin.shape:
        raise ValueError(f"cos and sin differ: {tuple(cos.shape)}, {tuple(sin.shape)}")
    if cos.ndim != 2 or cos.shape[0] == 0:
        raise ValueError(f"cos must be (positions, rotated / 2), got {tuple(cos.shape)}")
    rot = 2 * cos.shape[1]
    if rot % 16 or not 16 <= rot <= d:
        raise ValueError(f"the rotated width must be a multiple of 16 up to head_dim={d}, got {rot}")


_F32 = torch.float32


def _arguments(q, k, wq, wk, cos, sin, positions, eps, interleaved):
    """The C ABI's argument record, and what it points to (kept alive by the
    caller until the launch)."""
    q = _heads(q, "q")
    dev = q.device
    k = _heads(k, "k", dev)
    tokens, hq, d = q.shape
    k_tokens, hk, k_d = k.shape
    dtype = q.dtype
    if k_tokens != tokens or k_d != d or k.dtype is not dtype:
        raise ValueError(f"q and k differ: {tuple(q.shape)} {dtype}, {tuple(k.shape)} {k.dtype}")
    if d % 16 or not 16 <= d <= 256:
        raise ValueError(f"head_dim must be a multiple of 16 up to 256, got {d}")
    try:  # all at once (a single token's call is bound by the host)
        w_dtype, rows = wq.dtype, cos.shape
        fine = (w_dtype is wk.dtype and w_dtype in _IN_DT and wq.shape == wk.shape == (d,) and
                cos.dtype is _F32 and sin.dtype is _F32 and rows == sin.shape and
                len(rows) == 2 and rows[0] > 0 and rows[1] % 8 == 0 and 0 < 2 * rows[1] <= d and
                wq.device == wk.device == cos.device == sin.device == dev)
    except AttributeError:
        fine = False
    if not fine:
        _check_parameters(wq, wk, cos, sin, d, dev)
    pwq, pwk, pc, ps = wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr()
    if (pwq | pwk | pc | ps) % 16 or not (wq.is_contiguous() and wk.is_contiguous() and
                                          cos.is_contiguous() and sin.is_contiguous()):
        wq, wk, cos, sin = _plain(wq), _plain(wk), _plain(cos), _plain(sin)
        pwq, pwk, pc, ps = wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr()
    positions, is64 = _index(positions, "positions", tokens, dev)
    qs, ks = q.stride(), k.stride()
    a = _lib.NormRope(q.data_ptr(), k.data_ptr(), qs[0], qs[1], ks[0], ks[1], pwq, pwk, pc, ps,
                      positions.data_ptr(), tokens, rows[0], hq, hk, d, 2 * rows[1], _IN_DT[dtype],
                      _IN_DT[w_dtype], is64, 1 if interleaved else 0, eps)
    return a, q, k, (wq, wk, cos, sin, positions)


def _forward(a, q, k):
    q_out, k_out = _like(q), _like(k)
    _norm_rope(q.get_device(), addressof(a), q_out.data_ptr(), k_out.data_ptr())
    return q_out, k_out


def _shaped(t, like):
    return t if t.ndim == like.ndim else t.view(like.shape)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, eps, interleaved):
        a, q3, k3, rest = _arguments(q, k, wq, wk, cos, sin, positions, eps, interleaved)
        ctx.save_for_backward(q3, k3, *rest)
        ctx.record, ctx.shapes = a, (q.shape, k.shape)
        q_out, k_out = _forward(a, q3, k3)
        return _shaped(q_out, q), _shaped(k_out, k)

    @staticmethod
    def backward(ctx, gq, gk):
        # under create_graph the result is marked as not differentiable again;
        # without it there is nothing to mark (and the mark costs 5 us)
        return _backward_once(ctx, gq, gk) if torch.is_grad_enabled() else _backward(ctx, gq, gk)


def _backward(ctx, gq, gk):
    q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
    # what was saved may have been moved meanwhile (saved-tensor hooks)
    a = _lib.NormRope.from_buffer_copy(ctx.record)
    a.q, a.k, a.wq, a.wk = q.data_ptr(), k.data_ptr(), wq.data_ptr(), wk.data_ptr()
    a.cos, a.sin, a.positions = cos.data_ptr(), sin.data_ptr(), positions.data_ptr()
    a.q_token, a.q_head, _ = q.stride()
    a.k_token, a.k_head, _ = k.stride()
    gq, gk = _heads(gq, "gradient"), _heads(gk, "gradient")
    dq, dk, dwq, dwk = _like(q), _like(k), _like(wq), _like(wk)
    nbytes = _lib.lib().brc_qk_norm_rope_bwd_workspace(a.d)
    ws = q.new_empty(nbytes, dtype=torch.uint8)
    gqs, gks = gq.stride(), gk.stride()
    _norm_rope_bwd(q.get_device(), addressof(a), gq.data_ptr(), gk.data_ptr(), gqs[0], gqs[1],
                   gks[0], gks[1], dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(), dwk.data_ptr(),
                   ws.data_ptr(), nbytes)
    if len(ctx.shapes[0]) != 3:
        dq = dq.view(ctx.shapes[0])
    if len(ctx.shapes[1]) != 3:
        dk = dk.view(ctx.shapes[1])
    return dq, dk, dwq, dwk, None, None, None, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


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
    most 256. Returns new ``q`` and ``k`` of the inputs' dtype and shape. Forward-mode
    derivatives are refused."""
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad or
                                     k_weight.requires_grad)) or _in_dual_level():
        # (with a forward-mode tangent autograd refuses: there is no such derivative here)
        return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    a, q3, k3, _rest = _arguments(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    q_out, k_out = _forward(a, q3, k3)
    return _shaped(q_out, q), _shaped(k_out, k)


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
    a, q3, k3, _rest = _arguments(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    if q3.dtype is torch.float32:
        raise TypeError("qk_norm_rope_write takes bfloat16 or float16")
    cache._rows(k3, "k")
    v3 = cache._rows(v, "v")
    if v3.shape != k3.shape or v3.dtype is not k3.dtype:
        raise ValueError(f"k and v differ: {tuple(k3.shape)} {k3.dtype}, "
                         f"{tuple(v3.shape)} {v3.dtype}")
    slots, is64 = _index(slots, "slots", k3.shape[0], cache.device)
    q_out = _like(q3)
    vs = v3.stride()
    _norm_rope_write(cache._device_index, addressof(a), v3.data_ptr(), vs[0], vs[1],
                     q_out.data_ptr(), cache._desc, slots.data_ptr(), is64)
    return _shaped(q_out, q)
