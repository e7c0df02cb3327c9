"""Layers of the fusion block around the OT features, forward and backward, as HIP kernels.

The reference's model applies dropout, layer norm and a feed-forward block to the same fused
embeddings whose OT alignment ``fusion.ot_alignment_loss`` computes
(MRI_PET_OT_nojax.py:523-549,658-669; ``--projection-dropout``,
MRI_PET_OT_OT_per_epoch_attn.py:963-1065).  Here:

    dropout                  y = [residual +] keep * x / (1 - p), the mask never stored
    layer_norm               with the parameter gradients' reduction
    dropout_add_layer_norm   z = residual + dropout(x), y = LN(z), one pass over the rows
    gated_feed_forward       (act(x Wg^T) * (x Wu^T)) Wd^T on the matrix cores

Tensors live on a ROCm device; kernels run on the current stream of the tensors' device and
nothing synchronises, so every call can be captured into a graph.  Inputs are float32,
bfloat16 or float16; statistics and sums are float32.  Each function takes part in autograd;
without a gradient to compute, nothing is kept for backward.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from .ops import _EMB_DT

_NO_GUARD = contextlib.nullcontext()


def _on(device):
    """Kernels launch on the current device: make it the tensors' own."""
    return _NO_GUARD if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _input(t, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a ROCm device tensor")
    if t.dtype not in _EMB_DT:
        raise TypeError(f"{name}: float32, bfloat16 or float16, not {t.dtype}")
    return t


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """(..., cols) -> (rows, cols) with unit column stride and rows that do not overlap."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    return t if t.stride(1) == 1 and t.stride(0) >= cols else t.contiguous()


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _same_device(ref: torch.Tensor, **others):
    for name, t in others.items():
        if t is not None and t.device != ref.device:
            raise ValueError(f"{name} is on {t.device}, x on {ref.device}")


def _probability(p) -> float:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p} is not in [0, 1]")
    return p


def rng_state(seed: int, offset: int = 0, device="cuda") -> torch.Tensor:
    """The generator's state as the layers take it: a device int64 tensor ``[seed, offset]``.

    A mask is a function of (seed, offset, row, column, columns) alone.  Layers of one step that
    must not share a mask take different offsets (or seeds); between steps, advance the offset
    (``rng[1] += number_of_layers``) after backward: backward makes the mask again from the same
    tensor, and raises if it was changed in between.  Being read on the device, the state can
    advance between replays of a captured graph."""
    return torch.tensor([seed, offset], dtype=torch.int64, device=device)


def _rng(rng, x) -> torch.Tensor:
    if not isinstance(rng, torch.Tensor) or rng.dtype != torch.int64 or rng.shape != (2,) or not rng.is_contiguous():
        raise TypeError("rng must be a contiguous int64 tensor [seed, offset] (rng_state)")
    _same_device(x, rng=rng)
    return rng


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ----------------------------------------------------------------------------- dropout
def _dropout_call(x, residual, p, rng):
    shape, cols = x.shape, x.shape[-1] if x.dim() else 1
    if x.numel() == 0:
        return torch.empty(shape, dtype=x.dtype, device=x.device)
    x2 = _rows(x, cols)
    r2 = None if residual is None else _rows(residual, cols)
    y = torch.empty(x2.shape, dtype=x.dtype, device=x.device)
    with _on(x.device):
        L.check(L.lib().otf_dropout(x2.data_ptr(), _ld(x2), L.ptr(r2), 0 if r2 is None else _ld(r2), y.data_ptr(),
                                    cols, x2.shape[0], cols, _EMB_DT[x.dtype], p, rng.data_ptr(),
                                    L.stream_handle(x.device)), "otf_dropout")
    return y.view(shape)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng):
        ctx.save_for_backward(rng)
        ctx.p = p
        return _dropout_call(x, residual, p, rng)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        dx = _dropout_call(dy, None, ctx.p, rng) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``[residual +] dropout(x)`` (``--projection-dropout``).

    Each element is kept with probability ``1 - p`` (``p`` rounded to a multiple of 2^-16) and
    scaled by its inverse; a dropped one is exactly 0, whatever it held.  The mask comes from
    ``rng`` (see ``rng_state``) and the element's row and column and is made again in backward
    instead of being stored.  x: (..., cols); residual: the same shape and type."""
    _input(x, "x")
    if residual is not None:
        _input(residual, "residual")
        _same_device(x, residual=residual)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} differs from x {tuple(x.shape)} {x.dtype}")
    p, rng = _probability(p), _rng(rng, x)
    if _wants_grad(x, residual):
        return _Dropout.apply(x, residual, p, rng)
    return _dropout_call(x, residual, p, rng)


# -------------------------------------------------------------------------- layer norm
def _norm_params(x, weight, bias):
    """Checks, and the number of columns with the type that weight and bias share"""
    cols = x.shape[-1] if x.dim() else 0
    if cols == 0:
        raise ValueError(f"x {tuple(x.shape)}: layer norm needs a last dimension of at least 1")
    wdt = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _input(t, name)
        _same_device(x, **{name: t})
        if t.shape != (cols,):
            raise ValueError(f"{name} {tuple(t.shape)} must be ({cols},)")
        if t.dtype not in (x.dtype, torch.float32) or wdt not in (None, t.dtype):
            raise TypeError(f"weight and bias must share one type, x's ({x.dtype}) or float32")
        wdt = t.dtype
    return cols, wdt or torch.float32


def _dense(t):
    return None if t is None else t.detach().contiguous()


def _eps(eps) -> float:
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps {eps} must be finite and not negative")
    return eps


def _stats(rows: int, device):
    """Row means and inverse deviations for backward: the tensor and the two pointers"""
    s = torch.empty((2, rows), dtype=torch.float32, device=device)
    return s, s.data_ptr(), s.data_ptr() + 4 * rows


def _layer_norm_call(x2, weight, bias, wdt, eps, keep):
    rows, cols = x2.shape
    y = torch.empty((rows, cols), dtype=x2.dtype, device=x2.device)
    stats, mean, rstd = _stats(rows, x2.device) if keep else (None, None, None)
    if rows:
        with _on(x2.device):
            L.check(L.lib().otf_layer_norm(x2.data_ptr(), _ld(x2), _EMB_DT[x2.dtype], L.ptr(weight), L.ptr(bias),
                                           _EMB_DT[wdt], eps, rows, cols, y.data_ptr(), cols, mean, rstd,
                                           L.stream_handle(x2.device)), "otf_layer_norm")
    return y, stats


def _param_grads(cols, wdt, device, want_w, want_b):
    dw = torch.empty(cols, dtype=wdt, device=device) if want_w else None
    db = torch.empty(cols, dtype=wdt, device=device) if want_b else None
    return dw, db


def _scratch(size: int, device):
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _norm_workspace(rows, cols, device, wanted):
    size = L.lib().otf_layer_norm_backward_workspace_size(rows, cols) if wanted else 0
    return _scratch(size, device), size


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, cols, wdt):
        x2, w, b = _rows(x.detach(), cols), _dense(weight), _dense(bias)
        y, stats = _layer_norm_call(x2, w, b, wdt, eps, True)
        # a copied row layout is kept as copied; else the input itself, so that a change of it
        # before backward is noticed
        ctx.save_for_backward(x if x2.data_ptr() == x.data_ptr() else x2, weight, stats)
        ctx.cols, ctx.wdt = cols, wdt
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need, cols = ctx.needs_input_grad, ctx.cols
        x2, dy2, w = _rows(x, cols), _rows(dy, cols), _dense(weight)
        rows, dev = x2.shape[0], x2.device
        dx = torch.empty((rows, cols), dtype=x2.dtype, device=dev)
        dw, db = _param_grads(cols, ctx.wdt, dev, need[1], need[2])
        ws, size = _norm_workspace(rows, cols, dev, need[1] or need[2])
        with _on(dev):
            L.check(L.lib().otf_layer_norm_backward(
                dy2.data_ptr(), _ld(dy2), x2.data_ptr(), _ld(x2), _EMB_DT[x2.dtype], L.ptr(w), _EMB_DT[ctx.wdt],
                stats.data_ptr(), stats.data_ptr() + 4 * rows, rows, cols, dx.data_ptr(), cols, L.ptr(dw), L.ptr(db),
                L.ptr(ws), size, L.stream_handle(dev)), "otf_layer_norm_backward")
        return dx.view(dy.shape) if need[0] else None, dw, db, None, None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    (SelfAttentionBlock's norms, MRI_PET_OT_nojax.py:523-549).

    x: (..., cols); weight, bias: (cols,), of one type, x's or float32.  The gradients of
    weight and bias are sums in a fixed order: the same bits every call."""
    _input(x, "x")
    cols, wdt = _norm_params(x, weight, bias)
    eps = _eps(eps)
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps, cols, wdt)
    return _layer_norm_call(_rows(x, cols), _dense(weight), _dense(bias), wdt, eps, False)[0].view(x.shape)


def _add_norm_call(x2, r2, weight, bias, wdt, p, rng, eps, keep):
    rows, cols = x2.shape
    y = torch.empty((rows, cols), dtype=x2.dtype, device=x2.device)
    z = torch.empty((rows, cols), dtype=r2.dtype, device=x2.device)
    stats, mean, rstd = _stats(rows, x2.device) if keep else (None, None, None)
    if rows:
        with _on(x2.device):
            L.check(L.lib().otf_dropout_add_layer_norm(
                x2.data_ptr(), _ld(x2), _EMB_DT[x2.dtype], r2.data_ptr(), _ld(r2), _EMB_DT[r2.dtype], L.ptr(weight),
                L.ptr(bias), _EMB_DT[wdt], eps, p, rng.data_ptr(), rows, cols, y.data_ptr(), cols, z.data_ptr(), cols,
                mean, rstd, L.stream_handle(x2.device)), "otf_dropout_add_layer_norm")
    return y, z, stats


class _DropoutAddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, p, rng, eps, cols, wdt):
        ctx.set_materialize_grads(False)
        x2, r2 = _rows(x.detach(), cols), _rows(residual.detach(), cols)
        y, z, stats = _add_norm_call(x2, r2, _dense(weight), _dense(bias), wdt, p, rng, eps, True)
        z = z.view(x.shape)
        # a float32 z is the normalised sum itself; a rounded one is not: keep what it is the sum of
        kept = (z,) if z.dtype == torch.float32 else (x if x2.data_ptr() == x.data_ptr() else x2,
                                                       residual if r2.data_ptr() == residual.data_ptr() else r2)
        ctx.save_for_backward(weight, stats, rng, *kept)
        ctx.cols, ctx.wdt, ctx.p, ctx.dtype, ctx.rdtype = cols, wdt, p, x.dtype, z.dtype
        return y.view(x.shape), z

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dz):
        if dy is None and dz is None:
            return (None,) * 9
        weight, stats, rng, *kept = ctx.saved_tensors
        need, cols = ctx.needs_input_grad, ctx.cols
        shape, dev = (dz if dy is None else dy).shape, stats.device
        kept, w = [_rows(t, cols) for t in kept], _dense(weight)
        rows = stats.shape[1]
        if dy is None:
            dy = torch.zeros(shape, dtype=ctx.dtype, device=dev)
        dy2, dz2 = _rows(dy, cols), None if dz is None else _rows(dz, cols)
        dx = torch.empty((rows, cols), dtype=ctx.dtype, device=dev)
        dr = torch.empty((rows, cols), dtype=ctx.rdtype, device=dev)
        dw, db = _param_grads(cols, ctx.wdt, dev, need[2], need[3])
        ws, size = _norm_workspace(rows, cols, dev, need[2] or need[3])
        z2, x2, r2 = (kept[0], None, None) if len(kept) == 1 else (None, *kept)
        ld = lambda t: 0 if t is None else _ld(t)
        with _on(dev):
            L.check(L.lib().otf_dropout_add_layer_norm_backward(
                dy2.data_ptr(), _ld(dy2), L.ptr(dz2), ld(dz2), L.ptr(z2), ld(z2), L.ptr(x2), ld(x2), L.ptr(r2), ld(r2),
                _EMB_DT[ctx.dtype], _EMB_DT[ctx.rdtype], L.ptr(w), _EMB_DT[ctx.wdt], stats.data_ptr(),
                stats.data_ptr() + 4 * rows, ctx.p, rng.data_ptr(), rows, cols, dx.data_ptr(), cols, dr.data_ptr(),
                cols, L.ptr(dw), L.ptr(db), L.ptr(ws), size, L.stream_handle(dev)),
                "otf_dropout_add_layer_norm_backward")
        return (dx.view(shape) if need[0] else None, dr.view(shape) if need[1] else None, dw, db, None, None, None,
                None, None)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, p: float = 0.0, rng: torch.Tensor | None = None,
                           eps: float = 1e-5):
    """``z = residual + dropout(x)``, ``y = layer_norm(z)``; returns ``(y, z)``.

    residual and z: x's type or float32 (a 32-bit residual stream under 16-bit layers); y: x's
    type, of the float32 sum.  ``rng`` may be None where ``p`` is 0.  Backward keeps a float32 z,
    else x and residual."""
    _input(x, "x")
    _input(residual, "residual")
    _same_device(x, residual=residual)
    if residual.shape != x.shape:
        raise ValueError(f"residual {tuple(residual.shape)} differs from x {tuple(x.shape)}")
    if residual.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"residual must have x's type ({x.dtype}) or float32, not {residual.dtype}")
    cols, wdt = _norm_params(x, weight, bias)
    p, eps = _probability(p), _eps(eps)
    if rng is None:
        if p:
            raise ValueError("p > 0 needs rng (rng_state)")
        rng = torch.zeros(2, dtype=torch.int64, device=x.device)
    rng = _rng(rng, x)
    if _wants_grad(x, residual, weight, bias):
        return _DropoutAddLayerNorm.apply(x, residual, weight, bias, p, rng, eps, cols, wdt)
    y, z, _ = _add_norm_call(_rows(x, cols), _rows(residual, cols), _dense(weight), _dense(bias), wdt, p, rng, eps, False)
    return y.view(x.shape), z.view(x.shape)


# ------------------------------------------------------------------ gated feed-forward
_MAX_WIDTH = 1 << 20   # the kernels' row strides: 256 rows within a 31-bit byte offset


def _strided_rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """_rows, dense where the rows are further apart than the kernels take"""
    t = _rows(t, cols)
    return t if _ld(t) <= _MAX_WIDTH else t.contiguous()


def _pair(w_gate, w_up):
    """gate and up with one leading dimension"""
    a, b = _strided_rows(w_gate, w_gate.shape[1]), _strided_rows(w_up, w_up.shape[1])
    if _ld(a) != _ld(b):
        a, b = a.contiguous(), b.contiguous()
    return a, b


def _ffn_args(x2, w_gate, w_up, w_down, act) -> L.FfnArgs:
    a = L.FfnArgs()
    a.rows, a.d = x2.shape
    a.f = w_gate.shape[0]
    a.dtype, a.activation = _EMB_DT[x2.dtype], act
    a.x, a.ldx = x2.data_ptr(), _ld(x2)
    a.w_gate, a.w_up, a.ldw_in = w_gate.data_ptr(), w_up.data_ptr(), max(_ld(w_gate), _ld(w_up))
    a.w_down, a.ldw_down = w_down.data_ptr(), _ld(w_down)
    return a


def _ffn_call(x2, w_gate, w_up, w_down, act, keep):
    rows, d = x2.shape
    dev, lib = x2.device, L.lib()
    w_gate, w_up = _pair(w_gate, w_up)
    w_down = _strided_rows(w_down, w_down.shape[1])
    y = torch.empty((rows, d), dtype=x2.dtype, device=dev)
    a = _ffn_args(x2, w_gate, w_up, w_down, act)
    saved = torch.empty(lib.otf_gated_ffn_saved_size(rows, a.f, a.dtype), dtype=torch.uint8, device=dev) if keep else None
    a.y, a.ldy, a.saved = y.data_ptr(), d, L.ptr(saved)
    size = lib.otf_gated_ffn_workspace_size(ctypes.byref(a))
    ws = _scratch(size, dev)
    with _on(dev):
        L.check(lib.otf_gated_ffn(ctypes.byref(a), L.ptr(ws), size, L.stream_handle(dev)), "otf_gated_ffn")
    return y, saved


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act):
        d = x.shape[-1]
        y, saved = _ffn_call(_strided_rows(x.detach(), d), w_gate.detach(), w_up.detach(), w_down.detach(), act, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, saved)
        ctx.act = act
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_gate, w_up, w_down, saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        d = x.shape[-1]
        x2, dy2 = _strided_rows(x, d), _strided_rows(dy, d)
        wg, wu = _pair(w_gate, w_up)
        wd = _strided_rows(w_down, w_down.shape[1])
        dev, lib = x2.device, L.lib()
        a = _ffn_args(x2, wg, wu, wd, ctx.act)
        a.saved = L.ptr(saved)
        a.dy, a.lddy = dy2.data_ptr(), _ld(dy2)
        dx = torch.empty(x2.shape, dtype=x.dtype, device=dev) if need[0] else None
        dwg = dwu = None
        if need[1] or need[2]:   # one product over both
            dwg, dwu = (torch.empty(wg.shape, dtype=x.dtype, device=dev) for _ in range(2))
        dwd = torch.empty(wd.shape, dtype=x.dtype, device=dev) if need[3] else None
        a.dx, a.lddx = L.ptr(dx), d
        a.dw_gate, a.dw_up, a.lddw_in = L.ptr(dwg), L.ptr(dwu), d
        a.dw_down, a.lddw_down = L.ptr(dwd), a.f
        size = lib.otf_gated_ffn_backward_workspace_size(ctypes.byref(a))
        ws = _scratch(size, dev)
        with _on(dev):
            L.check(lib.otf_gated_ffn_backward(ctypes.byref(a), L.ptr(ws), size, L.stream_handle(dev)),
                    "otf_gated_ffn_backward")
        return dx.view(x.shape) if need[0] else None, dwg if need[1] else None, dwu if need[2] else None, dwd, None


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       activation: str = "silu") -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``: the gated form of the fusion block's
    feed-forward part (MRI_PET_OT_nojax.py:523-549).

    x: (..., d); w_gate, w_up: (f, d); w_down: (d, f), as ``torch.nn.Linear`` keeps them, all of
    x's type.  ``activation``: "silu" or "gelu" (the exact form).  Sums are float32; the hidden
    activations are rounded to x's type, the two products that backward needs are kept in float32."""
    _input(x, "x")
    for name, t in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        _input(t, name)
        _same_device(x, **{name: t})
        if t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, x is {x.dtype}")
    if activation not in L.ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: one of {sorted(L.ACTIVATIONS)}")
    d = x.shape[-1] if x.dim() else 0
    if w_gate.dim() != 2 or w_gate.shape[1] != d or w_up.shape != w_gate.shape or w_down.shape != (d, w_gate.shape[0]):
        raise ValueError(f"x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and w_down "
                         f"{tuple(w_down.shape)} must be (..., d), (f, d), (f, d) and (d, f)")
    if d == 0 or w_gate.shape[0] == 0 or max(d, w_gate.shape[0]) > _MAX_WIDTH:
        raise ValueError(f"widths d = {d} and f = {w_gate.shape[0]} must be between 1 and {_MAX_WIDTH}")
    act = L.ACTIVATIONS[activation]
    if _wants_grad(x, w_gate, w_up, w_down):
        return _GatedFeedForward.apply(x, w_gate, w_up, w_down, act)
    return _ffn_call(_strided_rows(x, d), w_gate, w_up, w_down, act, False)[0].view(x.shape)
