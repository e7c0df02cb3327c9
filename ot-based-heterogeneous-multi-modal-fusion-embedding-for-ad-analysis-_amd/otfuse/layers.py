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

import importlib.machinery
import importlib.util
import os

import torch

from . import _lib as L
from .ops import _EMB_DT

NODES_PATH = os.path.join(os.path.dirname(L.LIB_PATH), "_otf_layers.so")
_nodes = None


def _native():
    """The autograd nodes over libotfuse.so (csrc/otf_torch.cpp); raises if they have not been built."""
    global _nodes
    if _nodes is None:
        L.lib()
        if not os.path.exists(NODES_PATH):
            raise L.OtfError(f"otfuse layers not found at {NODES_PATH}; build them with "
                             "`python -c 'import __graft_entry__ as g; g.build()'`")
        loader = importlib.machinery.ExtensionFileLoader("_otf_layers", NODES_PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("_otf_layers", NODES_PATH, loader=loader))
        loader.exec_module(module)
        _nodes = module
    return _nodes


def _input(t, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a ROCm device tensor")
    if t.dtype not in _EMB_DT:
        raise TypeError(f"{name}: float32, bfloat16 or float16, not {t.dtype}")
    return t


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


# ----------------------------------------------------------------------------- dropout
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
    return _native().dropout(x, residual, _probability(p), _rng(rng, x))


# -------------------------------------------------------------------------- layer norm
def _norm_params(x, weight, bias):
    cols = x.shape[-1] if x.dim() else 0
    if cols == 0:
        raise ValueError(f"x {tuple(x.shape)}: layer norm needs a last dimension of at least 1")
    kind = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _input(t, name)
        _same_device(x, **{name: t})
        if t.shape != (cols,):
            raise ValueError(f"{name} {tuple(t.shape)} must be ({cols},)")
        if t.dtype not in (x.dtype, torch.float32) or kind not in (None, t.dtype):
            raise TypeError(f"weight and bias must share one type, x's ({x.dtype}) or float32")
        kind = t.dtype


def _eps(eps) -> float:
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps {eps} must be finite and not negative")
    return eps


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    (SelfAttentionBlock's norms, MRI_PET_OT_nojax.py:523-549).

    x: (..., cols); weight, bias: (cols,), of one type, x's or float32.  The gradients of
    weight and bias are sums in a fixed order: the same bits every call."""
    _input(x, "x")
    _norm_params(x, weight, bias)
    return _native().layer_norm(x, weight, bias, _eps(eps))


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
    _norm_params(x, weight, bias)
    p, eps = _probability(p), _eps(eps)
    if rng is None and p:
        raise ValueError("p > 0 needs rng (rng_state)")
    rng = None if rng is None else _rng(rng, x)
    return _native().dropout_add_layer_norm(x, residual, weight, bias, p, rng, eps)


# ------------------------------------------------------------------ gated feed-forward
_MAX_WIDTH = 1 << 20   # the kernels' row strides: 256 rows within a 31-bit byte offset


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
    return _native().gated_feed_forward(x, w_gate, w_up, w_down, L.ACTIVATIONS[activation])
