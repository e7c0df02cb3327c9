"""Layers of the fusion block around the OT features, forward and backward, as HIP kernels.

The reference's model applies dropout, layer norm and a feed-forward block to the same fused
embeddings whose OT alignment ``fusion.ot_alignment_loss`` computes
(MRI_PET_OT_nojax.py:523-549,658-669; ``--projection-dropout``,
MRI_PET_OT_OT_per_epoch_attn.py:963-1065).  Here:

    dropout                  y = [residual +] keep * x / (1 - p), the mask never stored
    layer_norm               with the parameter gradients' reduction
    dropout_add_layer_norm   z = residual + dropout(x), y = LN(z), one pass over the rows
    gated_feed_forward       (act(x Wg^T) * (x Wu^T)) Wd^T on the matrix cores, in the place of the
                             block's feed-forward part (parity with it unpinned)

Tensors live on a ROCm device; kernels run on the current stream of the tensors' device and
nothing synchronises, so every call can be captured into a graph: forward and backward together,
and with no eager graph of the same leaves alive (autograd runs a node on the stream that its
forward, or a leaf's first use in a graph that lives, ran on).  Inputs are float32, bfloat16 or
float16; statistics and sums are float32.  Each function takes part in autograd, in reverse
mode and once: second derivatives, forward-mode tangents, tracing and function transforms are refused.
Without a gradient to compute, nothing is kept for backward.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

import torch

from . import _lib as L

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


def rng_state(seed: int, offset: int = 0, device="cuda") -> torch.Tensor:
    """The generator's state as the layers take it: a device int64 tensor ``[seed, offset]``.

    A mask is a function of (seed, offset, row, column, columns) alone.  Layers of one step that
    must not share a mask take different offsets (or seeds); between steps, advance the offset
    (``rng[1] += number_of_layers``) after backward: backward makes the mask again from the same
    tensor, and raises if it was changed in between.  Being read on the device, the state can
    advance between replays of a captured graph."""
    return torch.tensor([seed, offset], dtype=torch.int64, device=device)


# ----------------------------------------------------------------------------- dropout
def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``[residual +] dropout(x)`` (``--projection-dropout``).

    Each element is kept with probability ``1 - p`` (``p`` rounded to a multiple of 2^-16) and
    scaled by its inverse; a dropped one is exactly 0, whatever it held.  The mask comes from
    ``rng`` (see ``rng_state``) and the element's row and column and is made again in backward
    instead of being stored.  x: (..., cols); residual: the same shape and type."""
    return _native().dropout(x, p, rng, residual)


# -------------------------------------------------------------------------- layer norm
def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    (SelfAttentionBlock's norms, MRI_PET_OT_nojax.py:523-549).

    x: (..., cols); weight, bias: (cols,), of one type, x's or float32.  The gradients of
    weight and bias are sums in a fixed order: the same bits every call."""
    return _native().layer_norm(x, weight, bias, eps)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, p: float = 0.0, rng: torch.Tensor | None = None,
                           eps: float = 1e-5):
    """``z = residual + dropout(x)``, ``y = layer_norm(z)``; returns ``(y, z)``.

    residual and z: x's type or float32 (a 32-bit residual stream under 16-bit layers); y: x's
    type, of the float32 sum.  ``rng`` may be None where ``p`` is 0.  Backward keeps a float32 z,
    else x and residual."""
    return _native().dropout_add_layer_norm(x, residual, weight, bias, p, rng, eps)


# ------------------------------------------------------------------ gated feed-forward
def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       activation: str = "silu") -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``: the gated form of the fusion block's
    feed-forward part (MRI_PET_OT_nojax.py:523-549).

    x: (..., d); w_gate, w_up: (f, d); w_down: (d, f), as ``torch.nn.Linear`` keeps them, all of
    x's type.  ``activation``: "silu" or "gelu" (the exact form).  Sums are float32.  The hidden
    activations and their gradients are rounded to x's type; up to 8 rows of 16-bit types they keep what
    that leaves out.  For backward the gate and up products are kept in float32 beside the hidden
    activations: 10 bytes a hidden value of 16-bit types, 12 of float32."""
    return _native().gated_feed_forward(x, w_gate, w_up, w_down, activation)
