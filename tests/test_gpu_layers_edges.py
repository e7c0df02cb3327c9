"""Calls of the fusion block's layers (otfuse.layers) at the edges of what they take."""
import pytest
import torch

import layers_plain as plain
from test_gpu_layers import T, U, _randn, _within, half

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ launches past 2^32 threads
def test_gated_feed_forward_copies_past_32_bit_thread_counts(dev):
    """Three unaligned weights of 1.3e10 elements: their copies are 4.9e9 groups of eight, one launch.
    All weights are 2^-17 (one buffer), so g = u = 131071 * 2^-17 exactly, h is act(g) u and y the sum of
    f equal terms: within f u of it and a rounding to the type."""
    from otfuse import layers
    d, f, t = 131071, 100000, torch.bfloat16
    flat = torch.full((d * f,), 2.0 ** -17, dtype=t, device=dev)
    with torch.no_grad():
        y = layers.gated_feed_forward(torch.ones(1, d, dtype=t, device=dev), flat.view(f, d), flat.view(f, d), flat.view(d, f))
    g = torch.tensor(d * 2.0 ** -17, dtype=torch.float64)
    want = (plain.act(g, "silu")[0] * g * f * 2.0 ** -17).expand(1, d)
    _within(y, want, (half(t) + f * U) * want)
    del flat, y
    torch.cuda.empty_cache()
