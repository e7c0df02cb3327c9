"""Calls of the fusion block's layers (otfuse.layers) at the edges of what they take."""
import pytest
import torch

import layers_plain as plain
from test_gpu_layers import T, U, _randn, _within, half

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ one row, wherever it lies
def _far_row(t):
    """t's one row at the end of a sequence of 2^21 elements: torch counts any stride of a single row as
    contiguous, so nothing makes it dense"""
    cols = t.shape[1]
    seq = torch.zeros(1, (1 << 21) // cols + 2, cols, dtype=t.dtype, device=t.device)
    row = seq[:, -1].copy_(t)
    assert row.stride(0) > 1 << 20 and row.is_contiguous()
    return row


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d,f", [(96, 120), (200, 1), (1, 77)])
def test_gated_feed_forward_of_one_far_row(dev, dt, d, f):
    """The last token of a long sequence, its gradient, and weights of one row."""
    from otfuse import layers
    t = T[dt]
    x, dy = (_randn(dev, i, 1, d, dtype=t) for i in (1, 5))
    w = [_randn(dev, i, *s, dtype=t, scale=s[1] ** -0.5) for i, s in ((2, (f, d)), (3, (f, d)), (4, (d, f)))]
    dense = [v.clone().requires_grad_(True) for v in (x, *w)]
    want = layers.gated_feed_forward(*dense)
    want_grads = torch.autograd.grad(want, dense, dy)
    far = [_far_row(v).requires_grad_(True) if v.shape[0] == 1 else v.clone().requires_grad_(True) for v in (x, *w)]
    got = layers.gated_feed_forward(*far)
    assert torch.equal(got, want)
    for g, h in zip(torch.autograd.grad(got, far, _far_row(dy)), want_grads):
        assert torch.equal(g, h)
    with torch.no_grad():
        assert torch.equal(layers.gated_feed_forward(*far), want)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_row_layers_of_one_far_row(dev, dt):
    from otfuse import layers
    x, dy = (_randn(dev, i, 1, 300, dtype=T[dt]) for i in (1, 2))
    rng = layers.rng_state(3, 4, dev)
    for call in (lambda v: layers.dropout(v, 0.3, rng, residual=v), layers.layer_norm,
                 lambda v: layers.dropout_add_layer_norm(v, v, p=0.3, rng=rng)[0]):
        near, far = x.clone().requires_grad_(True), _far_row(x).requires_grad_(True)
        y, z = call(near), call(far)
        assert torch.equal(y, z)
        assert torch.equal(torch.autograd.grad(y, near, dy)[0], torch.autograd.grad(z, far, _far_row(dy))[0])


# ------------------------------------------------------------------ lazily negated views
def test_imaginary_parts_of_conjugates(dev):
    """torch keeps them as a view with a sign to be applied: of one element, or made so by hand, it is
    contiguous and its memory holds the other sign."""
    from otfuse import layers
    rng = layers.rng_state(3, 4, dev)
    one = torch.complex(*(torch.randn(1, 1, device=dev) for _ in range(2))).conj().imag
    many = torch._neg_view(torch.randn(20, 72, device=dev))
    assert one.is_neg() and many.is_neg()
    for v in (one, many):
        plain_v, cols = v.resolve_neg().clone(), v.shape[1]
        w = torch.randn(24, cols, device=dev)
        for call in (lambda t, s: layers.dropout(t, 0.0, rng, residual=s), lambda t, s: layers.layer_norm(t, t[0], s[0]),
                     lambda t, s: layers.dropout_add_layer_norm(t, s)[0], lambda t, s: layers.gated_feed_forward(t, w, w, w.t()),
                     lambda t, s: layers.gated_feed_forward(s, t[:1], s[:1], t[:1].t())):
            a, b = v.detach().requires_grad_(True), plain_v.clone().requires_grad_(True)
            assert a.is_neg()
            y, z = call(a, plain_v), call(b, plain_v)
            assert torch.equal(y, z)
            assert torch.equal(*(torch.autograd.grad(o, leaf, torch.ones_like(z))[0] for o, leaf in ((y, a), (z, b))))
            with torch.no_grad():
                assert torch.equal(call(v, plain_v), z)


# ------------------------------------------------------------------ infinities
def _same_kind(got, want, name):
    """NaN where the 64-bit form has NaN, the same infinity where it has one, else finite"""
    got, want = got.detach().double().cpu(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), name


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,d,f", [(1, 72, 104), (4, 72, 104), (5, 72, 104), (8, 72, 104), (9, 72, 104), (16, 72, 104), (40, 72, 104),
                                     (8, 2048, 4104), (5, 2050, 4100), (3, 2048, 5632)])
@pytest.mark.parametrize("where", ["w_down", "w_up", "dy"])
def test_gated_feed_forward_infinities_do_not_depend_on_the_row_count(dev, dt, rows, d, f, where):
    """An infinite weight or gradient gives what the formula gives of it: an infinity where one term is
    infinite, not the difference of two that a value's parts would make."""
    from otfuse import layers
    t = T[dt]
    x = _randn(dev, 1, rows, d, dtype=t)
    w = [_randn(dev, i, *s, dtype=t, scale=s[1] ** -0.5) for i, s in ((2, (f, d)), (3, (f, d)), (4, (d, f)))]
    dy = _randn(dev, 5, rows, d, dtype=t)
    if where == "w_down":
        w[2][3, 7], w[2][d - 1, f - 1] = float("inf"), float("-inf")
    elif where == "w_up":
        w[1][f - 1, 5] = float("inf")
    else:
        dy[rows - 1, 2] = float("-inf")
    args = [v.requires_grad_(True) for v in (x, *w)]
    y = layers.gated_feed_forward(*args)
    got = (y, *torch.autograd.grad(y, args, dy))
    ref = plain.gated_feed_forward(*(v.detach().double().cpu() for v in args), "silu", dy.double().cpu())
    for name, g, r in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), got, ref):
        _same_kind(g, r, name)


# ------------------------------------------------------------------ the activation's tail
@pytest.mark.parametrize("dt,low,scale", [("bf16", -12.0, 1.0), ("f16", -5.5, 1024.0)])
@pytest.mark.parametrize("rows", [4, 12, 40])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_activation_tail(dev, dt, low, scale, rows, act):
    """act(g) and act'(g) one by one: the gate's weights pick a column of x each, the up product is
    `scale`, the down product copies.  So y is act(g) scale and dx act'(g) scale of one rounding to
    the type, up to the float32 evaluation: an exponential of at most 104 powers of two whose argument is
    seven roundings off, 104 * 7 * 2^-24 * ln 2 = 3e-5 of the value, and a few more: 2^-14."""
    from otfuse import layers
    t, n = T[dt], 63
    g = torch.linspace(low, 6.0, rows * n, dtype=torch.float64).view(rows, n).to(t)
    x = torch.ones(rows, n + 1, dtype=t)
    x[:, :n] = g
    eye = torch.zeros(n, n + 1, dtype=t)
    eye[:, :n] = torch.eye(n, dtype=t)
    up = torch.zeros(n, n + 1, dtype=t)
    up[:, n] = scale
    args = [v.to(dev) for v in (x, eye, up, eye.t().contiguous())]
    leaf = args[0].requires_grad_(True)
    y = layers.gated_feed_forward(*args, activation=act)
    (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    gd = g.double()
    value, slope = plain.act(gd, act)
    _within(y[:, :n], value * scale, (half(t) + 2.0 ** -14) * value.abs() * scale)
    terms = slope.abs() + 2 * (gd * torch.exp(-gd * gd / 2) / 2.5).abs() if act == "gelu" else slope.abs() + (value * (1 - torch.sigmoid(gd))).abs() * 2
    _within(dx[:, :n], slope * scale, scale * (half(t) * slope.abs() + 2.0 ** -14 * terms))


# ------------------------------------------------------------------ what is refused
def _calls(dev):
    from otfuse import layers
    rng = layers.rng_state(1, 2, dev)
    w, b = torch.ones(16, device=dev), torch.zeros(16, device=dev)
    wi, wo = torch.ones(24, 16, device=dev), torch.ones(16, 24, device=dev)
    return {"dropout": lambda x: layers.dropout(x, 0.1, rng), "dropout residual": lambda x: layers.dropout(torch.ones_like(w).expand(4, 16), 0.1, rng, residual=x),
            "layer_norm": lambda x: layers.layer_norm(x, w, b), "add_norm": lambda x: layers.dropout_add_layer_norm(x, torch.ones(4, 16, device=dev), w, b)[0],
            "add_norm residual": lambda x: layers.dropout_add_layer_norm(torch.ones(4, 16, device=dev), x, w, b)[0],
            "ffn": lambda x: layers.gated_feed_forward(x, wi, wi, wo)}


@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_is_refused(dev, leaf):
    """A tangent that the kernels do not carry on is an error, not a constant."""
    import torch.autograd.forward_ad as fwad
    from otfuse import layers
    x = torch.randn(4, 16, device=dev).requires_grad_(leaf)
    for name, call in _calls(dev).items():
        with fwad.dual_level():
            with pytest.raises(RuntimeError, match="forward"):
                call(fwad.make_dual(x, torch.ones(4, 16, device=dev)))
        call(x)
    v, m = torch.ones(16, device=dev), torch.ones(24, 16, device=dev)
    with fwad.dual_level():
        for call in (lambda: layers.layer_norm(x, fwad.make_dual(v, v)), lambda: layers.layer_norm(x, None, fwad.make_dual(v, v)),
                     lambda: layers.dropout_add_layer_norm(x, x, fwad.make_dual(v, v)),
                     lambda: layers.gated_feed_forward(x, fwad.make_dual(m, m), m, m.t()),
                     lambda: layers.gated_feed_forward(x, m, fwad.make_dual(m, m), m.t()),
                     lambda: layers.gated_feed_forward(x, m, m, fwad.make_dual(m, m).t())):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        if leaf:   # a tangent that reaches backward alone
            for call in _calls(dev).values():
                for y in call(x), *layers.dropout_add_layer_norm(x, x):
                    with pytest.raises(RuntimeError, match="forward"):
                        torch.autograd.grad((y * fwad.make_dual(torch.ones_like(y), torch.ones_like(y))).sum(), x)


def test_tracing_and_transforms_are_refused(dev):
    """A trace would hold the results' allocation without the kernels that fill them; a transform's
    wrapped tensors have no memory to read."""
    x = torch.randn(4, 16, device=dev)
    for name, call in _calls(dev).items():
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, (x,), check_trace=False)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x.expand(3, 4, 16))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(t).sum())(x)
        call(x)


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


def test_layer_norm_parameter_gradients_past_32_bit_thread_counts(dev):
    """Rows of more than 2^28 columns: none of them, and 65, whose sums two workgroups a column block
    share.  x is 1 in the first half of a row and -1 in the second, so mean 0, variance 1, and with
    dy = 1 a weight's gradient is 65 x / sqrt(1 + eps), 65 or -65 in bfloat16, a bias's 65."""
    from otfuse import layers
    rows, cols, t = 65, (1 << 28) + 64, torch.bfloat16
    w = torch.ones(cols, dtype=t, device=dev, requires_grad=True)
    none = torch.zeros(0, cols, dtype=t, device=dev)
    (dw,) = torch.autograd.grad(layers.layer_norm(none, w), w, none)
    assert torch.count_nonzero(dw) == 0
    b = torch.zeros(cols, dtype=t, device=dev, requires_grad=True)
    x = torch.ones(rows, cols, dtype=t, device=dev)
    x[:, cols // 2:] = -1
    y = layers.layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), torch.ones((), dtype=t, device=dev).expand(rows, cols))
    assert torch.equal(dw, x[0] * 65) and bool((db == 65).all())
    del none, x, y, dw, db, w, b
    torch.cuda.empty_cache()
