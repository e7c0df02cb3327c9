"""The fusion block's layers (otfuse.layers) against plain forms in 64 bits.

u = 2^-24 is float32's half step, h(t) = finfo(t).eps / 2 the half step of a result's type.

Rows are summed over at most 64 sequential and tree steps (32 elements of a thread, six lane
steps, sixteen waves; beyond 32768 columns one more element a step), so a row sum is within
64 u of the sum of magnitudes and everything formed from two of them within 128 u of the same
expression over magnitudes; a rounding to the result's type adds h(t) of the value.

The matrix products are compared in norm: a float32 sum over K terms is within K u of the sum of
magnitudes, hidden values rounded to 16 bits err by h(t) each with random sign, so a result's
relative 2-norm error is at most h(t) times the roundings on its path: y and dw_down 2 (h, own);
dx, dw_gate, dw_up 6 (g, whose derivative factor at most doubles it, u, dg or du, dh's other factor,
own).  Element by element: eight times that of the result's root mean square, plus as much of
the value (a sum of many independent roundings is within eight deviations)."""
import pytest
import torch

import layers_plain as plain

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def _randn(dev, seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(dev)


def _strided(t, pad, skip=0):
    """t's values in rows `pad` columns further apart, starting `skip` elements in"""
    buf = torch.zeros(t.shape[0] * (t.shape[1] + pad) + skip, dtype=t.dtype, device=t.device)
    v = buf[skip:].view(t.shape[0], -1)[:, :t.shape[1]]
    return v.copy_(t)


def _within(got, want, tol):
    """`tol` counts h(t) |value| for the rounding to got's type; below the smallest normal number the
    half step no longer shrinks with the value but stays at smallest_normal * h(t) (float16: 2^-25)."""
    tiny = torch.finfo(got.dtype).smallest_normal * half(got.dtype)
    got = got.detach().double().cpu()
    want, tol = want.cpu(), (tol.cpu() if isinstance(tol, torch.Tensor) else tol) + tiny
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    excess = ((got - want).abs() - tol).max().item() if got.numel() else 0.0
    assert excess <= 0, f"{excess:.3e} beyond the tolerance"


# ----------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,p,pad", [(1, 1, 0.5, 0), (8, 512, 0.1, 0), (37, 1237, 0.3, 0), (5, 16, 0.9, 3),
                                            (300, 72, 0.0, 8), (3, 9, 1.0, 1), (1000, 7, 0.99999, 0)])
def test_dropout(dev, dt, rows, cols, p, pad):
    from otfuse import layers
    seed, offset = (1 << 62) + rows, (3 << 33) + cols
    rng = layers.rng_state(seed, offset, dev)
    x = _strided(_randn(dev, 1, rows, cols, dtype=T[dt]), pad, pad % 3).requires_grad_(True)
    res = _randn(dev, 2, rows, cols, dtype=T[dt]).requires_grad_(True)
    dy = _randn(dev, 3, rows, cols, dtype=T[dt])
    f = plain.factor(rows, cols, p, seed, offset)
    xs = x.detach().double().cpu() * f
    h = half(T[dt])
    y = layers.dropout(x, p, rng)
    _within(y, xs, (h + 3 * U) * xs.abs())
    assert torch.count_nonzero(y.detach().cpu()[f == 0]) == 0
    z = layers.dropout(x, p, rng, residual=res)
    r = res.detach().double().cpu()
    _within(z, xs + r, h * (xs + r).abs() + 4 * U * (xs.abs() + r.abs()))
    dx, dr = torch.autograd.grad(z, (x, res), dy)
    ds = dy.double().cpu() * f
    _within(dx, ds, (h + 3 * U) * ds.abs())
    assert torch.equal(dr, dy)


def test_dropout_known_answer(dev):
    """Element (0, j) of seed 0, offset 0 is field j of the published vector for a zero counter."""
    from otfuse import layers
    words = (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    fields = [f for w in words for f in (w & 0xFFFF, w >> 16)]
    x = torch.ones(1, 8, device=dev)
    for f in fields:
        for t in (f, f + 1):
            keep = layers.dropout(x, t / 65536, layers.rng_state(0, 0, dev))[0] != 0
            assert keep.tolist() == [g >= t for g in fields]


def test_dropout_select_not_product(dev):
    from otfuse import layers
    x = torch.ones(64, 40, device=dev)
    rng = layers.rng_state(5, 6, dev)
    drop = layers.dropout(x, 0.5, rng) == 0
    for bad in (float("nan"), float("inf"), float("-inf")):
        v = torch.where(drop, torch.full_like(x, bad), x)
        y = layers.dropout(v, 0.5, rng)
        assert torch.equal(y, torch.where(drop, torch.zeros_like(x), x * 2))
        z, _ = layers.dropout_add_layer_norm(v, x, p=0.5, rng=rng)
        assert torch.isfinite(z).all()


def test_dropout_shapes_and_rate(dev):
    from otfuse import layers
    rng = layers.rng_state(11, 0, dev)
    x = torch.ones(4, 50, 1000, device=dev)
    y = layers.dropout(x, 0.1, rng)
    kept = float((y != 0).double().mean())
    assert abs(kept - (1 - 6554 / 65536)) < 6 * (0.09 / x.numel()) ** 0.5   # six deviations
    assert torch.equal(y.view(200, 1000), layers.dropout(x.view(200, 1000), 0.1, rng))
    assert layers.dropout(torch.ones((), device=dev), 0.0, rng).shape == ()
    assert layers.dropout(torch.ones(0, 8, device=dev), 0.5, rng).shape == (0, 8)
    assert layers.dropout(torch.ones(3, 0, device=dev), 0.5, rng).shape == (3, 0)
    # columns apart from rows: a transposed view is its values
    t = x[0].t()
    assert torch.equal(layers.dropout(t, 0.1, rng), layers.dropout(t.contiguous(), 0.1, rng))
    other = layers.dropout(x, 0.1, layers.rng_state(11, 1, dev))
    assert not torch.equal(other, y)


def test_dropout_backward_notices_a_changed_state(dev):
    from otfuse import layers
    rng = layers.rng_state(1, 1, dev)
    x = torch.ones(4, 8, device=dev, requires_grad=True)
    y = layers.dropout(x, 0.5, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# -------------------------------------------------------------------------- layer norm
NORMS = [(5, 5), (1000, 100), (257, 128), (2000, 65), (901, 200), (333, 256), (10, 16384), (6, 16400), (1, 1), (3, 8), (70, 33), (129, 512), (9, 1000), (40, 1531), (17, 2048), (6, 4096), (33, 4100), (5, 8192),
         (3, 12345), (2, 32768), (2, 40001), (700, 64), (3000, 24)]


def _norm_tolerance(x, w, dy, h_y, h_x, h_w, y, xhat, rstd, dx, dw, db):
    """the bounds of the module's docstring for y, dx, dw, db"""
    k = 128 * U
    e = xhat.abs() + rstd * x.abs().mean(1, keepdim=True)   # k e: error of xhat
    c = (dy * w).abs()
    m1, m2 = c.mean(1, keepdim=True), (c * xhat.abs()).mean(1, keepdim=True)
    ty = h_y * y.abs() + k * (e * w.abs() + (y - xhat * w).abs())
    tx = h_x * dx.abs() + k * rstd * (c + m1 + xhat.abs() * m2 + e * m2 + xhat.abs() * (c * e).mean(1, keepdim=True))
    tx = tx + k * dx.abs()
    tw = h_w * dw.abs() + k * (dy.abs() * (xhat.abs() + e)).sum(0)
    tb = h_w * db.abs() + k * dy.abs().sum(0)
    return ty, tx, tw, tb


@pytest.mark.parametrize("dt,wt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,cols", NORMS)
def test_layer_norm(dev, dt, wt, rows, cols):
    from otfuse import layers
    x = _randn(dev, 1, rows, cols, dtype=T[dt], scale=2.0, shift=0.5)
    if cols % 2:
        x = _strided(x, 5, 1)
    x.requires_grad_(True)
    w = _randn(dev, 2, cols, dtype=T[wt], scale=0.3, shift=1.0).requires_grad_(True)
    b = _randn(dev, 3, cols, dtype=T[wt]).requires_grad_(True)
    dy = _randn(dev, 4, rows, cols, dtype=T[dt])
    y = layers.layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    xd, wd, bd, dyd = (t.detach().double().cpu() for t in (x, w, b, dy))
    yr, xhat, rstd = plain.layer_norm(xd, wd, bd, 1e-5)
    ref = plain.layer_norm_backward(dyd, xhat, rstd, wd)
    tol = _norm_tolerance(xd, wd, dyd, half(T[dt]), half(T[dt]), half(T[wt]), yr, xhat, rstd, *ref)
    _within(y, yr, tol[0])
    for got, want, t in zip(grads, ref, tol[1:]):
        _within(got, want, t)
    with torch.no_grad():
        assert torch.equal(layers.layer_norm(x, w, b), y)   # nothing kept: the same result
    again = torch.autograd.grad(layers.layer_norm(x, w, b), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))   # fixed order: the same bits


def test_layer_norm_without_parameters_and_of_large_mean(dev):
    from otfuse import layers
    x = _randn(dev, 1, 50, 777, shift=1000.0).requires_grad_(True)
    dy = _randn(dev, 2, 50, 777)
    y = layers.layer_norm(x, eps=0.0)
    (dx,) = torch.autograd.grad(y, x, dy)
    one, zero = torch.ones(777, dtype=torch.float64), torch.zeros(777, dtype=torch.float64)
    xd, dyd = x.detach().double().cpu(), dy.double().cpu()
    yr, xhat, rstd = plain.layer_norm(xd, one, zero, 0.0)
    ref = plain.layer_norm_backward(dyd, xhat, rstd, one)
    tol = _norm_tolerance(xd, one, dyd, 0, 0, 0, yr, xhat, rstd, *ref)
    _within(y, yr, tol[0])
    _within(dx, ref[0], tol[1])
    b = torch.randn(777, device=dev, requires_grad=True)   # a bias alone
    yb = layers.layer_norm(x, None, b)
    (db,) = torch.autograd.grad(yb, b, dy)
    _within(db, dyd.sum(0), 128 * U * dyd.abs().sum(0))


def test_layer_norm_bad_rows_stay_alone(dev):
    from otfuse import layers
    x = _randn(dev, 1, 6, 100)
    clean = layers.layer_norm(x)
    x[2, 5] = float("nan")
    x[4, 99] = float("inf")
    y = layers.layer_norm(x)
    good = [0, 1, 3, 5]
    assert torch.equal(y[good], clean[good]) and torch.isnan(y[2]).all() and torch.isnan(y[4]).any()


def test_layer_norm_empty_and_refusals(dev):
    from otfuse import layers
    w = torch.ones(8, device=dev, requires_grad=True)
    x = torch.ones(0, 8, device=dev, requires_grad=True)
    y = layers.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert dx.shape == (0, 8) and torch.count_nonzero(dw) == 0
    x = torch.ones(2, 8, device=dev)
    for bad in (lambda: layers.layer_norm(torch.ones(2, 0, device=dev)), lambda: layers.layer_norm(x, w[:7]),
                lambda: layers.layer_norm(x, eps=-1.0), lambda: layers.layer_norm(x, eps=float("nan")),
                lambda: layers.dropout(x, 1.5, layers.rng_state(0, 0, dev)),
                lambda: layers.dropout(x, 0.5, layers.rng_state(0, 0, dev), residual=x[:1]),
                lambda: layers.dropout_add_layer_norm(x, x[:1], p=0.0), lambda: layers.dropout_add_layer_norm(x, x, p=0.5),
                lambda: layers.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64)),
                lambda: layers.gated_feed_forward(x, torch.ones(4, 8, device=dev), torch.ones(5, 8, device=dev),
                                                  torch.ones(8, 4, device=dev)),
                lambda: layers.gated_feed_forward(x, *[torch.ones(4, 8, device=dev)] * 2, torch.ones(8, 4, device=dev),
                                                  activation="tanh")):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: layers.layer_norm(x.double()), lambda: layers.layer_norm(x, w.half()),
                lambda: layers.layer_norm(x.half(), w.detach(), w.detach().half()),
                lambda: layers.dropout(x, 0.5, torch.zeros(2, device=dev)),
                lambda: layers.dropout_add_layer_norm(x, x.half(), p=0.0),
                lambda: layers.gated_feed_forward(x, *[torch.ones(4, 8, device=dev).half()] * 2, torch.ones(8, 4, device=dev))):
        with pytest.raises(TypeError):
            bad()


@pytest.mark.parametrize("dt,rt", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("rows,cols,p", [(1, 1, 0.0), (8, 2048, 0.1), (70, 333, 0.3), (12, 4096, 0.5), (3, 9000, 0.1),
                                        (2, 20000, 0.1), (2, 33001, 0.2), (600, 48, 0.1), (100, 120, 0.2), (77, 250, 0.0), (30, 1500, 0.1)])
def test_dropout_add_layer_norm(dev, dt, rt, rows, cols, p):
    from otfuse import layers
    seed, offset = 77 + rows, 5
    rng = layers.rng_state(seed, offset, dev)
    x = _randn(dev, 1, rows, cols, dtype=T[dt])
    if cols % 3 == 0:
        x = _strided(x, 2, 1)
    x.requires_grad_(True)
    res = _randn(dev, 2, rows, cols, dtype=T[rt], scale=2.0).requires_grad_(True)
    w = _randn(dev, 3, cols, scale=0.3, shift=1.0).requires_grad_(True)
    b = _randn(dev, 4, cols).requires_grad_(True)
    dy, dz = _randn(dev, 5, rows, cols, dtype=T[dt]), _randn(dev, 6, rows, cols, dtype=T[rt])
    y, z = layers.dropout_add_layer_norm(x, res, w, b, p, rng)
    grads = torch.autograd.grad((y, z), (x, res, w, b), (dy, dz), retain_graph=True)
    f = plain.factor(rows, cols, p, seed, offset)
    xd, rd, wd, bd, dyd, dzd = (t.detach().double().cpu() for t in (x, res, w, b, dy, dz))
    s = xd * f + rd
    _within(z, s, half(T[rt]) * s.abs() + 4 * U * ((xd * f).abs() + rd.abs()))
    zd = s   # y is the norm of the float32 sum: within 2 u of s an element, which the row sums' bound holds
    yr, xhat, rstd = plain.layer_norm(zd, wd, bd, 1e-5)
    g, dw, db = plain.layer_norm_backward(dyd, xhat, rstd, wd)
    ty, tg, tw, tb = _norm_tolerance(zd, wd, dyd, half(T[dt]), 0, U, yr, xhat, rstd, g, dw, db)
    _within(y, yr, ty)
    g = g + dzd
    tg = tg + U * (g.abs() + dzd.abs())
    _within(grads[0], g * f, tg * f + (half(T[dt]) + 3 * U) * (g * f).abs())
    _within(grads[1], g, tg + half(T[rt]) * g.abs())
    _within(grads[2], dw, tw)
    _within(grads[3], db, tb)
    if p == 0:   # no state needed
        y0, z0 = layers.dropout_add_layer_norm(x, res, w, b)
        assert torch.equal(y0, y) and torch.equal(z0, z)
        assert all(torch.equal(g0, g1) for g0, g1 in zip(torch.autograd.grad((y0, z0), (x, res, w, b), (dy, dz)), grads))
    # either output alone
    only = torch.autograd.grad(z, (x, res), dz, retain_graph=True)
    _within(only[1], dzd, half(T[rt]) * dzd.abs())
    _within(only[0], dzd * f, (half(T[dt]) + 3 * U) * (dzd * f).abs())
    (gy,) = torch.autograd.grad(y, res, dy)
    _within(gy, g - dzd, tg + half(T[rt]) * (g - dzd).abs() + U * dzd.abs())


# ------------------------------------------------------------------ gated feed-forward
def _close(got, want, roundings, dtype, depth):
    got = got.detach().double()
    assert got.shape == want.shape and torch.isfinite(got).all()
    bound = roundings * half(dtype) + depth * U
    err, rms = got - want, want.square().mean().sqrt()
    rel = float(err.norm() / want.norm())
    assert rel <= bound, f"relative 2-norm {rel:.3e} > {bound:.3e}"
    excess = float((err.abs() - 8 * bound * rms - bound * want.abs()).max())
    assert excess <= 0, f"an element is {excess:.3e} beyond eight deviations"


FFNS = [(7, 2056, 4100), (14, 4104, 2050), (9, 640, 48), (16, 48, 2100), (12, 1100, 600), (1, 8, 16), (1, 1, 1), (1, 1000, 333), (3, 64, 96), (16, 130, 100), (16, 512, 1032), (17, 72, 136), (33, 250, 71),
        (64, 64, 64), (130, 512, 264), (200, 1000, 334), (257, 136, 1100), (5, 2048, 40), (700, 40, 2056), (513, 1024, 1408)]


@pytest.mark.parametrize("dt,act", [("bf16", "silu"), ("f16", "gelu"), ("f32", "silu")])
@pytest.mark.parametrize("rows,d,f", FFNS)
def test_gated_feed_forward(dev, dt, act, rows, d, f):
    from otfuse import layers
    t = T[dt]
    x = _randn(dev, 1, rows, d, dtype=t).requires_grad_(True)
    wg = _randn(dev, 2, f, d, dtype=t, scale=d ** -0.5).requires_grad_(True)
    wu = _randn(dev, 3, f, d, dtype=t, scale=d ** -0.5).requires_grad_(True)
    wd = _randn(dev, 4, d, f, dtype=t, scale=f ** -0.5).requires_grad_(True)
    dy = _randn(dev, 5, rows, d, dtype=t)
    y = layers.gated_feed_forward(x, wg, wu, wd, activation=act)
    grads = torch.autograd.grad(y, (x, wg, wu, wd), dy)
    ref = plain.gated_feed_forward(*(v.detach().double() for v in (x, wg, wu, wd)), act, dy.double())
    one = 0 if dt == "f32" else 1   # float32 hidden values are not rounded further: the sums' bound holds it
    depth = 2 * (d + f) + rows + 16
    _close(y, ref[0], 2 * one + 1, t, depth)
    for got, want, n in zip(grads, ref[1:], (6, 6, 6, 2)):
        _close(got, want, n * one + 1, t, depth)
    with torch.no_grad():
        assert torch.equal(layers.gated_feed_forward(x, wg, wu, wd, activation=act), y)
    again = torch.autograd.grad(layers.gated_feed_forward(x, wg, wu, wd, activation=act), (x, wg, wu, wd), dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


# two products a launch with tiles of each side, in slabs and without, tile counts off multiples of eight
@pytest.mark.parametrize("dt,act,rows,d,f", [("f16", "gelu", 777, 1000, 2730), ("bf16", "silu", 1024, 2048, 2816), ("bf16", "gelu", 3001, 520, 1400),
                                             ("bf16", "silu", 100, 512, 1408), ("f32", "gelu", 700, 1024, 2050), ("f32", "silu", 260, 500, 2044),
                                             ("bf16", "silu", 70, 2056, 5000), ("f16", "silu", 2304, 1032, 4104)])
def test_gated_feed_forward_shared_launches(dev, dt, act, rows, d, f):
    test_gated_feed_forward(dev, dt, act, rows, d, f)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rows,d,f", [(1, 256, 96), (2, 128, 302), (5, 72, 1100), (8, 1024, 2050), (8, 2048, 4104), (3, 4096, 5632)])
def test_gated_feed_forward_few_rows_round_once(dev, dt, rows, d, f):
    """Up to eight rows: what lies between x and a result is held in 32 bits, or in 16 with what they
    leave out, 2^-16 and better of a value.  So a result differs from the rounding of the 64-bit one
    only where that lies within the sums' error of a tie: 2^-16 of the sum's terms, against a step of
    2^-7 or 2^-10 of the value, 2^-5 of the results at most for values of the terms' size (a hidden
    value rounded to T, half a step off itself, would move about a third of them)."""
    from otfuse import layers
    t = T[dt]
    x = _randn(dev, 1, rows, d, dtype=t)
    w = [_randn(dev, i, *s, dtype=t, scale=s[1] ** -0.5) for i, s in ((2, (f, d)), (3, (f, d)), (4, (d, f)))]
    dy = _randn(dev, 5, rows, d, dtype=t)
    args = [v.requires_grad_(True) for v in (x, *w)]
    y = layers.gated_feed_forward(*args)
    got = (y, *torch.autograd.grad(y, args, dy))
    ref = plain.gated_feed_forward(*(v.detach().double() for v in args), "silu", dy.double())
    for g, r in zip(got, ref):
        assert (g.detach() != r.to(t)).double().mean() <= 2.0 ** -4


def test_gated_feed_forward_few_rows_overflow(dev):
    """A hidden value past float16 is an infinity, as one rounding makes it, not a NaN."""
    from otfuse import layers
    x = torch.full((2, 64), 64.0, dtype=torch.float16, device=dev)
    x[1] = 0.25
    w = torch.full((16, 64), 0.25, dtype=torch.float16, device=dev)
    down = torch.full((64, 16), 0.5, dtype=torch.float16, device=dev)
    y = layers.gated_feed_forward(x, w, w, down)   # gate and up 1024: 2^20 hidden
    assert torch.isinf(y[0]).all() and torch.isfinite(y[1]).all()


@pytest.mark.parametrize("dt,act,rows,d,f", [("bf16", "gelu", 4200, 4100, 4110), ("f16", "silu", 4097, 4104, 4352)])
def test_gated_feed_forward_large_tiles(dev, dt, act, rows, d, f):
    """Every product in whole and ragged tiles of the largest size, odd widths among them."""
    t = T[dt]
    from otfuse import layers
    g = torch.Generator(device=dev).manual_seed(1)
    r = lambda k, *s: (torch.randn(*s, device=dev, generator=g) * k).to(t).requires_grad_(True)
    args = [r(1.0, rows, d), r(d ** -0.5, f, d), r(d ** -0.5, f, d), r(f ** -0.5, d, f)]
    dy = r(1.0, rows, d).detach()
    y = layers.gated_feed_forward(*args, activation=act)
    grads = torch.autograd.grad(y, args, dy)
    ref = plain.gated_feed_forward(*(v.detach().double() for v in args), act, dy.double())
    depth = 2 * (d + f) + rows + 16
    _close(y, ref[0], 3, t, depth)
    for got, want, n in zip(grads, ref[1:], (7, 7, 7, 3)):
        _close(got, want, n, t, depth)
    again = torch.autograd.grad(layers.gated_feed_forward(*args, activation=act), args, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [4, 60])
def test_gated_feed_forward_views(dev, dt, rows):
    """Gate and up as halves of one weight, strided rows, unaligned starts, a 3-D input, and each
    gradient alone."""
    from otfuse import layers
    t, d, f = T[dt], 96, 120
    both = _randn(dev, 2, 2 * f, d, dtype=t, scale=d ** -0.5)
    wd = _randn(dev, 4, d, f, dtype=t, scale=f ** -0.5)
    x = _randn(dev, 1, rows, d, dtype=t)
    want = layers.gated_feed_forward(x, both[:f].clone(), both[f:].clone(), wd)
    views = [_strided(x, 8), _strided(x, 3, 1), x.t().contiguous().t(), x.view(2, rows // 2, d)]
    for v in views:
        got = layers.gated_feed_forward(v, both[:f], both[f:], wd)
        assert got.shape == v.shape and torch.equal(got.reshape(rows, d), want)
    got = layers.gated_feed_forward(x, _strided(both[:f], 8), both[f:], _strided(wd, 5, 1))
    assert torch.equal(got, want)
    dy = _randn(dev, 5, rows, d, dtype=t)
    args = [v.clone().requires_grad_(True) for v in (x, both[:f], both[f:], wd)]
    full = torch.autograd.grad(layers.gated_feed_forward(*args), args, dy)
    for i in range(4):
        some = [v.detach().requires_grad_(j == i) for j, v in enumerate(args)]
        (g,) = torch.autograd.grad(layers.gated_feed_forward(*some), [some[i]], _strided(dy, 7))
        assert torch.equal(g, full[i]), i
    # a leading dimension past what the kernels index is made dense
    wide = torch.zeros(rows, (1 << 20) + 8, dtype=t, device=dev)[:, :d].copy_(x)
    assert torch.equal(layers.gated_feed_forward(wide, both[:f], both[f:], wd), want)


def test_gated_feed_forward_no_rows(dev):
    from otfuse import layers
    args = [torch.ones(0, 8, device=dev), torch.ones(4, 8, device=dev), torch.ones(4, 8, device=dev), torch.ones(8, 4, device=dev)]
    args = [a.requires_grad_(True) for a in args]
    y = layers.gated_feed_forward(*args)
    grads = torch.autograd.grad(y, args, torch.ones_like(y))
    assert y.shape == (0, 8) and grads[0].shape == (0, 8)
    assert all(torch.count_nonzero(g) == 0 for g in grads[1:])


@pytest.mark.parametrize("rows", [3, 40])
def test_gated_feed_forward_bad_rows_stay_alone(dev, rows):
    """A row of NaN or infinity reaches its own result only, and the padding of ragged tiles none."""
    from otfuse import layers
    d, f = 72, 104
    w = [_randn(dev, i, *s, dtype=torch.bfloat16, scale=0.1) for i, s in ((2, (f, d)), (3, (f, d)), (4, (d, f)))]
    x = _randn(dev, 1, rows, d, dtype=torch.bfloat16)
    clean = layers.gated_feed_forward(x, *w)
    x[1] = float("nan")
    x[rows - 1, 0] = float("inf")
    y = layers.gated_feed_forward(x, *w)
    keep = [r for r in range(rows) if r not in (1, rows - 1)]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[1]).all()


def test_gated_feed_forward_against_differences(dev):
    """The directional derivative along each gradient in float32.  Step 2^-7 of the leaf's norm:
    truncation ~ step^2 = 6e-5 of the value times an order-1 constant; the outputs' rounding errors
    (about 16 u each, random) sum to ~16 u |y| |dy| against a difference of step |grad| |leaf|
    ~ step |y| |dy| / 4: 16 * 6e-8 * 128 * 4 = 5e-4.  5e-3 holds both."""
    from otfuse import layers
    args = [_randn(dev, i, *s, scale=k) for i, (s, k) in enumerate((((40, 96), 1.0), ((160, 96), 0.1), ((160, 96), 0.1), ((96, 160), 0.08)))]
    dy = _randn(dev, 9, 40, 96)
    for act in ("silu", "gelu"):
        leaves = [a.clone().requires_grad_(True) for a in args]
        grads = torch.autograd.grad(layers.gated_feed_forward(*leaves, activation=act), leaves, dy)
        for i, g in enumerate(grads):
            step = 2.0 ** -7 * float(args[i].norm()) / float(g.norm())
            def loss(s):
                a = list(args)
                a[i] = args[i] + s * g
                return float((layers.gated_feed_forward(*a, activation=act).double() * dy.double()).sum())
            diff, want = (loss(step) - loss(-step)) / (2 * step), float(g.double().square().sum())
            scale = max(want, float(g.norm()) * float(dy.norm()) * float(layers.gated_feed_forward(*args, activation=act).norm()) / float(args[i].norm()))
            assert abs(diff - want) <= 5e-3 * scale, (act, i, diff, want)


def test_second_derivatives_are_refused(dev):
    from otfuse import layers
    x = torch.randn(4, 16, device=dev, requires_grad=True)
    w = torch.randn(24, 16, device=dev, requires_grad=True)
    rng = layers.rng_state(1, 2, dev)
    for y in (layers.dropout(x, 0.1, rng), layers.layer_norm(x), layers.dropout_add_layer_norm(x, x, p=0.1, rng=rng)[0],
              layers.gated_feed_forward(x, w, w, w.t())):
        (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            g.sum().backward()


# ------------------------------------------------------------------ past 2^31 elements
def test_rowwise_layers_past_32_bit_offsets(dev):
    """2.2e9 elements: the first and the last rows against the plain forms."""
    from otfuse import layers
    rows, cols, p, seed, offset = 270001, 8200, 0.25, 99, 3
    rng = layers.rng_state(seed, offset, dev)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev)
    block = _randn(dev, 1, 1009, cols, dtype=torch.bfloat16)
    for i in range(0, rows, 1009):
        x[i:i + 1009] = block[:min(1009, rows - i)]
    y, z = layers.dropout_add_layer_norm(x, x, p=p, rng=rng)
    d = layers.dropout(x, p, rng)
    n = layers.layer_norm(x)
    one, zero, h = torch.ones(cols, dtype=torch.float64), torch.zeros(cols, dtype=torch.float64), half(torch.bfloat16)
    for first in (0, rows - 5):
        f = plain.factor(5, cols, p, seed, offset, first)
        xs = x[first:first + 5].double().cpu()
        _within(d[first:first + 5], xs * f, (h + 3 * U) * (xs * f).abs())
        s = xs * f + xs
        _within(z[first:first + 5], s, h * s.abs() + 4 * U * 2 * xs.abs() * (1 + f))
        for got, v in ((y, s), (n, xs)):
            want, xhat, rstd = plain.layer_norm(v, one, zero, 1e-5)
            e = xhat.abs() + rstd * v.abs().mean(1, keepdim=True)
            _within(got[first:first + 5], want, h * want.abs() + 128 * U * e)
    del y, z, d
    leaf = x.requires_grad_(True)
    (dx,) = torch.autograd.grad(layers.layer_norm(leaf), leaf, n)
    for first in (0, rows - 5):
        v = x.detach()[first:first + 5].double().cpu()
        dy = n[first:first + 5].double().cpu()
        _, xhat, rstd = plain.layer_norm(v, one, zero, 1e-5)
        want, _, _ = plain.layer_norm_backward(dy, xhat, rstd, one)
        tol = _norm_tolerance(v, one, dy, 0, h, 0, xhat, xhat, rstd, want, zero, zero)[1]
        _within(dx[first:first + 5], want, tol)


def test_gated_feed_forward_past_32_bit_offsets(dev):
    """2.3e9 hidden values: y and dx of the last rows, which no other row reaches."""
    from otfuse import layers
    rows, d, f, t = 220001, 128, 10304, torch.bfloat16
    w = [_randn(dev, i, *s, dtype=t, scale=k) for i, s, k in ((2, (f, d), 0.09), (3, (f, d), 0.09), (4, (d, f), 0.01))]
    x = torch.zeros(rows, d, dtype=t, device=dev)
    x[-70:] = _randn(dev, 1, 70, d, dtype=t)
    dy = torch.zeros(rows, d, dtype=t, device=dev)
    dy[-70:] = _randn(dev, 5, 70, d, dtype=t)
    args = [v.requires_grad_(True) for v in (x, *w)]
    y = layers.gated_feed_forward(*args)
    grads = torch.autograd.grad(y, args, dy)
    ref = plain.gated_feed_forward(x.detach()[-70:].double(), *(v.detach().double() for v in w), "silu", dy[-70:].double())
    depth = 2 * (d + f) + 70 + 16
    _close(y[-70:], ref[0], 3, t, depth)
    _close(grads[0][-70:], ref[1], 7, t, depth)
    assert torch.count_nonzero(y[:-70]) == 0 and torch.count_nonzero(grads[0][:-70]) == 0
    for got, want, n in zip(grads[1:], ref[2:], (7, 7, 3)):   # only the last rows contribute
        _close(got, want, n, t, depth)


# ----------------------------------------------------------------- streams, graphs, the block
def _step(leaves, rng, dy):
    from otfuse import layers
    x, res, w, b, wg, wu, wd = leaves
    h, z = layers.dropout_add_layer_norm(x, res, w, b, 0.1, rng)
    y = layers.dropout(layers.gated_feed_forward(layers.layer_norm(h, w, b), wg, wu, wd), 0.2, rng, residual=z)
    return (y,) + torch.autograd.grad(y, leaves, dy)


def _leaves(dev, rows, d, f, dtype):
    s = [_randn(dev, 1, rows, d, dtype=dtype), _randn(dev, 2, rows, d, dtype=dtype), _randn(dev, 3, d, dtype=dtype),
         _randn(dev, 4, d, dtype=dtype), _randn(dev, 5, f, d, dtype=dtype, scale=d ** -0.5),
         _randn(dev, 6, f, d, dtype=dtype, scale=d ** -0.5), _randn(dev, 7, d, f, dtype=dtype, scale=f ** -0.5)]
    return [t.requires_grad_(True) for t in s]


@pytest.mark.parametrize("rows,d,f,dtype", [(8, 512, 1032, torch.float32), (300, 200, 330, torch.bfloat16)])
def test_captured_step_replays(dev, rows, d, f, dtype):
    """Forward and backward in one graph; the state advances between replays, eager work and
    synchronisations in between."""
    from otfuse import layers
    dy = _randn(dev, 8, rows, d, dtype=dtype)
    rng = layers.rng_state(9, 0, dev)
    leaves = _leaves(dev, rows, d, f, dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(leaves, rng, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(leaves, rng, dy)
    eager = [t.detach().clone().requires_grad_(True) for t in leaves]
    for i in range(4):
        rng.copy_(layers.rng_state(9, 100 + i, dev))
        with torch.no_grad():
            leaves[0].add_(0.125)
            eager[0].add_(0.125)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(eager, rng.clone(), dy)
        for got, ref in zip(out, want):
            assert torch.equal(got, ref), i


def test_two_streams_at_once(dev):
    """Calls of the same sizes on two streams: no workspace is shared."""
    from otfuse import layers
    sets = [(_leaves(dev, 200, 264, 520, torch.bfloat16), layers.rng_state(s, 0, dev)) for s in (1, 2)]
    with torch.no_grad():
        sets[1][0][0].mul_(-1.5)
    dy = _randn(dev, 8, 200, 264, dtype=torch.bfloat16)
    want = [_step(l, r, dy) for l, r in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        got.append([])
        for s, (l, r) in zip(streams, sets):
            with torch.cuda.stream(s):
                got[-1].append(_step(l, r, dy))
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_feed_forward_block_with_alignment_loss(dev):
    """The block, its classifier features and the OT alignment loss of one training step, against the
    same step with the block in 64 bits (the plan given)."""
    from otfuse import layers
    from otfuse.fusion import FeedForwardBlock, cosine_loss, ot_alignment_loss
    B, d, f, p = 8, 512, 1024, 0.1
    torch.manual_seed(0)
    block = FeedForwardBlock(d, f, p, device=dev)
    attended, fused = (_randn(dev, s, B, d) for s in (1, 2))
    pet = _randn(dev, 3, B, d).requires_grad_(True)
    plan = torch.rand(d, d, device=dev)
    plan = plan / plan.sum(1, keepdim=True)
    rng = layers.rng_state(3, 40, dev)
    leaves = [attended.requires_grad_(True), fused.requires_grad_(True)] + list(block.parameters())
    out = block(attended, fused, rng)
    loss, _, _ = ot_alignment_loss(out, pet, plan)
    total = loss + out.square().mean()
    grads = torch.autograd.grad(total, leaves + [pet])

    dbl = [t.detach().double().requires_grad_(True) for t in leaves + [pet]]
    a, r, w1, b1, w2, b2, wg, wu, wd, pt = dbl
    names = [n for n, _ in block.named_parameters()]
    assert names == ["norm1.weight", "norm1.bias", "norm2.weight", "norm2.bias", "gate.weight", "up.weight", "down.weight"]
    k1, k2 = (plain.factor(B, d, p, 3, o).to(dev) for o in (40, 41))
    h = plain.layer_norm(r + a * k1, w1, b1, 1e-5)[0]
    g = h @ wg.t()
    ffn = (g * torch.sigmoid(g) * (h @ wu.t())) @ wd.t()
    ref = plain.layer_norm(h + ffn * k2, w2, b2, 1e-5)[0]
    want = cosine_loss(ref, pt @ plan.double().t()) + ref.square().mean()
    wgrads = torch.autograd.grad(want, dbl)
    # float32 throughout: sums of at most 1024 terms in a chain of six such steps
    bound = 6 * 1024 * U
    assert float((out.double() - ref).norm() / ref.norm()) < bound
    assert abs(float(total) - float(want)) < bound * abs(float(want))
    for n, x, y in zip(["attended", "fused"] + names + ["pet"], grads, wgrads):
        assert float((x.double() - y).norm()) <= 4 * bound * float(y.norm()) + 1e-9, n
    block.eval()
    with torch.no_grad():
        e = block(attended, fused)
    h = plain.layer_norm((r + a).detach(), w1.detach(), b1.detach(), 1e-5)[0]
    ffn = plain.gated_feed_forward(h, wg.detach(), wu.detach(), wd.detach(), "silu")
    ref = plain.layer_norm(h + ffn, w2.detach(), b2.detach(), 1e-5)[0]
    assert float((e.double() - ref).norm() / ref.norm()) < bound
