"""The fusion block's layers without a GPU: the plain forms the GPU tests compare with (published
generator vectors, gradients against differences) and what the C entry points refuse."""
import ctypes

import pytest
import torch

import layers_plain as plain


@pytest.mark.parametrize("counter,key,want", [
    # the known-answer vectors published with the generator
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))])
def test_generator_known_answers(counter, key, want):
    assert tuple(plain.philox(counter, key)) == want


@pytest.mark.parametrize("rows,cols,p,seed,offset", [(3, 21, 0.25, (1 << 62) + 12345, (7 << 32) + 5), (2, 8, 0.5, 0, 0)])
def test_plain_mask_is_the_generator(rows, cols, p, seed, offset):
    f = plain.factor(rows, cols, p, seed, offset)
    groups, t = (cols + 7) // 8, plain.threshold(p)
    for r in range(rows):
        for c in range(cols):
            i = r * groups + c // 8
            w = plain.philox((i & 0xFFFFFFFF, i >> 32, offset & 0xFFFFFFFF, offset >> 32), (seed & 0xFFFFFFFF, seed >> 32))
            field = (w[(c % 8) // 2] >> (16 * (c % 2))) & 0xFFFF
            assert float(f[r, c]) == (65536 / (65536 - t) if field >= t else 0.0)


def _difference(f, x, v, h=1e-5):
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


def test_plain_gradients_against_differences():
    """Central differences of step 1e-5 in float64: truncation ~ h^2 = 1e-10 and rounding
    ~ 2^-53 / h = 1e-11, both relative to sums of at most ~100 terms of order 1: 1e-6 holds."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, dtype=torch.float64, generator=g)
    x, w, b, dy = r(5, 12), r(12), r(12), r(5, 12)
    _, xhat, rstd = plain.layer_norm(x, w, b, 1e-5)
    dx, dw, db = plain.layer_norm_backward(dy, xhat, rstd, w)
    loss = lambda x, w, b: (plain.layer_norm(x, w, b, 1e-5)[0] * dy).sum()
    for grad, f, at in ((dx, lambda t: loss(t, w, b), x), (dw, lambda t: loss(x, t, b), w), (db, lambda t: loss(x, w, t), b)):
        v = r(*at.shape)
        assert abs(float(_difference(f, at, v) - (grad * v).sum())) < 1e-6
    for name in ("silu", "gelu"):
        args = [r(4, 6), r(9, 6), r(9, 6), r(6, 9)]
        dy2 = r(4, 6)
        _, *grads = plain.gated_feed_forward(*args, name, dy2)
        for i, grad in enumerate(grads):
            v = r(*args[i].shape)
            f = lambda t: (plain.gated_feed_forward(*args[:i], t, *args[i + 1:], name) * dy2).sum()
            assert abs(float(_difference(f, args[i], v) - (grad * v).sum())) < 1e-6 * max(1.0, float(grad.norm()))


# ---------------------------------------------------------------- refusals (no HIP call is made)
@pytest.fixture(scope="module")
def clib():
    from otfuse import _lib as L
    return L, L.lib()


BUF = (ctypes.c_char * 4096)()
P = (ctypes.addressof(BUF) + 255) // 256 * 256   # 256-byte aligned host memory: never read by a refused call


def test_dropout_refuses(clib):
    L, lib = clib
    def call(x=P, ldx=8, res=None, ldr=0, y=P, ldy=8, rows=2, cols=8, dt=L.OTF_F32, p=0.5, rng=P):
        return lib.otf_dropout(x, ldx, res, ldr, y, ldy, rows, cols, dt, p, rng, None)
    for kw in (dict(x=None), dict(y=None), dict(rng=None), dict(rng=P + 4), dict(ldx=7), dict(ldy=7), dict(res=P, ldr=7),
               dict(rows=-1), dict(cols=-1), dict(dt=L.OTF_F64), dict(dt=9), dict(p=-0.1), dict(p=1.1),
               dict(p=float("nan")), dict(x=P + 2), dict(y=P + 1, dt=L.OTF_F16)):
        assert call(**kw) == L.OTF_EINVAL, kw
    assert call(cols=2 ** 31, ldx=2 ** 31, ldy=2 ** 31) == L.OTF_EUNSUPPORTED
    assert call(rows=0, x=None, y=None) == L.OTF_OK and call(cols=0) == L.OTF_OK
    assert call(p=2.0 ** -17, rng=None) == L.OTF_EINVAL   # rounds to 2^-16: needs the state


def test_layer_norm_refuses(clib):
    L, lib = clib
    def fwd(x=P, ldx=8, dt=L.OTF_F16, w=P, b=P, wdt=L.OTF_F32, eps=1e-5, rows=2, cols=8, y=P, ldy=8, mean=P, rstd=P):
        return lib.otf_layer_norm(x, ldx, dt, w, b, wdt, eps, rows, cols, y, ldy, mean, rstd, None)
    for kw in (dict(x=None), dict(y=None), dict(ldx=7), dict(ldy=7), dict(cols=0), dict(rows=-1), dict(eps=-1.0),
               dict(eps=float("nan")), dict(mean=None), dict(rstd=None), dict(dt=L.OTF_F64), dict(wdt=L.OTF_BF16),
               dict(x=P + 1), dict(w=P + 2), dict(b=P + 1)):
        assert fwd(**kw) == L.OTF_EINVAL, kw
    assert fwd(cols=2 ** 31, ldx=2 ** 31, ldy=2 ** 31) == L.OTF_EUNSUPPORTED
    assert fwd(rows=0, x=None) == L.OTF_OK
    need = lib.otf_layer_norm_backward_workspace_size(1000, 8)
    assert need > 0 and lib.otf_layer_norm_backward_workspace_size(0, 8) == 0
    def bwd(dy=P, x=P, mean=P, rows=1000, dx=P, dw=P, ws=P, size=need, lddy=8, dt=L.OTF_F16, wdt=L.OTF_F32):
        return lib.otf_layer_norm_backward(dy, lddy, x, 8, dt, P, wdt, mean, P, rows, 8, dx, 8, dw, P, ws, size, None)
    for kw in (dict(dy=None), dict(x=None), dict(mean=None), dict(dx=None), dict(ws=None), dict(size=need - 1),
               dict(ws=P + 4), dict(lddy=7), dict(dw=P + 2), dict(dt=L.OTF_F64), dict(wdt=L.OTF_BF16)):
        assert bwd(**kw) == L.OTF_EINVAL, kw


def test_dropout_add_layer_norm_refuses(clib):
    L, lib = clib
    def fwd(x=P, dt=L.OTF_BF16, r=P, rdt=L.OTF_F32, p=0.1, rng=P, y=P, z=P, rows=2, ldz=8, ldr=8):
        return lib.otf_dropout_add_layer_norm(x, 8, dt, r, ldr, rdt, P, P, L.OTF_F32, 1e-5, p, rng, rows, 8, y, 8, z, ldz,
                                              None, None, None)
    for kw in (dict(x=None), dict(r=None), dict(y=None), dict(z=None), dict(rng=None), dict(rng=P + 4), dict(p=2.0),
               dict(rdt=L.OTF_F16), dict(ldz=7), dict(ldr=7), dict(z=P + 2), dict(dt=L.OTF_F64)):
        assert fwd(**kw) == L.OTF_EINVAL, kw
    assert fwd(rows=0, x=None) == L.OTF_OK
    def bwd(dy=P, z=P, x=None, r=None, ldr=8, rdt=L.OTF_F32, p=0.1, rng=P, dx=P, dr=P, dz=P, lddz=8):
        return lib.otf_dropout_add_layer_norm_backward(dy, 8, dz, lddz, z, 8, x, 8, r, ldr, L.OTF_BF16, rdt, P, L.OTF_F32, P,
                                                       P, p, rng, 2, 8, dx, 8, dr, 8, None, None, None, 0, None)
    for kw in (dict(dy=None), dict(z=None), dict(p=-1.0), dict(rng=None), dict(dx=None), dict(dr=None), dict(lddz=7),
               dict(dz=P + 2), dict(rdt=L.OTF_BF16), dict(rdt=L.OTF_BF16, x=P), dict(rdt=L.OTF_BF16, r=P),
               dict(rdt=L.OTF_BF16, x=P, r=P, ldr=7), dict(rdt=L.OTF_BF16, x=P, r=P + 1)):
        assert bwd(**kw) == L.OTF_EINVAL, kw


def _args(L, **kw):
    a = L.FfnArgs(rows=20, d=16, f=24, dtype=L.OTF_BF16, activation=0, x=P, ldx=16, w_gate=P, w_up=P, ldw_in=16, w_down=P,
                  ldw_down=24, y=P, ldy=16, saved=P, dy=P, lddy=16, dx=P, lddx=16, dw_gate=P, dw_up=P, lddw_in=16,
                  dw_down=P, lddw_down=24)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_gated_ffn_refuses(clib):
    L, lib = clib
    def fwd(ws=P, size=1 << 30, **kw):
        return lib.otf_gated_ffn(ctypes.byref(_args(L, **kw)), ws, size, None)
    def bwd(ws=P, size=1 << 30, **kw):
        return lib.otf_gated_ffn_backward(ctypes.byref(_args(L, **kw)), ws, size, None)
    for kw in (dict(x=None), dict(w_gate=None), dict(w_up=None), dict(w_down=None), dict(y=None), dict(ldx=15),
               dict(ldw_in=15), dict(ldw_down=23), dict(ldy=15), dict(d=0), dict(f=0), dict(rows=-1), dict(dtype=L.OTF_F64),
               dict(activation=2), dict(x=P + 1), dict(saved=P + 8), dict(ws=P + 8), dict(ldx=(1 << 20) + 8)):
        assert fwd(**kw) == L.OTF_EINVAL, kw
    need = lib.otf_gated_ffn_workspace_size(ctypes.byref(_args(L, saved=None)))
    assert need >= 20 * 24 * 2   # h
    assert fwd(saved=None, ws=None) == L.OTF_EINVAL and fwd(saved=None, size=need - 1) == L.OTF_EINVAL
    assert fwd(d=(1 << 20) + 1) == L.OTF_EUNSUPPORTED and fwd(rows=1 << 30) == L.OTF_EUNSUPPORTED
    assert fwd(d=1 << 18, f=1 << 18) == L.OTF_EUNSUPPORTED and fwd(rows=1 << 26, f=1 << 12) == L.OTF_EUNSUPPORTED
    assert fwd(rows=0, x=None) == L.OTF_OK
    for kw in (dict(dy=None), dict(saved=None), dict(w_down=None), dict(w_up=None), dict(dw_up=None), dict(dw_gate=None),
               dict(lddy=15), dict(lddx=15), dict(lddw_in=15), dict(lddw_down=23), dict(x=None), dict(dx=P + 1),
               dict(ws=None), dict(dtype=7)):
        assert bwd(**kw) == L.OTF_EINVAL, kw
    size = lib.otf_gated_ffn_backward_workspace_size(ctypes.byref(_args(L)))
    assert bwd(size=size - 1) == L.OTF_EINVAL
    # unaligned operands are copied: the workspace grows by them
    odd = lib.otf_gated_ffn_workspace_size(ctypes.byref(_args(L, d=15, x=P + 2)))
    assert odd > lib.otf_gated_ffn_workspace_size(ctypes.byref(_args(L)))


def test_python_entry_points_refuse_host_tensors():
    from otfuse import layers
    x, rng = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: layers.dropout(x, 0.1, rng), lambda: layers.layer_norm(x),
                 lambda: layers.dropout_add_layer_norm(x, x, p=0.1, rng=rng),
                 lambda: layers.gated_feed_forward(x, torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(8, 4))):
        with pytest.raises(TypeError, match="device tensor"):
            call()


def test_missing_nodes_fail_loudly(monkeypatch, tmp_path):
    from otfuse import _lib as L
    from otfuse import layers
    monkeypatch.setattr(layers, "NODES_PATH", str(tmp_path / "missing.so"))
    monkeypatch.setattr(layers, "_nodes", None)
    with pytest.raises(L.OtfError):
        layers._native()
