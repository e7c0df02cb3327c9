"""Plain 64-bit forms of the fusion block's layers (otfuse.layers), for the tests."""
import math

import torch


def philox(counter, key):
    """Philox4x32-10 (Salmon et al., SC 2011) in Python integers: 4 words -> 4 words."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def threshold(p):
    return 65536 if p >= 1 else min(65535, int(math.floor(p * 65536 + 0.5)))


def factor(rows, cols, p, seed, offset, first=0):
    """keep / (1 - p) of rows first... as float64 (rows, cols), on the CPU"""
    t = threshold(p)
    scale = 0.0 if t == 65536 else 65536.0 / (65536 - t)
    groups = (cols + 7) // 8
    off, key = (offset & 0xFFFFFFFF, (offset >> 32) & 0xFFFFFFFF), (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)
    # word arithmetic on int64 tensors: 32 x 32 -> 64 products by 16-bit halves
    at = torch.arange(first * groups, (first + rows) * groups, dtype=torch.int64)
    m32 = 0xFFFFFFFF

    def mul(a, m):
        lo, hi = a * (m & 0xFFFF), a * (m >> 16)
        hi = hi + (lo >> 16)
        return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)

    c = [at & m32, at >> 32, torch.full_like(at, off[0]), torch.full_like(at, off[1])]
    k = list(key)
    for _ in range(10):
        h0, l0 = mul(c[0], 0xD2511F53)
        h1, l1 = mul(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k[0], l1, h0 ^ c[3] ^ k[1], l0]
        k = [(k[0] + 0x9E3779B9) & m32, (k[1] + 0xBB67AE85) & m32]
    fields = torch.stack([f for w in c for f in (w & 0xFFFF, w >> 16)], 1).view(rows, groups * 8)[:, :cols]
    return (fields >= t).double() * scale


def layer_norm(x, w, b, eps):
    """y, xhat, rstd of float64 rows"""
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xhat = (x - mean) * rstd
    return xhat * w + b, xhat, rstd


def layer_norm_backward(dy, xhat, rstd, w):
    """dx, dw, db"""
    c = dy * w
    dx = rstd * (c - c.mean(1, keepdim=True) - xhat * (c * xhat).mean(1, keepdim=True))
    return dx, (dy * xhat).sum(0), dy.sum(0)


def act(g, name):
    """act(g), act'(g)"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * torch.special.erfc(-g / math.sqrt(2))
    return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def gated_feed_forward(x, wg, wu, wd, name, dy=None):
    """y, or with dy also dx, dwg, dwu, dwd"""
    g, u = x @ wg.t(), x @ wu.t()
    a, da = act(g, name)
    h = a * u
    y = h @ wd.t()
    if dy is None:
        return y
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    return y, dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ h
