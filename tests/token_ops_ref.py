"""Plain 64-bit forms of the transformer-block operators (CPU) with the error bounds that the tests of the kernels use.

Every bound is worst-case arithmetic: u = 2^-24 per fp32 operation, half(t) = eps(t) / 2 per rounding to the tensor's type, a sum of n terms in any order is off
by at most n u times the sum of the magnitudes."""
import math

import torch

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half(t):
    return torch.finfo(t).eps / 2


def within(got, ref, bound, what=""):
    """every element finite where the reference is, and within its bound"""
    got = got.detach().to(ref.device).double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got - ref).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].max()), float((bound + torch.zeros_like(off))[bad].min()))


# ------------------------------------------------------------------------------------------------ rotary positions
def rope(x, pos, heads, parts, rotated, dh, axes, theta, layout, inverse):
    """(y, bound) in 64 bits; x any type"""
    v = x.detach().cpu().double().reshape(-1, heads, parts, dh)
    y, mag = v.clone(), torch.zeros_like(v)
    n = sum(axes) // 2
    p = 0
    for a, w in enumerate(axes):
        for j in range(w // 2):
            ang = pos[:, a].cpu().double() * theta ** (-2.0 * j / w)
            c, s = torch.cos(ang)[:, None, None], torch.sin(ang)[:, None, None] * (-1.0 if inverse else 1.0)
            i1, i2 = (p, p + n) if layout == "halves" else (2 * p, 2 * p + 1)
            x1, x2 = v[:, :, :rotated, i1], v[:, :, :rotated, i2]
            y[:, :, :rotated, i1], y[:, :, :rotated, i2] = x1 * c - x2 * s, x1 * s + x2 * c
            mag[:, :, :rotated, i1] = mag[:, :, :rotated, i2] = x1.abs() + x2.abs()
            p += 1
    # sine / cosine: the turn rounded to fp32 (2 pi 2^-26), the function within 2 ulp (4 u), a product and a sum each (2 u)
    bound = mag * (2 * math.pi * 2.0 ** -26 + 6 * U) + torch.where(mag > 0, half(x.dtype) * y.abs() * 1.001 + 2.0 ** -25 * (x.dtype == torch.float16), 0.0)
    return y.reshape(x.shape), bound.reshape(x.shape)


# ------------------------------------------------------------------------------------------------ dropout
def kept(seed, offset, count, keep):
    """Philox4x32-10 in Python integers: does the generator keep element i?"""
    out = []
    lim = math.ceil(float(torch.tensor(keep, dtype=torch.float32)) * 2 ** 24)
    M = 0xFFFFFFFF
    for call in range((count + 3) // 4):
        at = (offset + call) & 0xFFFFFFFFFFFFFFFF
        c, k0, k1 = [at & M, at >> 32, 0x5355, 0x4850], seed & M, (seed >> 32) & M
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k0, b & M, (a >> 32) ^ c[3] ^ k1, a & M]
            k0, k1 = (k0 + 0x9E3779B9) & M, (k1 + 0xBB67AE85) & M
        out += [(w >> 8) < lim for w in c]
    return torch.tensor(out[:count], dtype=torch.bool)


def dropout(x, held, keep, skip=None):
    v = x.detach().cpu().double()
    d = torch.where(held.view(v.shape), v / keep, torch.zeros((), dtype=torch.float64))
    y = d if skip is None else d + skip.detach().cpu().double()
    # keep and 1 / keep in fp32 (2 u), the product (u), the sum (u), the rounding to the type: half(t) of the value, but below 2^-14 the steps of fp16 are
    # 2^-24 wide whatever the value (subnormals), so the rounding there is off by up to 2^-25
    bound = 4 * U * (d.abs() + (0 if skip is None else skip.detach().cpu().double().abs())) + half(x.dtype) * 1.001 * y.abs()
    if x.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    return y, bound


# ------------------------------------------------------------------------------------------------ layer norm
def layernorm(x, dy, eps, gamma, beta, skip=None):
    """dict of (value, bound) for y, dx, dgamma, dbeta"""
    t, c, rows = x.dtype, x.shape[-1], x.numel() // x.shape[-1]
    X, D = x.cpu().double().reshape(rows, c), dy.cpu().double().reshape(rows, c)
    G = gamma.cpu().double() if gamma is not None else torch.ones(c, dtype=torch.float64)
    B = beta.cpu().double() if beta is not None else torch.zeros(c, dtype=torch.float64)
    mean = X.mean(1, keepdim=True)
    var = ((X - mean) ** 2).mean(1, keepdim=True)
    rs = 1 / torch.sqrt(var + eps)
    xh = (X - mean) * rs
    y = xh * G + B
    # mean: c additions; variance: c additions of squares of differences that are off by the mean's error; root, division, products
    n = c + 4
    e_mean = n * U * X.abs().mean(1, keepdim=True)
    e_diff = e_mean + 2 * U * ((X - mean).abs() + e_mean)
    e_rs = rs * (0.5 * (n * U + 2 * (e_diff * (X - mean).abs()).mean(1, keepdim=True) / (var + eps) + (e_diff ** 2).mean(1, keepdim=True) / (var + eps)) + 4 * U)
    e_xh = e_diff * rs + (X - mean).abs() * e_rs + 2 * U * xh.abs()
    out = {"y": (y, e_xh * G.abs() + 3 * U * (xh.abs() * G.abs() + B.abs()) + half(t) * 1.001 * y.abs() + 2.0 ** -25)}
    g = D * G
    s0, s1 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rs * (g - s0 - xh * s1)
    e_s0 = n * U * g.abs().mean(1, keepdim=True)
    e_s1 = n * U * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    inner = g.abs() + s0.abs() + xh.abs() * s1.abs()
    e_dx = rs * (e_s0 + e_xh * s1.abs() + xh.abs() * e_s1 + 5 * U * inner) + e_rs * inner
    if skip is not None:
        dx = dx + skip.cpu().double().reshape(rows, c)
    out["dx"] = (dx, e_dx * 1.01 + U * dx.abs() + half(t) * 1.001 * dx.abs() + 2.0 ** -25)
    out["dgamma"] = ((D * xh).sum(0), (rows + 4) * U * (D * xh).abs().sum(0) + (D.abs() * e_xh).sum(0) + 1e-30)
    out["dbeta"] = (D.sum(0), (rows + 4) * U * D.abs().sum(0) + 1e-30)
    return {k: (v.reshape(x.shape) if k in ("y", "dx") else v, b.reshape(x.shape) if k in ("y", "dx") else b) for k, (v, b) in out.items()}


# ------------------------------------------------------------------------------------------------ gated feed-forward block
def _phi(g):
    return 0.5 * torch.erfc(-g / math.sqrt(2.0))


def act(g, name):
    """act, act', and bounds of |act'| and |act''|"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), 1.1, 0.5
    if name == "gelu":
        return g * _phi(g), _phi(g) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi), 1.13, 0.8
    if name == "sigmoid":
        s = torch.sigmoid(g)
        return s, s * (1 - s), 0.25, 0.1
    if name == "none":
        return g, torch.ones_like(g), 1.0, 0.0
    raise ValueError(name)


def gated_ffn(x, wg, wu, wd, bg, bu, bd, dy, name, grad_type=None, device="cpu"):
    """dict of (value, bound): y and, with dy, dx, dwg, dwu, dwd, dbg, dbu, dbd (64-bit products on `device`)"""
    t = x.dtype
    r = half(t) * 1.001
    tiny = 2.0 ** -24 if t == torch.float16 else 0.0                    # (half a step of fp16's subnormals)
    f = lambda v: v.detach().to(device).double()  # noqa: E731
    X, G, W, D = f(x).reshape(-1, x.shape[-1]), f(wg), f(wu), f(wd)
    k, n, o = G.shape[1], G.shape[0], D.shape[0]
    zero = lambda c: torch.zeros(c, dtype=torch.float64, device=device)  # noqa: E731
    Bg, Bu, Bd = (f(b) if b is not None else zero(c) for b, c in ((bg, n), (bu, n), (bd, o)))
    g, u = X @ G.t() + Bg, X @ W.t() + Bu
    e_g = (k + 2) * U * (X.abs() @ G.abs().t() + Bg.abs())
    e_u = (k + 2) * U * (X.abs() @ W.abs().t() + Bu.abs())
    a, da, d1, d2 = act(g, name)
    # the activation itself: exponential and reciprocal within a few u, the error function within 1.5e-7 + 2 u
    e_act = lambda z: (2e-7 + 8 * U) * (1 + z.abs()) if name != "none" else 0.0  # noqa: E731
    h = a * u
    e_a = d1 * e_g + e_act(g)
    e_h = e_a * u.abs() + a.abs() * e_u + e_a * e_u + U * h.abs()
    e_h = e_h + r * (h.abs() + e_h) + tiny
    y = h @ D.t() + Bd
    e_y = e_h @ D.abs().t() + (n + 2) * U * ((h.abs() + e_h) @ D.abs().t() + Bd.abs())
    out = {"y": (y, e_y + r * (y.abs() + e_y) + tiny)}
    if dy is not None:
        Y = f(dy).reshape(-1, o)
        q = half(grad_type) * 1.001 if grad_type is not None else r
        # the backward works on g and u as they were kept: the upper 24 bits, 15 of them behind the leading one
        kept = 2.0 ** -15
        eg, eu = e_g + kept * (g.abs() + e_g), e_u + kept * (u.abs() + e_u)
        dh = Y @ D
        e_dh = (o + 2) * U * (Y.abs() @ D.abs())
        e_da = d2 * eg + e_act(g)
        dg, du = dh * u * da, dh * a
        ua, ea = u.abs() + eu, d1 * eg + e_act(g)
        e_dg = e_dh * ua * (da.abs() + e_da) + dh.abs() * (eu * (da.abs() + e_da) + u.abs() * e_da) + 3 * U * dg.abs()
        e_du = e_dh * (a.abs() + ea) + dh.abs() * ea + 2 * U * du.abs()
        e_dg, e_du = e_dg + r * (dg.abs() + e_dg) + tiny, e_du + r * (du.abs() + e_du) + tiny
        Ag, Au = dg.abs() + e_dg, du.abs() + e_du
        dx = dg @ G + du @ W
        e_dx = e_dg @ G.abs() + e_du @ W.abs() + (2 * n + 2) * U * (Ag @ G.abs() + Au @ W.abs())
        out["dx"] = (dx, e_dx + r * (dx.abs() + e_dx) + tiny)
        m = X.shape[0]
        for key, left, e_left, right, e_right in (("dwg", dg, e_dg, X, None), ("dwu", du, e_du, X, None), ("dwd", Y, None, h, e_h)):
            v = left.t() @ right
            al, ar = left.abs() + (e_left if e_left is not None else 0), right.abs() + (e_right if e_right is not None else 0)
            e = (m + 2) * U * (al.t() @ ar)
            if e_left is not None:
                e = e + e_left.t() @ ar
            if e_right is not None:
                e = e + al.t() @ e_right
            out[key] = (v, e + q * (v.abs() + e) + tiny)
        for key, v, e in (("dbg", dg, e_dg), ("dbu", du, e_du), ("dbd", Y, torch.zeros_like(Y))):
            s = v.sum(0)
            es = e.sum(0) + (m + 2) * U * (v.abs() + e).sum(0)
            out[key] = (s, es + q * (s.abs() + es) + tiny)
    shape = {"y": x.shape[:-1] + (o,), "dx": x.shape}
    return {key: (v.reshape(shape.get(key, v.shape)), b.reshape(shape.get(key, b.shape))) for key, (v, b) in out.items()}
