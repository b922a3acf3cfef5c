"""Workloads of the transformer-block operators: rotary positions with several axes, the gated feed-forward block, dropout without a stored mask
and 16-bit layer norm, each forward and backward, with their plain forms in elementary torch operations.

A case is a dict with "op" and that operator's sizes.  Types are named "fp32", "bf16", "fp16"; `run` takes the plain form or, where `own` is true,
the calls that a program makes of semiuhpe_amd.kernels.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one new token through a feed-forward block: the weights are read once for one row
        dict(name="ffn_token_bf16", op="ffn", m=1, k=2048, n=5632, out=2048, dtype="bf16", act="silu", bias=False, train=False),
        # a handful of rows (a small batch of crops' class tokens), fp16, biases, sizes that no vector width divides
        dict(name="ffn_few_fp16", op="ffn", m=13, k=1001, n=2727, out=1001, dtype="fp16", act="gelu", bias=True, train=False),
        # the last TinyViT stage's block at the training batch (32 + 128 images of 7 x 7 tokens, 576 channels), forward and backward in fp32
        dict(name="ffn_stage_fp32", op="ffn", m=7840, k=576, n=1536, out=576, dtype="fp32", act="silu", bias=True, train=True),
        # the 14 x 14 stage (160 x 196 tokens, 384 channels), forward and backward in bf16
        dict(name="ffn_stage_bf16", op="ffn", m=31360, k=384, n=1024, out=384, dtype="bf16", act="silu", bias=True, train=True),
        # a large block's training pass
        dict(name="ffn_large_bf16", op="ffn", m=16384, k=2048, n=5632, out=2048, dtype="bf16", act="silu", bias=False, train=True),
        # q and k of the 14 x 14 stage's packed qkv rows (12 heads of 32), two axes (height, width)
        dict(name="rope_stage_fp32", op="rope", t=160, h=14, w=14, heads=12, dh=32, parts=3, axes="16,16", layout="halves", inverse=False, far=0, dtype="fp32"),
        # gradient of the queries of a clip: 16 frames of 45 x 80 patches, three axes
        dict(name="rope_clip_bf16", op="rope", t=16, h=45, w=80, heads=16, dh=128, parts=1, axes="32,48,48", layout="halves", inverse=True, far=0, dtype="bf16"),
        # one new token far into a stream, adjacent pairs, a head whose last channels stay as they are
        dict(name="rope_token_fp16", op="rope", t=1, h=1, w=1, heads=32, dh=80, parts=1, axes="32,16,16", layout="adjacent", inverse=False, far=900001, dtype="fp16"),
        # the regression head's dropout on the pooled features of one batch, forward and gradient
        dict(name="dropout_head_fp32", op="dropout", rows=160, c=1280, keep=0.8, skip=False, dtype="fp32"),
        # a block's residual connection: skip + dropout(branch), and the branch's gradient
        dict(name="dropout_residual_bf16", op="dropout", rows=125440, c=192, keep=0.9, skip=True, dtype="bf16"),
        # the norm before a block of the 28 x 28 stage (160 x 784 tokens, 192 channels), forward and backward
        dict(name="norm_stage_bf16", op="norm", rows=125440, c=192, dtype="bf16"),
        # a width that no vector divides
        dict(name="norm_odd_fp16", op="norm", rows=4099, c=1357, dtype="fp16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "rope", "dropout", "norm"])
    if op == "ffn":
        train = rng.random() < 0.6
        m = _log(rng, 64, 16384) if train else _log(rng, 1, 2048)
        if rng.random() < 0.25:                                        # any width
            k, n = _log(rng, 48, 1500), _log(rng, 64, 4000)
        else:                                                          # multiples of 8
            k, n = 8 * _log(rng, 12, 256), 8 * _log(rng, 16, 704)
        return dict(op=op, m=m, k=k, n=n, out=k if rng.random() < 0.8 else 8 * _log(rng, 12, 256), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    act=rng.choice(["silu", "gelu"]), bias=rng.random() < 0.5, train=train)
    if op == "rope":
        dh = rng.choice([24, 32, 48, 64, 80, 96, 128])
        axes = ",".join(str(v) for v in rng.choice([[dh], [dh // 4 * 2, dh - dh // 4 * 2], [dh // 8 * 2] * 3]))
        parts = rng.choice([1, 3])
        return dict(op=op, t=_log(rng, 1, 24), h=_log(rng, 1, 48), w=_log(rng, 1, 48), heads=rng.randint(1, 20), dh=dh, parts=parts, axes=axes,
                    layout=rng.choice(["halves", "adjacent"]), inverse=rng.random() < 0.5, far=rng.choice([0, _log(rng, 1000, 1000000)]),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]))
    if op == "dropout":
        return dict(op=op, rows=_log(rng, 1, 130000), c=_log(rng, 1, 400), keep=rng.choice([0.5, 0.8, 0.9, 0.95]), skip=rng.random() < 0.5,
                    dtype=rng.choice(["fp32", "bf16", "fp16"]))
    return dict(op=op, rows=_log(rng, 1, 40000), c=_log(rng, 8, 1500), dtype=rng.choice(["bf16", "fp16"]))


def _normal(gen, shape, scale, dtype):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(TYPES[dtype])


def _axes(case):
    return [int(v) for v in case["axes"].split(",")]


def _positions(case):
    grids = torch.meshgrid(torch.arange(case["t"]), torch.arange(case["h"]), torch.arange(case["w"]), indexing="ij")
    every = torch.stack([g.reshape(-1) for g in grids], dim=1)         # (tokens, 3): time, height, width
    return (every[:, 3 - len(_axes(case)):] + case["far"]).to(torch.int32).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    d = case["dtype"]
    s = dict(case=case)
    if case["op"] == "ffn":
        m, k, n, o = case["m"], case["k"], case["n"], case["out"]
        s.update(x=_normal(gen, (m, k), 1.0, d), wg=_normal(gen, (n, k), k ** -0.5, d), wu=_normal(gen, (n, k), k ** -0.5, d),
                 wd=_normal(gen, (o, n), n ** -0.5, d), bg=None, bu=None, bd=None)
        if case["bias"]:
            s.update(bg=_normal(gen, (n,), 0.1, d), bu=_normal(gen, (n,), 0.1, d), bd=_normal(gen, (o,), 0.1, d))
        if case["train"]:
            s.update(dy=_normal(gen, (m, o), 1.0, d))
    elif case["op"] == "rope":
        rows = case["t"] * case["h"] * case["w"]
        s.update(x=_normal(gen, (rows, case["heads"] * case["parts"] * case["dh"]), 1.0, d), pos=_positions(case).cuda())
        if own:                                                        # the frequency table that a model builds once
            from semiuhpe_amd import kernels as K
            s.update(plan=K.RopeAxes(case["dh"], _axes(case), theta=10000.0, layout=case["layout"], device="cuda"))
    elif case["op"] == "dropout":
        shape = (case["rows"], case["c"])
        s.update(x=_normal(gen, shape, 1.0, d), skip=_normal(gen, shape, 1.0, d) if case["skip"] else None, dy=_normal(gen, shape, 1.0, d),
                 counter=torch.tensor([0x5DEECE66D * (seed + 1) % (1 << 62), 1000003 * seed], dtype=torch.int64, device="cuda"), position=77)
    else:
        shape = (case["rows"], case["c"])
        s.update(x=_normal(gen, shape, 1.5, d) + 0.5, gamma=1.0 + 0.1 * torch.randn(case["c"], generator=gen, device="cuda"),
                 beta=0.1 * torch.randn(case["c"], generator=gen, device="cuda"), dy=_normal(gen, shape, 1.0, d))
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _act(g, act):
    """act(g) and act'(g)"""
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return g * p, p * (1.0 + g * (1.0 - p))
    c = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * c, c + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_ffn(s):
    case, t = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[n].float() for n in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        g, u = g + s["bg"].float(), u + s["bu"].float()
    a, da = _act(g, case["act"])
    h = a * u
    y = h @ wd.t()
    if case["bias"]:
        y = y + s["bd"].float()
    if not case["train"]:
        return [y.to(t)]
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    out = [y, dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ h]
    if case["bias"]:
        out += [dg.sum(0), du.sum(0), dy.sum(0)]
    return [o.to(t) for o in out]


def _pair_axes(case):
    """(axis, index within the axis' pairs, axis width) of every rotated pair"""
    return [(a, j, w) for a, w in enumerate(_axes(case)) for j in range(w // 2)]


def _plain_rope(s):
    case, x = s["case"], s["x"]
    pairs = torch.tensor(_pair_axes(case), device=x.device)
    freq = torch.exp(-math.log(10000.0) * 2.0 * pairs[:, 1].double() / pairs[:, 2].double())
    angle = s["pos"].double()[:, pairs[:, 0]] * freq                   # (rows, pairs)
    cos, sin = torch.cos(angle).float()[:, None, None], torch.sin(angle).float()[:, None, None]
    if case["inverse"]:
        sin = -sin
    n = pairs.shape[0]
    at = torch.arange(n, device=x.device)
    first, second = (at, at + n) if case["layout"] == "halves" else (2 * at, 2 * at + 1)
    y = x.view(x.shape[0], case["heads"], case["parts"], case["dh"]).float()
    turned = 2 if case["parts"] == 3 else 1
    x1, x2 = y[:, :, :turned, first], y[:, :, :turned, second]
    y = y.clone()
    y[:, :, :turned, first] = x1 * cos - x2 * sin
    y[:, :, :turned, second] = x1 * sin + x2 * cos
    return [y.view_as(x).to(x.dtype)]


def _times(a, m):
    """high and low 32 bits of the product of 32-bit values a (held in int64) and the constant m"""
    lo, hi = a * (m & 0xFFFF), a * (m >> 16)
    mid = (lo >> 16) + (hi & 0xFFFF)
    return (hi >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)


def _uniform(counter, position, count):
    """`count` 24-bit uniform numbers of the Philox4x32-10 generator keyed by counter[0], from call counter[1] + position on"""
    mask = 0xFFFFFFFF
    at = torch.arange((count + 3) // 4, device=counter.device) + (counter[1] + position)
    c0, c1 = at & mask, (at >> 32) & mask
    c2, c3 = torch.full_like(c0, 0x5355), torch.full_like(c0, 0x4850)
    k0, k1 = counter[0] & mask, (counter[0] >> 32) & mask
    for _ in range(10):
        h0, l0 = _times(c0, 0xD2511F53)
        h1, l1 = _times(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:count]
    return (words >> 8).float() * 2.0 ** -24


def _plain_dropout(s):
    x, keep = s["x"], s["case"]["keep"]
    held = (_uniform(s["counter"], s["position"], x.numel()) < torch.tensor(keep, dtype=torch.float32, device=x.device)).view(x.shape)
    scale = torch.where(held, 1.0 / keep, 0.0)
    y = x.float() * scale
    if s["skip"] is not None:
        y = s["skip"].float() + y
    return [y.to(x.dtype), (s["dy"].float() * scale).to(x.dtype)]


def _plain_norm(s):
    x, dy, gamma = s["x"].float(), s["dy"].float(), s["gamma"]
    centred = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + 1e-5)
    xhat = centred * rstd
    y = xhat * gamma + s["beta"]
    t = dy * gamma
    dx = rstd * (t - t.mean(1, keepdim=True) - xhat * (t * xhat).mean(1, keepdim=True))
    return [y.to(s["x"].dtype), dx.to(s["x"].dtype), (dy * xhat).sum(0), dy.sum(0)]


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_ffn(s):
    from semiuhpe_amd import kernels as K
    case = s["case"]
    w = [s[n] for n in ("wg", "wu", "wd")]
    b = [s[n] for n in ("bg", "bu", "bd")]
    y, saved = K.gated_ffn_fwd(s["x"], *w, *b, act=case["act"], save=case["train"])
    if not case["train"]:
        return [y]
    dw = [torch.empty_like(v) for v in w]
    db = [torch.empty_like(v) for v in b if v is not None]
    dx = K.gated_ffn_bwd(s["dy"], s["x"], *w, saved, case["act"], *dw, *db)
    return [y, dx] + dw + db


def _own_rope(s):
    from semiuhpe_amd import kernels as K
    case = s["case"]
    return [K.rope_axes(s["x"], s["pos"], s["plan"], case["heads"], parts=case["parts"], rotated=2 if case["parts"] == 3 else 1, inverse=case["inverse"])]


def _own_dropout(s):
    from semiuhpe_amd import kernels as K
    keep = s["case"]["keep"]
    return [K.dropout_apply(s["x"], keep, s["counter"], s["position"], skip=s["skip"]), K.dropout_apply(s["dy"], keep, s["counter"], s["position"])]


def _own_norm(s):
    from semiuhpe_amd import kernels as K
    x, c = s["x"], s["x"].shape[1]
    y, mean, rstd = K.layernorm_fwd(x, c, 1e-5, s["gamma"], s["beta"])
    dgamma, dbeta = torch.empty_like(s["gamma"]), torch.empty_like(s["beta"])
    dx = K.layernorm_bwd(x, s["dy"], c, mean, rstd, s["gamma"], dgamma, dbeta)
    return [y, dx, dgamma, dbeta]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"ffn": _own_ffn, "rope": _own_rope, "dropout": _own_dropout, "norm": _own_norm}[op](state)
    return {"ffn": _plain_ffn, "rope": _plain_rope, "dropout": _plain_dropout, "norm": _plain_norm}[op](state)


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "ffn":
        m, k, n, o = case["m"], case["k"], case["n"], case["out"]
        weights = 2 * n * k + o * n + ((2 * n + o) if case["bias"] else 0)
        if case["train"]:
            return dict(bytes=size * (2 * m * k + 2 * m * o + 2 * weights), flops=6 * m * n * (2 * k + o))
        return dict(bytes=size * (m * k + m * o + weights), flops=2 * m * n * (2 * k + o))
    if case["op"] == "rope":
        rows = case["t"] * case["h"] * case["w"]
        elements = rows * case["heads"] * case["parts"] * case["dh"]
        turned = rows * case["heads"] * (2 if case["parts"] == 3 else 1) * sum(_axes(case))
        return dict(bytes=2 * size * elements + 4 * rows * len(_axes(case)), flops=3 * turned)
    count = case["rows"] * case["c"]
    if case["op"] == "dropout":
        return dict(bytes=size * count * (5 if case["skip"] else 4), flops=2 * count * 2)
    return dict(bytes=size * count * 5 + 16 * case["c"], flops=20 * count)  # forward: x, y; backward: x, dy, dx


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def _exact_ffn(s):
    case = s["case"]
    D = {n: s[n].double() if s[n] is not None else 0.0 for n in ("x", "wg", "wu", "wd", "bg", "bu", "bd")}
    gate = torch.addmm(D["bg"] + torch.zeros(case["n"], dtype=torch.float64, device="cuda"), D["x"], D["wg"].t())
    up = torch.addmm(D["bu"] + torch.zeros(case["n"], dtype=torch.float64, device="cuda"), D["x"], D["wu"].t())
    if case["act"] == "silu":
        sig = torch.sigmoid(gate)
        a, slope = gate * sig, sig + gate * sig * (1 - sig)
    else:
        cdf = 0.5 * torch.erfc(-gate / math.sqrt(2))
        a, slope = gate * cdf, cdf + gate * torch.exp(-gate ** 2 / 2) / math.sqrt(2 * math.pi)
    h = a * up
    y = torch.mm(h, D["wd"].t()) + D["bd"]
    if not case["train"]:
        return [y]
    dy = s["dy"].double()
    dh = torch.mm(dy, D["wd"])
    dgate, dup = dh * up * slope, dh * a
    out = [y, torch.mm(dgate, D["wg"]) + torch.mm(dup, D["wu"]), torch.mm(dgate.t(), D["x"]), torch.mm(dup.t(), D["x"]), torch.mm(dy.t(), h)]
    if case["bias"]:
        out += [dgate.sum(0), dup.sum(0), dy.sum(0)]
    return out


def _exact_rope(s):
    case = s["case"]
    heads = s["x"].double().reshape(-1, case["heads"], case["parts"], case["dh"]).clone()
    sign = -1.0 if case["inverse"] else 1.0
    half = sum(_axes(case)) // 2
    for part in range(2 if case["parts"] == 3 else 1):
        for p, (axis, j, width) in enumerate(_pair_axes(case)):
            i1, i2 = (p, p + half) if case["layout"] == "halves" else (2 * p, 2 * p + 1)
            turn = torch.polar(torch.ones(heads.shape[0], dtype=torch.float64, device="cuda"), sign * s["pos"][:, axis].double() * 10000.0 ** (-2.0 * j / width))
            z = torch.complex(heads[:, :, part, i1], heads[:, :, part, i2]) * turn[:, None]
            heads[:, :, part, i1], heads[:, :, part, i2] = z.real, z.imag
    return [heads.reshape(s["x"].shape)]


def _exact_dropout(s):
    """the generator in numpy's unsigned 64-bit integers"""
    count, keep = s["x"].numel(), np.float32(s["case"]["keep"])
    seed, base = (int(v) for v in s["counter"].cpu())
    low = np.uint64(0xFFFFFFFF)
    at = np.arange((count + 3) // 4, dtype=np.uint64) + np.uint64(base + s["position"])
    c = [at & low, at >> np.uint64(32), np.full_like(at, 0x5355), np.full_like(at, 0x4850)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    held = ((np.stack(c, 1).reshape(-1)[:count] >> np.uint64(8)).astype(np.float32) * np.float32(2.0 ** -24)) < keep
    held = torch.from_numpy(held).cuda().view(s["x"].shape)
    pick = lambda v: torch.where(held, v.double() / s["case"]["keep"], torch.zeros((), dtype=torch.float64, device="cuda"))  # noqa: E731
    y = pick(s["x"])
    return [y if s["skip"] is None else y + s["skip"].double(), pick(s["dy"])]


def _exact_norm(s):
    x, dy, gamma = s["x"].double(), s["dy"].double(), s["gamma"].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    xhat = (x - mean) / torch.sqrt(var + 1e-5)
    t = dy * gamma
    along = (t * xhat).sum(1, keepdim=True) / x.shape[1]
    dx = (t - t.sum(1, keepdim=True) / x.shape[1] - xhat * along) / torch.sqrt(var + 1e-5)
    return [xhat * gamma + s["beta"].double(), dx, (dy * xhat).sum(0), dy.sum(0)]


def exact(case, seed):
    return {"ffn": _exact_ffn, "rope": _exact_rope, "dropout": _exact_dropout, "norm": _exact_norm}[case["op"]](prepare(case, seed))
