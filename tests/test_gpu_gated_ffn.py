"""The gated feed-forward block, forward and backward, against its 64-bit form (tests/token_ops_ref.py: the bounds and their arithmetic)."""
import pytest
import torch

import token_ops_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from semiuhpe_amd import kernels
    return kernels


def normal(shape, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(R.TYPES[dtype])


def block(m, k, n, o, dtype, bias):
    x = normal((m, k), dtype, 1)
    w = [normal((n, k), dtype, 2, k ** -0.5), normal((n, k), dtype, 3, k ** -0.5), normal((o, n), dtype, 4, n ** -0.5)]
    b = [normal((c,), dtype, 5 + i, 0.3) if bias else None for i, c in enumerate((n, n, o))]
    return x, w, b, normal((m, o), dtype, 9)


def cuda(ts):
    return [t.cuda() if t is not None else None for t in ts]


def run(K, x, w, b, dy, act, gtype=None):
    xs, ws, bs = x.cuda(), cuda(w), cuda(b)
    y, saved = K.gated_ffn_fwd(xs, *ws, *bs, act=act)
    dw = [torch.full_like(v, float("nan"), dtype=gtype or v.dtype) for v in ws]
    db = [torch.full_like(v, float("nan"), dtype=gtype or v.dtype) if v is not None else None for v in bs]
    dx = K.gated_ffn_bwd(dy.cuda(), xs, *ws, saved, act, *dw, *db)
    return dict(y=y, dx=dx, dwg=dw[0], dwu=dw[1], dwd=dw[2], dbg=db[0], dbu=db[1], dbd=db[2]), (xs, ws, bs, saved, dw, db)


SIZES = [
    # m, k, n, o
    (1, 8, 8, 8),
    (1, 1, 1, 1),
    (1, 64, 128, 64),
    (3, 7, 5, 9),
    (16, 96, 256, 96),
    (2, 9, 8, 3),
    (4, 130, 71, 1),
    (5, 257, 1025, 17),
    (8, 1000, 40, 33),
    (13, 1001, 2727, 1001),
    (32, 200, 333, 70),
    (7, 3, 900, 5),
    (20, 900, 2, 900),
    (17, 33, 65, 31),
    (64, 64, 64, 64),
    (65, 72, 136, 40),
    (49, 192, 512, 192),
    (127, 100, 260, 60),
    (130, 256, 264, 128),
    (257, 136, 328, 200),
    (1000, 16, 24, 16),
    (300, 577, 129, 255),
]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("cfg", SIZES, ids=[str(c) for c in SIZES])
def test_gated_ffn(K, cfg, dtype):
    m, k, n, o = cfg
    bias = m % 2 == 1
    x, w, b, dy = block(m, k, n, o, dtype, bias)
    act = ("silu", "gelu")[k % 2]
    ref = R.gated_ffn(x, *w, *b, dy, act)
    got, (xs, ws, bs, saved, dw, db) = run(K, x, w, b, dy, act)
    for key, (value, bound) in ref.items():
        if got[key] is not None:
            R.within(got[key], value, bound, key)
    y2, none = K.gated_ffn_fwd(xs, *ws, *bs, act=act, save=False)          # serving form: the same values
    assert none is None
    R.within(y2, *ref["y"], "y, save=False")
    again = K.gated_ffn_bwd(dy.cuda(), xs, *ws, saved, act)                # no parameter gradients wanted
    assert torch.equal(again, got["dx"])
    before = [t.clone() for t in dw]
    assert K.gated_ffn_bwd(dy.cuda(), xs, *ws, saved, act, *dw, need_dx=False) is None
    assert all(torch.equal(p, q) for p, q in zip(before, dw))              # (the same bits again)


@pytest.mark.parametrize("cfg", [(4100, 3080, 3336, 3600, "bf16"), (2300, 1000, 2504, 1000, "fp16"), (2100, 520, 1304, 520, "fp32"), (1500, 1003, 1503, 1005, "bf16"),
                                 (20000, 96, 136, 96, "bf16")], ids=str)
def test_large_sizes(K, cfg):
    """the large tiles, reductions split over many workgroups and rows of no whole vector, against 64-bit products"""
    m, k, n, o, dtype = cfg
    x, w, b, dy = block(m, k, n, o, dtype, m % 200 == 100)
    ref = R.gated_ffn(x, *w, *b, dy, "silu", device="cuda")
    got, _ = run(K, x, w, b, dy, "silu")
    for key, (value, bound) in ref.items():
        if got[key] is not None:
            R.within(got[key], value, bound, key)
            off = (got[key].double() - value).norm() / value.norm()
            # random roundings add up as squares: a few half steps of the type (fp32: of its sums of up to 20000 terms) in the 2-norm
            assert float(off) < (6 * R.half(x.dtype) if dtype != "fp32" else 1e-5), (key, float(off))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_more_small_tiles_than_compute_units(K, dtype):
    """small tiles, two to a compute unit (sizes of some hundred small tiles in each product): the form with two buffers"""
    x, w, b, dy = block(4000, 1496, 1520, 1504, dtype, True)
    ref = R.gated_ffn(x, *w, *b, dy, "gelu", device="cuda")
    got, _ = run(K, x, w, b, dy, "gelu")
    for key, (value, bound) in ref.items():
        R.within(got[key], value, bound, key)


def test_saved_must_be_contiguous(K):
    x, w, b, dy = block(40, 16, 24, 16, "bf16", True)
    xs, ws = x.cuda(), cuda(w)
    _, (kept, h) = K.gated_ffn_fwd(xs, *ws, *cuda(b))
    with pytest.raises(ValueError, match="saved"):
        K.gated_ffn_bwd(dy.cuda(), xs, *ws, (torch.zeros(2 * kept.numel(), dtype=torch.uint8, device="cuda")[::2], h))


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "none"])
def test_activations(K, act):
    x, w, b, dy = block(40, 48, 56, 32, "fp32", True)
    ref = R.gated_ffn(x, *w, *b, dy, act)
    got, _ = run(K, x, w, b, dy, act)
    for key, (value, bound) in ref.items():
        R.within(got[key], value, bound, key)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("act", ["relu", "relu6"])
def test_whole_numbers_are_exact(K, act, dtype):
    """small whole numbers: every sum, product and rounding is exact (also at the corners of ReLU and ReLU6), so the results equal the 64-bit form's bits"""
    g = torch.Generator().manual_seed(7)
    pick = lambda *s: torch.randint(-1, 2, s, generator=g).to(R.TYPES[dtype])  # noqa: E731
    m, k, n, o = 24, 8, 16, 8
    x, wg, wu, wd, dy = pick(m, k), pick(n, k), pick(n, k), pick(o, n), pick(m, o)
    X, G, W, D, Y = (t.double() for t in (x, wg, wu, wd, dy))
    gg, uu = X @ G.t(), X @ W.t()
    a = gg.clamp(min=0) if act == "relu" else gg.clamp(0, 6)
    da = ((gg > 0) if act == "relu" else (gg > 0) & (gg < 6)).double()
    h, dh = a * uu, Y @ D
    dg, du = dh * uu * da, dh * a
    got, _ = run(K, x, [wg, wu, wd], [None] * 3, dy, act, torch.float32)
    ref = dict(y=h @ D.t(), dx=dg @ G + du @ W, dwg=dg.t() @ X, dwu=du.t() @ X, dwd=Y.t() @ h)
    for key, v in ref.items():
        assert torch.equal(got[key].cpu(), v.to(got[key].dtype)), key


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_fp32_gradients_and_accumulation(K, dtype):
    x, w, b, dy = block(96, 64, 72, 48, dtype, True)
    ref = R.gated_ffn(x, *w, *b, dy, "silu", grad_type=torch.float32)
    got, (xs, ws, bs, saved, dw, db) = run(K, x, w, b, dy, "silu", torch.float32)
    for key, (value, bound) in ref.items():
        R.within(got[key], value, bound, key)
    once = [t.clone() for t in dw + db]
    K.gated_ffn_bwd(dy.cuda(), xs, *ws, saved, "silu", *dw, *db, accumulate=True)
    assert all(torch.equal(t, 2 * v) for t, v in zip(dw + db, once))


@pytest.mark.parametrize("m", [96, 1500])
def test_accumulation_in_the_weights_type(K, m):
    x, w, b, dy = block(m, 64, 72, 48, "bf16", True)
    _, (xs, ws, bs, saved, dw, db) = run(K, x, w, b, dy, "silu")
    held = [normal(t.shape, "bf16", 30 + i).cuda() for i, t in enumerate(dw + db)]
    out = [t.clone() for t in held]
    exact = [torch.empty_like(t, dtype=torch.float32) for t in dw + db]
    K.gated_ffn_bwd(dy.cuda(), xs, *ws, saved, "silu", *exact)
    K.gated_ffn_bwd(dy.cuda(), xs, *ws, saved, "silu", *out, accumulate=True)
    for t, h0, e in zip(out, held, exact):                              # added in fp32 and rounded once
        assert torch.equal(t, (h0.float() + e).to(torch.bfloat16))


def test_gradients_against_differences(K):
    x, w, b, dy = block(5, 12, 16, 8, "fp32", True)
    got, _ = run(K, x, w, b, dy, "gelu")
    ref = R.gated_ffn(x, *w, *b, dy, "gelu")
    P = [t.double() for t in [x] + w + b]
    f = lambda p: float((R.gated_ffn(p[0], *p[1:4], *p[4:], None, "gelu")["y"][0] * dy.double()).sum())  # noqa: E731
    e = 1e-5
    for i, key in enumerate(("dx", "dwg", "dwu", "dwd", "dbg", "dbu", "dbd")):
        v = normal(P[i].shape, "fp32", 50 + i).double()
        up, down = list(P), list(P)
        up[i], down[i] = P[i] + e * v, P[i] - e * v
        diff = (f(up) - f(down)) / (2 * e)
        bound = float((ref[key][1] * v.abs()).sum()) + 1e-6 * abs(diff) + 1e-6      # (third derivatives times e^2 and 64-bit cancellation: far below)
        assert abs(float((got[key].cpu().double() * v).sum()) - diff) <= bound, key


def test_rows_do_not_touch_each_other(K):
    """a row's result depends on that row alone, bit for bit; a NaN row stays one row; zero rows; leading dimensions"""
    x, w, b, dy = block(70, 64, 96, 64, "bf16", True)
    x[33] = float("nan")
    ws, bs = cuda(w), cuda(b)
    y, _ = K.gated_ffn_fwd(x.cuda(), *ws, *bs)
    assert torch.equal(torch.isnan(y.cpu()).any(1), torch.arange(70) == 33)
    y3, _ = K.gated_ffn_fwd(x[:30].cuda().view(5, 6, 64), *ws, *bs)
    assert y3.shape == (5, 6, 64)
    e = x[:0].cuda()
    y0, saved = K.gated_ffn_fwd(e, *ws, *bs)
    assert y0.shape == (0, 64)
    dw = [torch.full_like(v, 2.0) for v in ws]
    db = [torch.full_like(v, 2.0) for v in bs]
    assert K.gated_ffn_bwd(y0, e, *ws, saved, "silu", *dw, *db, accumulate=True).shape == (0, 64)
    assert all((t == 2).all() for t in dw + db)
    K.gated_ffn_bwd(y0, e, *ws, saved, "silu", *dw, *db)
    assert all((t == 0).all() for t in dw + db)


def test_unaligned_views(K):
    """contiguous views that start off a 16-byte boundary give the aligned copies' results"""
    x, w, b, dy = block(80, 64, 96, 64, "bf16", True)

    def shifted(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.cuda().reshape(-1)
        return buf[1:].view(t.shape)
    ref, _ = run(K, x, w, b, dy, "silu")
    xs, ws, bs, ds = shifted(x), [shifted(t) for t in w], [shifted(t) for t in b], shifted(dy)
    y, saved = K.gated_ffn_fwd(xs, *ws, *bs)
    assert torch.equal(y, ref["y"])
    dw, db = [shifted(torch.zeros_like(t)) for t in w], [shifted(torch.zeros_like(t)) for t in b]
    dx = K.gated_ffn_bwd(ds, xs, *ws, saved, "silu", *dw, *db)
    for got, key in zip([dx] + dw + db, ("dx", "dwg", "dwu", "dwd", "dbg", "dbu", "dbd")):
        assert torch.equal(got, ref[key]), key


def test_buffers_keep_what_lies_behind_them(K):
    """gradient buffers with a guard row behind them"""
    m, k, n, o = 70, 40, 72, 24
    x, w, b, dy = block(m, k, n, o, "bf16", True)
    xs, ws, bs = x.cuda(), cuda(w), cuda(b)
    _, saved = K.gated_ffn_fwd(xs, *ws, *bs)
    guard = [torch.full((t.numel() + 512,), 3.0, dtype=t.dtype, device="cuda") for t in ws + bs]
    K.gated_ffn_bwd(dy.cuda(), xs, *ws, saved, "silu", *[g[:t.numel()].view(t.shape) for g, t in zip(guard, ws + bs)])
    assert all((g[t.numel():] == 3).all() for g, t in zip(guard, ws + bs))


def test_streams_and_graph(K):
    """a captured forward + backward replays to the eager bits, also with another graph captured after it and eager calls between the replays"""
    x, w, b, dy = block(200, 96, 128, 96, "bf16", True)
    x2 = normal((200, 96), "bf16", 77)
    ws, bs = cuda(w), cuda(b)
    xs, ds = x.cuda(), dy.cuda()

    def step(xin):
        y, saved = K.gated_ffn_fwd(xin, *ws, *bs)
        dw, db = [torch.empty_like(t) for t in ws], [torch.empty_like(t) for t in bs]
        dx = K.gated_ffn_bwd(ds, xin, *ws, saved, "silu", *dw, *db)
        return [y, dx] + dw + db
    eager = [[t.clone() for t in step(v)] for v in (xs, x2.cuda())]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step(xs)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(on_side, eager[0]))
    ins, graphs, outs = [xs.clone(), x2.cuda()], [], []
    for v in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(v))
        graphs.append(g)
    for turn in range(3):
        for i in (0, 1):
            for t in outs[i]:
                t.zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs[i], eager[i])), (turn, i)
            step(x2.cuda())
    ins[0].copy_(ins[1])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs[0], eager[1]))


def test_refusals(K):
    x, w, b, dy = block(8, 16, 24, 16, "bf16", True)
    xs, ws, bs, ds = x.cuda(), cuda(w), cuda(b), dy.cuda()
    y, saved = K.gated_ffn_fwd(xs, *ws, *bs)
    for bad in (dict(wu=ws[1][:, :8].contiguous()), dict(wd=ws[2].t().contiguous().t()), dict(wg=ws[0].float()), dict(bg=bs[0][:3]), dict(bd=bs[2].float()),
                dict(act="tanh"), dict(x=xs[:, :8].contiguous()), dict(x=xs.double()), dict(wu=ws[1].cpu())):
        args = dict(x=xs, wg=ws[0], wu=ws[1], wd=ws[2], bg=bs[0], bu=bs[1], bd=bs[2], act="silu")
        args.update(bad)
        with pytest.raises((ValueError, RuntimeError)):
            K.gated_ffn_fwd(**args)
    dw = [torch.empty_like(t) for t in ws]
    for bad in (dict(saved=None), dict(dy=ds[:4]), dict(dwg=dw[0]), dict(dwg=dw[0], dwu=dw[1], dwd=dw[2].float()), dict(dbg=bs[0].half()),
                dict(saved=(saved[0], saved[1][:4])), dict(saved=(saved[0][:4], saved[1])), dict(dwg=dw[0], dwu=dw[1], dwd=dw[1])):
        args = dict(dy=ds, x=xs, wg=ws[0], wu=ws[1], wd=ws[2], saved=saved, act="silu")
        args.update(bad)
        with pytest.raises(ValueError):
            K.gated_ffn_bwd(**args)
