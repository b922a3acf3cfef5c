"""Rotary positions, dropout without a stored mask and 16-bit LayerNorm against 64-bit forms (tests/token_ops_ref.py: the bounds and their arithmetic)."""
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


# ------------------------------------------------------------------------------------------------ rotary positions
ROPE = [
    # rows, heads, parts, rotated, dh, axes
    (1, 1, 1, 1, 2, (2,)),
    (1, 32, 1, 1, 80, (32, 16, 16)),
    (37, 3, 3, 2, 32, (16, 16)),            # packed qkv rows
    (196, 12, 3, 2, 32, (16, 16)),
    (5, 2, 3, 1, 24, (8, 8)),               # channels 16 .. 23 stay
    (9, 5, 2, 2, 48, (16, 16, 16)),
    (7, 3, 1, 1, 33, (10, 6)),              # odd head width: element by element
    (3, 1, 1, 1, 14, (0, 14)),              # an axis without channels
    (2, 2, 1, 1, 512, (512,)),
    (1025, 1, 1, 1, 8, (4, 4)),
]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout", ["halves", "adjacent"])
@pytest.mark.parametrize("cfg", ROPE, ids=[str(c) for c in ROPE])
def test_rope_axes(K, cfg, layout, dtype):
    rows, heads, parts, rotated, dh, axes = cfg
    x = normal((rows, heads * parts * dh), dtype, seed=rows)
    g = torch.Generator().manual_seed(1)
    pos = torch.randint(-50, 1000, (rows, len(axes)), generator=g, dtype=torch.int32)
    plan = K.RopeAxes(dh, axes, theta=10000.0, layout=layout, device="cuda")
    for inverse in (False, True):
        y_ref, bound = R.rope(x, pos, heads, parts, rotated, dh, axes, 10000.0, layout, inverse)
        y = K.rope_axes(x.cuda(), pos.cuda(), plan, heads, parts=parts, rotated=rotated, inverse=inverse)
        R.within(y, y_ref, bound, "out of place")
        z = x.cuda()
        assert K.rope_axes(z, pos.cuda(), plan, heads, parts=parts, rotated=rotated, inverse=inverse, out=z) is z
        assert torch.equal(z, y)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_rope_positions_far_and_fractional(K, kind):
    """position types; a position of 2^30 + 1 is as exact as a small one (the whole turns are dropped in 64 bits)"""
    pos = torch.tensor([[0, 0], [1, -1], [900001, 123456789], [2 ** 30 + 1, 7]], dtype=torch.float64)
    pos = (torch.tensor([[0, 0.5], [1.25, -0.75], [900001.5, 16777215], [2 ** 24, 7.125]], dtype=torch.float32) if kind == torch.float32 else pos.to(kind))
    x = normal((4, 2 * 64), "fp32", seed=3)
    plan = K.RopeAxes(64, (32, 32), theta=500.0, device="cuda")
    y_ref, bound = R.rope(x, pos, 2, 1, 1, 64, (32, 32), 500.0, "halves", False)
    R.within(K.rope_axes(x.cuda(), pos.cuda(), plan, 2), y_ref, bound + 2e-7 * x.abs().max())    # (2^30 pos: 64-bit product and reference angle, 2^-22 each)


def test_rope_unaligned_rows_and_views(K):
    """a contiguous view that starts off a 16-byte boundary, leading dimensions, and zero rows"""
    base = normal((1 + 6 * 64,), "bf16", seed=5).cuda()
    x = base[1:].view(2, 3, 64)
    pos = torch.arange(6, dtype=torch.int64).view(6, 1).cuda()
    plan = K.RopeAxes(64, (64,), device="cuda")
    y_ref, bound = R.rope(x, pos, 1, 1, 1, 64, (64,), 10000.0, "halves", False)
    y = K.rope_axes(x, pos, plan, 1)
    assert y.shape == x.shape
    R.within(y, y_ref, bound)
    assert K.rope_axes(x[:0], pos[:0], plan, 1).shape == (0, 3, 64)


def test_rope_gradient_against_differences(K):
    """L = <dy, rope(x)> is linear in x: its differences in 64 bits are exact, the kernel's gradient is rope(dy, inverse=True)"""
    x, dy, v = (normal((6, 2 * 3 * 16), "fp32", seed=s) for s in (1, 2, 3))
    pos = torch.randint(0, 99, (6, 2), generator=torch.Generator().manual_seed(4))
    plan = K.RopeAxes(16, (8, 8), layout="adjacent", device="cuda")
    dx = K.rope_axes(dy.cuda(), pos.cuda(), plan, 2, parts=3, rotated=2, inverse=True).cpu().double()
    f = lambda z: float((R.rope(z, pos, 2, 3, 2, 16, (8, 8), 10000.0, "adjacent", False)[0] * dy.double()).sum())  # noqa: E731
    diff = (f(x.double() + v.double()) - f(x.double() - v.double())) / 2
    _, bound = R.rope(dy, pos, 2, 3, 2, 16, (8, 8), 10000.0, "adjacent", True)
    assert abs(float((dx * v.double()).sum()) - diff) <= float((bound * v.double().abs()).sum()) + 1e-9


def test_rope_nan_and_inf_stay_in_their_pairs(K):
    x = normal((4, 64), "fp32", seed=1)
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    plan = K.RopeAxes(64, (32, 32), device="cuda")
    y = K.rope_axes(x.cuda(), torch.ones(4, 2, dtype=torch.int32).cuda(), plan, 1).cpu()
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[1, [3, 35]] = True
    want[2, [5, 37]] = True
    assert torch.equal(bad, want)


def test_rope_refusals(K):
    plan = K.RopeAxes(32, (16, 16), device="cuda")
    x, pos = torch.zeros(4, 96, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    for bad in (dict(heads=2), dict(heads=1, parts=3, rotated=4), dict(heads=0, parts=3)):
        with pytest.raises(ValueError):
            K.rope_axes(x, pos, plan, **bad)
    for bad_pos in (pos[:3], pos[:, :1], pos.to(torch.float64), pos.cpu(), torch.zeros(2, 4, dtype=torch.int32, device="cuda").t()):
        with pytest.raises(ValueError):
            K.rope_axes(x, bad_pos, plan, 1, parts=3)
    with pytest.raises(ValueError, match="contiguous"):
        K.rope_axes(torch.zeros(96, 4, device="cuda").t(), pos, plan, 1, parts=3)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        K.rope_axes(x.double(), pos, plan, 1, parts=3)
    buf = torch.zeros(5 * 96, device="cuda")
    with pytest.raises(ValueError, match="shares no memory"):
        K.rope_axes(buf[:384].view(4, 96), pos, plan, 1, parts=3, out=buf[96:].view(4, 96))


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("count", [1, 3, 4, 7, 8, 1000, 4099])
@pytest.mark.parametrize("keep", [0.9, 0.5, 0.0, 1.0])
def test_dropout_apply(K, dtype, count, keep):
    x, skip = normal((count,), dtype, 1), normal((count,), dtype, 2)
    ctr = torch.tensor([0x123456789ABCDEF, 2 ** 32 - 3], dtype=torch.int64, device="cuda")      # (the position passes 32 bits)
    held = R.kept(0x123456789ABCDEF, 2 ** 32 - 3 + 11, count, keep)
    kf = float(torch.tensor(keep, dtype=torch.float32)) or 1.0
    for s in (None, skip):
        ref, bound = R.dropout(x, held, kf, s)
        y = K.dropout_apply(x.cuda(), keep, ctr, 11, skip=s.cuda() if s is not None else None)
        R.within(y, ref, bound)
        z = x.cuda()
        assert torch.equal(K.dropout_apply(z, keep, ctr, 11, skip=s.cuda() if s is not None else None, out=z), y)
    z = skip.cuda()
    assert torch.equal(K.dropout_apply(x.cuda(), keep, ctr, 11, skip=z, out=z), y)


@pytest.mark.parametrize("shape", [(160, 1280), (33, 7), (2, 3, 5)])
def test_dropout_equals_the_stored_mask(K, shape):
    """the running generator: dropout_fwd at a position gives x * dropout_mask's values at that position bit for bit, and both move it on by the same amount"""
    dev = torch.device("cuda", 0)
    x = normal(shape, "fp32", 3).cuda() + 0.25
    K.rng_counter(x.device, seed=77)
    m1, after = K.dropout_mask(shape, 0.8, x.device), K.dropout_mask((4,), 0.8, x.device)
    K.rng_counter(x.device, seed=77)
    y, draw = K.dropout_fwd(x, 0.8)
    assert torch.equal(K.dropout_mask((4,), 0.8, x.device), after)
    assert torch.equal(y, K.mul(x, m1)) or torch.equal(y + 0.0, K.mul(x, m1) + 0.0)
    assert torch.equal(K.dropout_bwd(torch.ones_like(x), draw), m1)
    assert dev.type == "cuda"


def test_dropout_drops_nan_and_inf(K):
    x = torch.full((64,), float("nan"), device="cuda")
    ctr = torch.tensor([5, 0], dtype=torch.int64, device="cuda")
    held = R.kept(5, 0, 64, 0.5)
    y = K.dropout_apply(x, 0.5, ctr, 0).cpu()
    assert torch.equal(torch.isnan(y), held) and (y[~held] == 0).all()


def test_dropout_unaligned_and_empty(K):
    base = normal((1 + 4096,), "fp16", 4).cuda()
    ctr = torch.tensor([9, 100], dtype=torch.int64, device="cuda")
    aligned = base[1:].clone()
    assert torch.equal(K.dropout_apply(base[1:], 0.7, ctr, 5), K.dropout_apply(aligned, 0.7, ctr, 5))
    assert K.dropout_apply(base[:0], 0.7, ctr, 5).numel() == 0


def test_dropout_graph_replays_draw_fresh_numbers(K):
    """forward and gradient of one captured step share their draw; dropout_advance gives the next replay another one"""
    x = torch.ones(4096, device="cuda")
    ctr = torch.tensor([21, 0], dtype=torch.int64, device="cuda")
    K.dropout_apply(x, 0.5, ctr, 0)
    K.dropout_advance(ctr, 0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = K.dropout_apply(x, 0.5, ctr, 3)
        dx = K.dropout_apply(x, 0.5, ctr, 3)
        K.dropout_advance(ctr, 1024)
    for replay in range(4):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dx)
        want = R.kept(21, 3 + 1024 * replay, 4096, 0.5)
        assert torch.equal(y.cpu() > 0, want), replay
        (x * 2).sum().item()                                           # eager work between the replays
    assert ctr.tolist() == [21, 4 * 1024]


def test_dropout_refusals(K):
    x = torch.zeros(64, device="cuda")
    ctr = torch.zeros(2, dtype=torch.int64, device="cuda")
    for bad in (dict(keep=1.5), dict(keep=-0.1), dict(keep=float("nan")), dict(position=-1), dict(counter=ctr.cpu()), dict(counter=ctr.int()), dict(skip=x[:3]),
                dict(skip=x.half()), dict(out=x.half())):
        args = dict(keep=0.5, counter=ctr, position=0)
        args.update(bad)
        with pytest.raises(ValueError):
            K.dropout_apply(x, **args)
    with pytest.raises(ValueError, match="shares no memory"):
        K.dropout_apply(x[:32], 0.5, ctr, 0, out=x[16:48])


# ------------------------------------------------------------------------------------------------ 16-bit LayerNorm
LN = [(1, 1), (1, 8), (3, 5), (4, 64), (17, 192), (33, 384), (5, 576), (2, 1357), (9, 2048), (300, 96), (1, 5000), (3, 4096), (70, 40), (129, 1001),
      (5000, 192), (2100, 33), (3000, 517), (1, 9), (7, 7), (50, 127), (40, 250), (20, 380), (20, 770), (3, 1537), (700, 2051), (3, 8192), (2, 8200), (600, 4099)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cfg", LN, ids=[str(c) for c in LN])
def test_layernorm16(K, cfg, dtype):
    rows, c = cfg
    x, dy, skip = normal((rows, c), dtype, 1, 1.5) + 0.5, normal((rows, c), dtype, 2), normal((rows, c), dtype, 3)
    gamma, beta = 1 + 0.2 * normal((c,), "fp32", 4), 0.3 * normal((c,), "fp32", 5)
    ref = R.layernorm(x, dy, 1e-5, gamma, beta)
    y, mean, rstd = K.layernorm_fwd(x.cuda(), c, 1e-5, gamma.cuda(), beta.cuda())
    R.within(y, *ref["y"], "y")
    dg, db = torch.full((c,), 7.0, device="cuda"), torch.full((c,), 7.0, device="cuda")
    dx = K.layernorm_bwd(x.cuda(), dy.cuda(), c, mean, rstd, gamma.cuda(), dg, db)
    R.within(dx, *ref["dx"], "dx")
    R.within(dg, *ref["dgamma"], "dgamma")
    R.within(db, *ref["dbeta"], "dbeta")
    dg2, db2 = dg.clone(), db.clone()
    dxs = K.layernorm_bwd(x.cuda(), dy.cuda(), c, mean, rstd, gamma.cuda(), dg2, db2, accumulate=True, skip=skip.cuda())
    assert torch.equal(dg2, dg + dg) and torch.equal(db2, db + db)     # (the sums of two calls on the same inputs are the same bits)
    R.within(dxs, *R.layernorm(x, dy, 1e-5, gamma, beta, skip=skip)["dx"], "dx + skip")
    y0, m0, r0 = K.layernorm_fwd(x.cuda(), c, 1e-5, None, None)
    plain = R.layernorm(x, dy, 1e-5, None, None)
    R.within(y0, *plain["y"], "no parameters")
    R.within(K.layernorm_bwd(x.cuda(), dy.cuda(), c, m0, r0, None), *plain["dx"], "dx without parameters")


def test_layernorm16_constant_and_offset_rows(K):
    """a constant row normalises to beta (variance exactly 0); rows far from zero keep their statistics"""
    x = torch.full((3, 256), 100.0).to(torch.bfloat16)
    beta = normal((256,), "fp32", 1)
    y, _, rstd = K.layernorm_fwd(x.cuda(), 256, 1e-5, torch.ones(256, device="cuda"), beta.cuda())
    assert torch.equal(y.cpu(), beta.to(torch.bfloat16).expand(3, 256))
    x = (normal((5, 768), "fp32", 2) + 200).to(torch.float16)
    ref = R.layernorm(x, torch.zeros_like(x), 1e-5, None, None)
    R.within(K.layernorm_fwd(x.cuda(), 768, 1e-5, None, None)[0], *ref["y"])


def test_layernorm16_rows_do_not_touch_each_other(K):
    """a NaN row stays one row; rows behind the last one are left as they were; a view that starts off a 16-byte boundary; no rows at all"""
    x = normal((6, 192), "bf16", 1)
    x[2, 5] = float("nan")
    y, mean, rstd = K.layernorm_fwd(x.cuda(), 192, 1e-5, None, None)
    nan = torch.isnan(y.cpu()).all(1)
    assert torch.equal(nan, torch.tensor([i == 2 for i in range(6)]))
    base = normal((1 + 6 * 192,), "bf16", 2).cuda()
    off = base[1:].view(6, 192)
    assert torch.equal(K.layernorm_fwd(off, 192, 1e-5, None, None)[0], K.layernorm_fwd(off.clone(), 192, 1e-5, None, None)[0])
    dg = torch.full((192,), 3.0, device="cuda")
    e = off[:0]
    ye, me, re = K.layernorm_fwd(e, 192, 1e-5, None, None)
    assert ye.shape == (0, 192)
    K.layernorm_bwd(e, e, 192, me, re, None, dg, None)
    assert (dg == 0).all()


def test_layernorm16_gradient_against_differences(K):
    x, dy, v = (normal((4, 24), "fp32", s).to(torch.bfloat16) for s in (1, 2, 3))
    gamma = 1 + 0.2 * normal((24,), "fp32", 4)
    f = lambda z: float((torch.nn.functional.layer_norm(z, (24,), gamma.double(), None, 1e-5) * dy.double()).sum())  # noqa: E731
    e = 1e-5
    diff = (f(x.double() + e * v.double()) - f(x.double() - e * v.double())) / (2 * e)
    _, mean, rstd = K.layernorm_fwd(x.cuda(), 24, 1e-5, gamma.cuda(), None)
    dx = K.layernorm_bwd(x.cuda(), dy.cuda(), 24, mean, rstd, gamma.cuda()).cpu().double()
    bound = R.layernorm(x, dy, 1e-5, gamma, None)["dx"][1]
    assert abs(float((dx * v.double()).sum()) - diff) <= float((bound * v.double().abs()).sum()) + 1e-6 * abs(diff) + 1e-7


def test_layernorm16_refusals(K):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    g = torch.ones(64, device="cuda")
    with pytest.raises(ValueError):
        K.layernorm_fwd(x, 64, 1e-5, g.half(), None)
    with pytest.raises(ValueError):
        K.layernorm_fwd(x, 32, 1e-5, g[:32], None)
    with pytest.raises(ValueError):
        K.layernorm_fwd(x.t(), 4, 1e-5, None, None)
    y, m, r = K.layernorm_fwd(x, 64, 1e-5, g, None)
    for bad in (dict(dy=x.half()), dict(dy=x[:2]), dict(mean=m[:2]), dict(dgamma=g.bfloat16()), dict(skip=x[:1])):
        args = dict(x=x, dy=x, c=64, mean=m, rstd=r, gamma=g)
        args.update(bad)
        with pytest.raises(ValueError):
            K.layernorm_bwd(**args)
