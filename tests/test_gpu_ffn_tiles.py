"""The feed-forward block's products in every form that the tile choice (plan_gemm in csrc/gemm_lowp.inl) reaches: small tiles with two and with four buffers and large
ones, reduced whole, split along the reduction, or some of each -- the sizes below add to tests/test_gpu_gated_ffn.py those that no size there takes, by type and product."""
import pytest
import torch

import token_ops_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from semiuhpe_amd import kernels
    return kernels


def normal(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).to(R.TYPES[dtype])


FORMS = {
    # m, k, n, o: which products take which form there
    "fp32": [(12307, 136, 2456, 136),                       # large tiles for all; y, dx and the weights' gradients split
             (2351, 2728, 1216, 960), (2153, 4000, 1048, 4000),      # small: some whole, some split (dw, dx, y); dw large and whole
             (25484, 472, 32, 416), (654, 680, 9216, 680),  # dx, y large and whole; dw large, mixed
             (27965, 648, 344, 56), (21316, 48, 680, 1008)],         # dx, y large, mixed
    "bf16": [(11391, 40, 5872, 40), (8264, 144, 5816, 144),
             (2374, 40, 9752, 840), (32909, 152, 1560, 152),
             (1636, 3640, 664, 3640), (17052, 40, 6136, 144),
             (16754, 952, 608, 952), (4853, 80, 2568, 3336)],
    "fp16": [(12155, 40, 6312, 40), (25484, 472, 32, 416), (8264, 144, 5816, 144),
             (2374, 40, 9752, 840), (32909, 152, 1560, 152),
             (1636, 3640, 664, 3640), (979, 480, 10968, 480), (17052, 40, 6136, 144),
             (16754, 952, 608, 952), (4853, 80, 2568, 3336)],
}


@pytest.mark.parametrize("dtype,cfg", [(t, c) for t, cs in FORMS.items() for c in cs], ids=str)
def test_every_form_of_the_products(K, dtype, cfg):
    m, k, n, o = cfg
    x, dy = normal((m, k), dtype, 1), normal((m, o), dtype, 9)
    w = [normal((n, k), dtype, 2, k ** -0.5), normal((n, k), dtype, 3, k ** -0.5), normal((o, n), dtype, 4, n ** -0.5)]
    b = [normal((c,), dtype, 5 + i, 0.3) for i, c in enumerate((n, n, o))]
    y, saved = K.gated_ffn_fwd(x, *w, *b, act="silu")
    grads = [torch.full_like(t, float("nan")) for t in w + b]
    dx = K.gated_ffn_bwd(dy, x, *w, saved, "silu", *grads)
    got = dict(zip(("y", "dx", "dwg", "dwu", "dwd", "dbg", "dbu", "dbd"), [y, dx] + grads))
    for key, (value, bound) in R.gated_ffn(x, *w, *b, dy, "silu", device="cuda").items():
        R.within(got[key], value, bound, key)
    again = [torch.empty_like(t) for t in grads]
    y2, saved2 = K.gated_ffn_fwd(x, *w, *b, act="silu")
    assert torch.equal(K.gated_ffn_bwd(dy, x, *w, saved2, "silu", *again), dx) and torch.equal(y2, y)
    assert all(torch.equal(p, q) for p, q in zip(again, grads))         # the same bits from call to call


@pytest.mark.parametrize("m,k,n", [(70, 1, 1), (64, 3, 2), (300, 40, 24), (1000, 264, 520)])
def test_fp32_keeps_both_projections_whole(K, m, k, n):
    """What the backward gets in fp32 is g and u as they were summed (16-bit types: cut to 24 bits, off by up to 2^-15)"""
    x, w = normal((m, k), "fp32", 1), [normal((n, k), "fp32", 2), normal((n, k), "fp32", 3), normal((2, n), "fp32", 4)]
    b = [normal((n,), "fp32", 5), normal((n,), "fp32", 6)]
    _, (kept, _) = K.gated_ffn_fwd(x, *w, *b)
    g, u = kept.view(torch.float32).view(2, m, n)
    for got, weight, bias in ((g, w[0], b[0]), (u, w[1], b[1])):
        want = x.double() @ weight.double().t() + bias.double()
        bound = (k + 2) * 2.0 ** -24 * (x.double().abs() @ weight.double().abs().t() + bias.double().abs())
        R.within(got, want, bound, "kept")


@pytest.mark.parametrize("m,k,n,o", [(512, 1, 1, 1), (600, 3, 2, 3)])
def test_fp32_gradients_are_not_off_by_24_bits(K, m, k, n, o):
    """sums of a few terms: every gradient within a few fp32 roundings of the terms' absolute sum, where projections of 24 bits would be off by up to 2^-15 = 512 of them"""
    x, dy = normal((m, k), "fp32", 1), normal((m, o), "fp32", 9)
    w = [normal((n, k), "fp32", 2), normal((n, k), "fp32", 3), normal((o, n), "fp32", 4)]
    _, saved = K.gated_ffn_fwd(x, *w, act="none")           # (act none: dg = dh u, du = dh g)
    dx = K.gated_ffn_bwd(dy, x, *w, saved, "none")
    X, G, W, D, Y = (t.double() for t in (x, *w, dy))

    def terms(f):
        X_, G_, W_, D_, Y_ = (f(t) for t in (X, G, W, D, Y))
        dh = Y_ @ D_
        return (dh * (X_ @ W_.t())) @ G_ + (dh * (X_ @ G_.t())) @ W_
    # dh: o roundings, a projection: k, their product and dg's: 2, the sum over 2 n terms: 2 n; twice 2 for second-order terms and the bias of zero
    rounds = o + k + 2 + 2 * n + 4
    R.within(dx, terms(lambda t: t), rounds * 2.0 ** -24 * terms(torch.abs), "dx")
