"""The feed-forward block's few-row (serving) form: operands at any address, against the 64-bit form (tests/token_ops_ref.py)."""
import pytest
import torch

import token_ops_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from semiuhpe_amd import kernels
    return kernels


def normal(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(R.TYPES[dtype])


def shifted(t, by):
    """the tensor `by` elements into a buffer of NaN on the device"""
    buf = torch.full((t.numel() + 32,), float("nan"), dtype=t.dtype, device="cuda")
    out = buf[by:by + t.numel()].view(t.shape)
    out.copy_(t)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m", [1, 3, 16])
@pytest.mark.parametrize("k,n,o", [(8, 8, 8), (8, 8, 3), (8, 21, 5), (9, 8, 8), (16, 24, 8)])
def test_operands_off_every_boundary(K, dtype, m, k, n, o):
    """rows of one chunk and more, every operand one element into a buffer (nothing before or behind a row is taken into it)"""
    from semiuhpe_amd import _lib
    x, wg, wu, wd = normal((m, k), dtype, 1), normal((n, k), dtype, 2, k ** -0.5), normal((n, k), dtype, 3, k ** -0.5), normal((o, n), dtype, 4, n ** -0.5)
    dx, dg, du, dd = (shifted(t, 1) for t in (x, wg, wu, wd))
    h, y = torch.empty((m, n), dtype=x.dtype, device="cuda"), torch.empty((m, o), dtype=x.dtype, device="cuda")
    code = K._DTYPES[x.dtype]
    need = _lib.load().suhpe_gated_ffn_fwd_workspace_bytes(code, m, k, n, o)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    _lib.call("suhpe_gated_ffn_fwd", code, K.ACT["silu"], m, k, n, o, dx.data_ptr(), dg.data_ptr(), du.data_ptr(), dd.data_ptr(), None, None, None, None,
              h.data_ptr(), y.data_ptr(), ws.data_ptr() if need else None, need)
    ref = R.gated_ffn(x, wg, wu, wd, None, None, None, torch.zeros((m, o), dtype=x.dtype), "silu")
    R.within(y, *ref["y"], "y")


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,k,n,o,copies", [(1, 128, 136, 64, 0), (32, 72, 40, 9, 0), (2, 33, 57, 33, 0), (40, 64, 72, 24, 4), (40, 33, 57, 19, 0), (3, 2, 8, 8, 1), (40, 64, 33, 24, 3)])
def test_operands_are_copied_only_where_the_kernel_asks(K, monkeypatch, dtype, m, k, n, o, copies):
    """views into a larger buffer: none is copied for few rows (of 16 bytes and more: with k = 2 the tile kernel runs, and wd is copied), nor where the rows are copied to padded ones anyway; the same bits as with operands of their own"""
    x, wg, wu, wd = normal((m, k), dtype, 1), normal((n, k), dtype, 2, k ** -0.5), normal((n, k), dtype, 3, k ** -0.5), normal((o, n), dtype, 4, n ** -0.5)
    want, _ = K.gated_ffn_fwd(*(t.cuda() for t in (x, wg, wu, wd)), save=False)
    views = [shifted(t, 1) for t in (x, wg, wu, wd)]
    made = []
    clone = torch.Tensor.clone
    monkeypatch.setattr(torch.Tensor, "clone", lambda t, *a, **kw: made.append(t) or clone(t, *a, **kw))
    y, _ = K.gated_ffn_fwd(*views, save=False)
    monkeypatch.undo()
    assert len(made) == copies
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m", [1, 3, 7, 13, 16])
@pytest.mark.parametrize("k,n,o", [(64, 512, 96), (33, 517, 37), (64, 516, 24), (8, 8, 9), (40, 9, 40), (16, 15, 8)])
@pytest.mark.parametrize("save", [True, False])
def test_h_keeps_more_than_its_type_between_the_products(K, dtype, m, k, n, o, save):
    """Up to 16 rows y is not off by h's rounding (2^-8 or 2^-11 of every term): of a term, the two parts of h leave out half a step of half a step, 2^-16 (bf16) or
    2^-22 (fp16, 2^-25 where the second part is below fp16's normal numbers); then fp32 sums, and one rounding of y"""
    x, wg, wu, wd = normal((m, k), dtype, 1), normal((n, k), dtype, 2, k ** -0.5), normal((n, k), dtype, 3, k ** -0.5), normal((o, n), dtype, 4, n ** -0.5)
    bg, bu, bd = normal((n,), dtype, 5, 0.3), normal((n,), dtype, 6, 0.3), normal((o,), dtype, 7, 0.3)
    y, _ = K.gated_ffn_fwd(*(t.cuda() for t in (x, wg, wu, wd, bg, bu, bd)), save=save)
    U, r = 2.0 ** -24, R.half(x.dtype) * 1.001
    X, G, W, D = x.double(), wg.double(), wu.double(), wd.double()
    g, u = X @ G.t() + bg.double(), X @ W.t() + bu.double()
    a, _, d1, _ = R.act(g, "silu")
    h = a * u
    e_g, e_u = ((k + 2) * U * (X.abs() @ w.abs().t() + b.double().abs()) for w, b in ((G, bg), (W, bu)))
    e_a = d1 * e_g + (2e-7 + 8 * U) * (1 + g.abs())
    e_h = e_a * u.abs() + a.abs() * e_u + e_a * e_u + U * h.abs()
    left = R.half(x.dtype) ** 2 * 1.01
    e_h = e_h + left * (h.abs() + e_h) + (2.0 ** -25 if dtype == "fp16" else 0.0)
    want = h @ D.t() + bd.double()
    bound = e_h @ D.abs().t() + (2 * n + 2) * U * ((h.abs() + e_h) @ D.abs().t() + bd.double().abs())
    bound = bound + r * (want.abs() + bound) + (2.0 ** -25 if dtype == "fp16" else 0.0)
    R.within(y, want, bound, "y")


def test_h_beyond_fp16_is_an_infinity_for_few_rows_too(K):
    one = torch.ones((1, 8), dtype=torch.float16, device="cuda")
    w = torch.full((8, 8), 40.0, dtype=torch.float16, device="cuda")    # g = u = 320, h = 102 400
    down = torch.eye(8, dtype=torch.float16, device="cuda")[:2] + 0.5
    y, _ = K.gated_ffn_fwd(one, w, w, down, act="none", save=False)
    assert torch.isinf(y).all() and (y > 0).all()
    w[0, 0] = float("nan")
    y, _ = K.gated_ffn_fwd(one, w, w, down, act="none", save=False)
    assert torch.isnan(y).all()
