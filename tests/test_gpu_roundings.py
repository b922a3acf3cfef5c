"""The last bit of kernels whose roundings are written out (csrc/common.h: add_product and its neighbours): which products are fused into a sum must not hang on
the instructions that the compiler has.  Results are compared bit for bit with the same roundings on the CPU; a fused multiply-add is a product and a sum in 64
bits of mantissa, rounded once."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from semiuhpe_amd import kernels
    return kernels


def fma(a, b, c):
    return (a.astype(np.longdouble) * b.astype(np.longdouble) + c.astype(np.longdouble)).astype(np.float32)


def _rand(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def test_ema_and_adam_round_every_product(K):
    e, p, g, m, v = (_rand(i, 5003) for i in range(5))
    v = np.abs(v)
    for alpha in (0.999, 0.75):
        out = _dev(e)
        K.ema_update(out, _dev(p), alpha)
        al = np.float32(alpha)
        want = e * al + (np.float32(1) - al) * p
        assert np.array_equal(out.cpu().numpy(), want)
    pt, mt, vt = _dev(p), _dev(m), _dev(v)
    K.adam_step(pt, _dev(g), mt, vt, 1e-3, 0.9, 0.999, 1e-8, 0.0, 3)
    b1, b2, one = np.float32(0.9), np.float32(0.999), np.float32(1)
    assert np.array_equal(mt.cpu().numpy(), b1 * m + (one - b1) * g)
    assert np.array_equal(vt.cpu().numpy(), b2 * v + (one - b2) * g * g)


def test_add_rowscale_is_one_fused_sum(K):
    a, b, s = _rand(1, 7, 5, 5, 24), _rand(2, 7, 5, 5, 24), _rand(3, 7)
    got = K.add_rowscale(_dev(a), _dev(b), _dev(s)).cpu().numpy()
    assert np.array_equal(got, fma(b, np.broadcast_to(s[:, None, None, None], b.shape), a))


@pytest.mark.parametrize("mode", [0, 1])
def test_rotation_adjustment(K, mode):
    A, G = _rand(10 + mode, 3001, 9), _rand(20 + mode, 3001, 9)
    got = K.rot_adjust(_dev(A), _dev(G), mode).cpu().numpy()
    second, plain = ((0x023, 0x100), (0x0b5, 0x145))[mode]
    sign = np.array([1, -1, -1], np.float32)
    M = (sign[:, None] * sign[None, :]).reshape(9) * G
    for i in range(3):
        for j in range(3):
            k = 3 * i + j
            if mode == 0:
                f = [(G[:, 3 * i + q], A[:, 3 * q + j]) for q in range(3)]
            else:
                f = [(A[:, 3 * i + q], M[:, 3 * j + q]) for q in range(3)]
            lo, hi = (f[0], f[1]) if second >> k & 1 else (f[1], f[0])
            t = fma(hi[0], hi[1], lo[0] * lo[1])
            want = t + f[2][0] * f[2][1] if plain >> k & 1 else fma(f[2][0], f[2][1], t)
            assert np.array_equal(got[:, k], want), (i, j)


def test_strided_depthwise_conv_with_statistics(K):
    """3 x 3, stride 2 (one output row a thread): with statistics, taps 2, 3, 6, 7 and 8 of every column but the first keep both roundings"""
    n, h, c = 2, 20, 24
    x, w = _rand(30, n, h, h, c), _rand(31, c, 3, 3)
    wt = K.to_filter_layout(_dev(w.reshape(c, 1, 3, 3)))
    y = K.dwconv_fwd_stats(_dev(x), wt, 2, 1)[0].cpu().numpy()
    xp = np.zeros((n, h + 2, h + 2, c), np.float32)
    xp[:, 1:-1, 1:-1] = x
    want = np.zeros_like(y)
    for ow in range(y.shape[2]):
        acc = np.zeros_like(y[:, :, 0])
        for tap in range(9):
            r, q = divmod(tap, 3)
            rows = xp[:, r:r + 2 * y.shape[1]:2, 2 * ow + q]
            f = np.broadcast_to(w[:, r, q], rows.shape)
            acc = acc + rows * f if ow > 0 and 0x1cc >> tap & 1 else fma(rows, f, acc)
        want[:, :, ow] = acc
    assert np.array_equal(y, want)


@pytest.mark.parametrize("rows", [7, 300])
def test_layernorm_gradient_of_short_rows(K, rows):
    """s1 = sum of dy xhat keeps both roundings: one lane holds the row (c = 4), so the order of the sum is known"""
    c = 4
    x, dy = _rand(40, rows, c), _rand(41, rows, c)
    mean, rstd = x.mean(1, dtype=np.float32), (np.float32(1) / np.sqrt(x.var(1) + np.float32(1e-5))).astype(np.float32)
    gamma = np.ones(c, np.float32)
    got = K.layernorm_bwd(_dev(x), _dev(dy), c, _dev(mean), _dev(rstd), _dev(gamma)).cpu().numpy()
    xh = (x - mean[:, None]) * rstd[:, None]
    s0, s1 = np.zeros(rows, np.float32), np.zeros(rows, np.float32)
    for e in range(c):
        s0 = s0 + dy[:, e]
        s1 = s1 + dy[:, e] * xh[:, e]
    s0, s1 = s0 / np.float32(c), s1 / np.float32(c)
    want = fma(np.broadcast_to(rstd[:, None], x.shape), fma(-xh, np.broadcast_to(s1[:, None], x.shape), dy - s0[:, None]), np.zeros_like(x))
    assert np.array_equal(got, want)
