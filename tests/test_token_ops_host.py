"""Refusals of the transformer-block operators that the C ABI decides on the host, and the plans' checks: nothing is launched, no GPU needed."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(1 << 20)                                           # 16-byte aligned, never dereferenced
F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    from semiuhpe_amd import _lib
    return _lib.load()


def test_rope_axes_refusals(lib):
    def rope(dtype=F32, rows=4, heads=2, parts=3, rotated=2, dh=32, pos_type=0, naxes=2, pairs=16, x=P):
        return lib.suhpe_rope_axes(x, dtype, rows, heads, parts, rotated, dh, P, pos_type, naxes, P, P, pairs, 1, 0, P, None)
    for bad in (dict(dtype=3), dict(rows=-1), dict(heads=0), dict(rotated=0), dict(rotated=4), dict(dh=1), dict(pos_type=3), dict(pos_type=-1), dict(naxes=0), dict(pairs=0),
                dict(pairs=17), dict(dh=20000, pairs=5000), dict(heads=1 << 20, dh=64), dict(x=None)):
        assert rope(**bad) == -1, bad
        assert b"suhpe_rope_axes" in lib.suhpe_last_error()
    assert rope(rows=0) == 0                                           # no rows: nothing to do


def test_dropout_refusals(lib):
    def drop(dtype=F32, count=16, keep=0.5, counter=P):
        return lib.suhpe_dropout_apply(P, dtype, count, ctypes.c_float(keep), counter, 0, None, P, None)
    for bad in (dict(dtype=7), dict(count=-1), dict(keep=1.01), dict(keep=-0.5), dict(keep=float("nan")), dict(counter=None)):
        assert drop(**bad) == -1, bad
        assert b"suhpe_dropout_apply" in lib.suhpe_last_error()
    assert drop(count=0) == 0
    assert lib.suhpe_dropout_advance(None, 4, None) == -1


def test_layernorm16_refusals(lib):
    assert lib.suhpe_layernorm16_fwd(P, F32, 4, 64, ctypes.c_float(1e-5), None, None, P, P, P, None) == -1
    assert lib.suhpe_layernorm16_fwd(P, BF16, -1, 64, ctypes.c_float(1e-5), None, None, P, P, P, None) == -1
    assert lib.suhpe_layernorm16_fwd(P, BF16, 4, 0, ctypes.c_float(1e-5), None, None, P, P, P, None) == -1
    assert lib.suhpe_layernorm16_fwd(P, BF16, 0, 64, ctypes.c_float(1e-5), None, None, P, P, P, None) == 0
    need = lib.suhpe_layernorm16_bwd_workspace_bytes(64)
    assert need > 0
    assert lib.suhpe_layernorm16_bwd(P, P, BF16, 4, 64, P, P, None, None, P, P, P, 0, P, need - 1, None) == -3
    assert lib.suhpe_layernorm16_bwd(P, P, BF16, 4, 64, P, P, None, None, P, P, P, 0, None, need, None) == -1
    assert lib.suhpe_layernorm16_bwd(P, None, BF16, 4, 64, P, P, None, None, P, P, P, 0, P, need, None) == -1


def test_gated_ffn_refusals(lib):
    def fwd(dtype=BF16, act=3, m=8, k=16, n=24, o=16, x=P, h=P):
        ws = max(1, lib.suhpe_gated_ffn_fwd_workspace_bytes(max(0, min(2, dtype)), 8, 16, 24, 16))
        return lib.suhpe_gated_ffn_fwd(dtype, act, m, k, n, o, x, P, P, P, None, None, None, P, h, P, P, ws, None)
    for bad in (dict(dtype=5), dict(act=9), dict(act=-1), dict(m=-1), dict(k=0), dict(n=-4), dict(o=0), dict(k=1 << 21), dict(x=None), dict(h=None)):
        assert fwd(**bad) == -1, bad
        assert b"suhpe_gated_ffn_fwd" in lib.suhpe_last_error()
    assert fwd(m=0) == 0
    assert lib.suhpe_gated_ffn_kept_bytes(F32, 10, 7) == 560 and lib.suhpe_gated_ffn_kept_bytes(BF16, 10, 7) == 420 and lib.suhpe_gated_ffn_kept_bytes(4, 10, 7) == -1
    need = lib.suhpe_gated_ffn_bwd_workspace_bytes(BF16, 8, 16, 24, 16)
    assert need > 0

    def bwd(grad=BF16, dy=P, dwg=P, dwu=P, dwd=P, nbytes=need, ws=P):
        return lib.suhpe_gated_ffn_bwd(BF16, 3, 8, 16, 24, 16, dy, P, P, P, P, P, P, P, dwg, dwu, dwd, None, None, None, grad, 0, ws, nbytes, None)
    for bad in (dict(grad=F16), dict(grad=4), dict(dy=None), dict(dwg=None), dict(dwd=None)):
        assert bwd(**bad) == -1, bad
        assert b"suhpe_gated_ffn_bwd" in lib.suhpe_last_error()
    assert lib.suhpe_gated_ffn_bwd(BF16, 3, 0, 16, 24, 16, None, None, None, None, None, None, None, None, None, None, None, None, None, None, BF16, 0, None, 0, None) == 0
    assert lib.suhpe_gated_ffn_bwd_workspace_bytes(BF16, 0, 16, 24, 16) == 0
    assert bwd(nbytes=need - 1) == -3
    assert bwd(ws=None) == -3


def test_rope_plan():
    from semiuhpe_amd import kernels as K
    plan = K.RopeAxes(32, (16, 8), device="cpu")
    assert plan.pairs == 12 and plan.axis.tolist() == [0] * 8 + [1] * 4
    assert float(plan.freq[0]) * 2 * 3.141592653589793 == pytest.approx(1.0, rel=1e-15)
    assert float(plan.freq[9]) * 2 * 3.141592653589793 == pytest.approx(10000.0 ** -0.25, rel=1e-14)
    for axes in ((), (7, 9), (16, 18), (-2, 8), (0,)):
        with pytest.raises(ValueError):
            K.RopeAxes(32, axes, device="cpu")
    with pytest.raises(ValueError):
        K.RopeAxes(32, (16, 16), layout="split", device="cpu")
    with pytest.raises(ValueError):
        K.RopeAxes(32, (16, 16), theta=0.0, device="cpu")


def test_no_cpu_path():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    from semiuhpe_amd import kernels as K
    x = torch.zeros(4, 32)
    plan = K.RopeAxes(32, (32,), device="cpu")
    w = torch.zeros(8, 32)
    for call in (lambda: K.rope_axes(x, torch.zeros(4, 1, dtype=torch.int32), plan, 1), lambda: K.dropout_apply(x, 0.5, torch.zeros(2, dtype=torch.int64), 0),
                 lambda: K.layernorm_fwd(x.bfloat16(), 32, 1e-5, None, None), lambda: K.gated_ffn_fwd(x, w, w, torch.zeros(4, 8))):
        with pytest.raises(RuntimeError, match="no CPU|no HIP"):
            call()


def test_generator_in_integers():
    """the oracle's Philox4x32-10 keeps about keep of the elements and is a function of (seed, position) alone"""
    import token_ops_ref as R
    a = R.kept(1234, 10, 4000, 0.75)
    assert torch.equal(a[8:], R.kept(1234, 12, 3992, 0.75))
    assert abs(float(a.float().mean()) - 0.75) < 5 * (0.75 * 0.25 / 4000) ** 0.5


def test_outputs_that_share_memory(lib):
    """one buffer for two gradients, or a gradient over an input, is refused before anything runs: the products of a launch write side by side"""
    need = lib.suhpe_gated_ffn_bwd_workspace_bytes(BF16, 8, 16, 24, 16)
    # 8 x 16, 24 x 16 and 16 x 24 of 2 bytes fit 768 bytes; kept: 8 * 24 * 6 bytes
    place = {name: 0x100000 + 0x1000 * i for i, name in enumerate(("dy", "x", "wg", "wu", "wd", "kept", "h", "dx", "dwg", "dwu", "dwd", "dbg", "dbu", "dbd"))}

    def bwd(**moved):
        at = dict(place, **moved)
        return lib.suhpe_gated_ffn_bwd(BF16, 3, 8, 16, 24, 16, *(ctypes.c_void_p(p) for p in at.values()), BF16, 0, P, need, None)
    for bad in (dict(dwu=place["dwg"]), dict(dwd=place["dwg"] + 766), dict(dbu=place["dbg"] + 46), dict(dx=place["x"]), dict(dx=place["dy"]), dict(dwg=place["wg"]),
                dict(dwd=place["h"]), dict(dbd=place["kept"] + 8 * 24 * 6 - 2)):
        assert bwd(**bad) == -1, bad
        assert b"share no memory" in lib.suhpe_last_error()
    need = lib.suhpe_layernorm16_bwd_workspace_bytes(64)
    a, b = ctypes.c_void_p(0x100000), ctypes.c_void_p(0x100000 + 252)
    for dg, db in ((a, a), (a, b), (b, a)):
        assert lib.suhpe_layernorm16_bwd(P, P, BF16, 4, 64, P, P, None, None, P, dg, db, 0, P, need, None) == -1
        assert b"share no memory" in lib.suhpe_last_error()
