"""What the C entry points of the transformer-block operators refuse about memory: decided on the host, nothing is launched."""
import ctypes

import pytest

BF16 = 1
AT = 1 << 30


def P(offset=0):
    return ctypes.c_void_p(AT + offset)


@pytest.fixture(scope="module")
def lib():
    from semiuhpe_amd import _lib
    return _lib.load()


ROWS, C = 100, 60                                           # 12 000 bytes a tensor of rows, 240 a parameter
PLACES = dict(x=0, dy=1 << 16, dx=2 << 16, skip=3 << 16, mean=4 << 16, rstd=5 << 16, gamma=6 << 16, dgamma=7 << 16, dbeta=8 << 16, ws=1 << 24)


def backward(lib, **moved):
    at = {k: P(moved.get(k, v)) for k, v in PLACES.items()}
    need = lib.suhpe_layernorm16_bwd_workspace_bytes(C)
    return lib.suhpe_layernorm16_bwd(at["x"], at["dy"], BF16, ROWS, C, at["mean"], at["rstd"], at["gamma"], at["skip"], at["dx"], at["dgamma"], at["dbeta"], 0, at["ws"], need, None)


@pytest.mark.parametrize("moved", [dict(dx=PLACES["x"]), dict(dx=PLACES["dy"]), dict(dx=PLACES["skip"]), dict(dx=PLACES["skip"] + 11998), dict(dx=PLACES["dy"] - 11998),
                                   dict(dgamma=PLACES["gamma"]), dict(dgamma=PLACES["dbeta"] - 236), dict(dbeta=PLACES["x"] + 4), dict(dgamma=PLACES["mean"] + 396),
                                   dict(dx=PLACES["rstd"]), dict(ws=PLACES["dx"]), dict(ws=PLACES["gamma"] - 1024), dict(dgamma=PLACES["ws"] + 64)])
def test_layernorm16_backward_refuses_shared_memory(lib, moved):
    assert backward(lib, **moved) == -1, moved
    assert b"suhpe_layernorm16_bwd" in lib.suhpe_last_error() and b"share no memory" in lib.suhpe_last_error()


@pytest.mark.parametrize("moved", [dict(y=2), dict(y=-11998), dict(mean=PLACES["x"]), dict(rstd=PLACES["mean"] + 396), dict(mean=PLACES["gamma"] - 396), dict(y=PLACES["rstd"])])
def test_layernorm16_forward_refuses_shared_memory(lib, moved):
    at = {k: P(moved.get(k, v)) for k, v in dict(PLACES, y=2 << 16, beta=9 << 16).items()}
    assert lib.suhpe_layernorm16_fwd(at["x"], BF16, ROWS, C, ctypes.c_float(1e-5), at["gamma"], at["beta"], at["y"], at["mean"], at["rstd"], None) == -1, moved
    assert b"share no memory" in lib.suhpe_last_error()


def test_rope_axes_refuses_more_than_one_launch_holds(lib):
    """2^31 - 1 rows of 64 fp32 elements: 64 rows a workgroup of 256 threads would be 2^33 threads"""
    assert lib.suhpe_rope_axes(P(), 0, (1 << 31) - 1, 1, 1, 1, 64, P(1 << 20), 0, 1, P(2 << 20), P(3 << 20), 32, 1, 0, P(), None) == -1
    assert b"one launch" in lib.suhpe_last_error()


ROPE = dict(x=0, y=1 << 16, pos=2 << 16, freq=3 << 16, axis=4 << 16)      # 50 rows of 2 x 3 x 8 bf16: 4 800 bytes, positions 400, 3 pairs


@pytest.mark.parametrize("moved", [dict(y=2), dict(y=-4798), dict(y=ROPE["pos"] + 398), dict(y=ROPE["freq"] - 4798), dict(y=ROPE["axis"] + 10)])
def test_rope_axes_refuses_shared_memory(lib, moved):
    at = {k: P(moved.get(k, v)) for k, v in ROPE.items()}
    assert lib.suhpe_rope_axes(at["x"], BF16, 50, 2, 3, 2, 8, at["pos"], 0, 2, at["freq"], at["axis"], 3, 1, 0, at["y"], None) == -1, moved
    assert b"suhpe_rope_axes" in lib.suhpe_last_error() and b"shares no memory" in lib.suhpe_last_error()


@pytest.mark.parametrize("moved", [dict(y=4), dict(y=-198), dict(y=(1 << 16) + 2), dict(y=(1 << 16) - 198), dict(y=(3 << 16) + 14)])
def test_dropout_apply_refuses_shared_memory(lib, moved):
    at = {k: P(moved.get(k, v)) for k, v in dict(x=0, skip=1 << 16, y=2 << 16, counter=3 << 16).items()}
    assert lib.suhpe_dropout_apply(at["x"], BF16, 100, ctypes.c_float(0.5), at["counter"], 0, at["skip"], at["y"], None) == -1, moved
    assert b"suhpe_dropout_apply" in lib.suhpe_last_error() and b"shares no memory" in lib.suhpe_last_error()


FFN = dict(x=0, wg=1 << 20, wu=2 << 20, wd=3 << 20, bg=4 << 20, bu=5 << 20, bd=6 << 20, kept=7 << 20, h=8 << 20, y=9 << 20, ws=10 << 20)


@pytest.mark.parametrize("m", [4, 40])
@pytest.mark.parametrize("moved", [dict(h=FFN["x"]), dict(h=FFN["wd"] + 16), dict(h=FFN["bu"]), dict(kept=FFN["h"] + 16), dict(kept=FFN["wg"]), dict(y=FFN["h"]), dict(y=FFN["wd"]),
                                   dict(y=FFN["bd"] + 30), dict(y=FFN["kept"] + 16), dict(ws=FFN["x"]), dict(ws=FFN["y"]), dict(ws=FFN["h"])])
def test_gated_ffn_forward_refuses_shared_memory(lib, m, moved):
    """k = 36 and n = 44 are no whole 16-byte pieces: both forms, few rows and tiles, have a workspace"""
    at = {k: P(moved.get(k, v)) for k, v in FFN.items()}
    need = lib.suhpe_gated_ffn_fwd_workspace_bytes(BF16, m, 36, 44, 16)
    assert need > 0
    assert lib.suhpe_gated_ffn_fwd(BF16, 3, m, 36, 44, 16, *(at[k] for k in ("x", "wg", "wu", "wd", "bg", "bu", "bd", "kept", "h", "y", "ws")), need, None) == -1, moved
    assert b"suhpe_gated_ffn_fwd" in lib.suhpe_last_error() and b"share no memory" in lib.suhpe_last_error()
