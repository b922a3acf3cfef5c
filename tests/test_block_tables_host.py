"""Tables that blocks keep on the device (rotary positions): what is handed out stays, on the CPU."""
import pytest
import torch


def test_rotary_position_tables_are_kept():
    from semiuhpe_amd import kernels as K
    first = K.rope_grid(3, 5, 4, "cpu")
    want = torch.cartesian_prod(torch.arange(5), torch.arange(4)).to(torch.int32).repeat(3, 1)
    assert first.dtype == torch.int32 and first.is_contiguous() and torch.equal(first, want)
    at = first.data_ptr()
    fewer, more = K.rope_grid(2, 5, 4, "cpu"), K.rope_grid(7, 5, 4, "cpu")
    assert fewer.data_ptr() == at and fewer.shape == (40, 2) and fewer.is_contiguous()
    assert more.shape == (140, 2) and torch.equal(more[:60], want)
    del first
    again = K.rope_grid(3, 5, 4, "cpu")                     # another batch size in between: the same memory still holds the same table
    assert again.data_ptr() == at and torch.equal(again, want)
    assert K.rope_grid(3, 4, 5, "cpu").data_ptr() != at
    plan = K.rope_plan(32, (16, 16), "cpu")
    assert K.rope_plan(32, [16, 16], "cpu") is plan and K.rope_plan(32, (8, 8), "cpu") is not plan


def test_no_table_is_made_inside_a_capture(monkeypatch):
    from semiuhpe_amd import kernels as K
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    K._made_outside_capture("cpu", "x")                     # nothing to do with a device that captures nothing
    with pytest.raises(RuntimeError, match="capture"):
        K.rope_grid(11, 13, 17, "cuda")
    with pytest.raises(RuntimeError, match="capture"):
        K.rope_plan(96, (48, 48), "cuda")
