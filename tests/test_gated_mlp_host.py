"""GatedMlp stands in Mlp's place but closes no residual connection itself: asked to, it must not pass in silence."""
import pytest
import torch


def test_gated_mlp_takes_no_residual():
    from semiuhpe_amd.src.tiny_vit import GatedMlp
    with pytest.raises(TypeError):
        GatedMlp(24, 96).fwd(torch.zeros(1, 24), None, residual=(torch.zeros(1, 24), None))
