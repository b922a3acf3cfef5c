"""Layers of transformer blocks in the modes that a user switches to: evaluation, no dropout, other batch sizes, captured graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    from semiuhpe_amd import layers
    return layers


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("training,p", [(False, 0.3), (True, 0.0), (False, 0.0)])
def test_residual_dropout_that_drops_nothing(L, dtype, training, p):
    """skip + branch, rounded once; the gradient goes to both as it is"""
    g = torch.Generator(device="cuda").manual_seed(3)
    branch, skip, dy = (torch.randn(5, 7, 33, generator=g, device="cuda").to(dtype) for _ in range(3))
    layer = L.ResidualDropout(p).train(training)
    tape = []
    y = layer.fwd2(branch, skip, tape)
    assert torch.equal(y, (skip.double() + branch.double()).to(dtype))
    assert torch.equal(layer.fwd2(branch, skip, None), y)
    d_branch, d_skip = layer.bwd2(dy, tape)
    assert torch.equal(d_branch, dy) and torch.equal(d_skip, dy) and not tape
