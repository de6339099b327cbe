"""Every expert of every token, and nearly: as many chosen experts per warp as there are (512: 32 tokens with 16, 16 with 32), and groups of tiny numbers."""
import pytest
import torch

import mgpt_b200
from tests.test_routing_gpu import _bias, _check, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,E,k", [(19001, 16, 16), (19001, 16, 15), (9503, 32, 32), (9503, 32, 31), (70, 16, 16), (70, 32, 32), (9503, 32, 17)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(n, E, k, score):
    z = _logits(n, E, seed=n + k)
    for bias in (None, _bias(E, seed=E)):
        _check(z, k, score=score, bias=bias, renormalise=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_kept_values_below_the_smallest_unit(dtype):
    """Half a unit of 2^-126 whatever the largest; 1/127 of it from 2^-120 on."""
    x = torch.randn(400, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).double()
    x = (x * 2.0 ** -(100.0 + torch.arange(400, device="cuda", dtype=torch.float64)[:, None] * 0.1)).to(dtype)
    back = mgpt_b200.restore8(mgpt_b200.keep8(x))
    off = (back.double() - x.double()).abs().view(400, 2, 32).amax(2)
    largest = x.double().abs().view(400, 2, 32).amax(2)
    assert (off <= torch.clamp(largest / 127, min=2.0 ** -127)).all()
    low = largest <= 2.0 ** -127
    assert low.any() and (back.view(400, 2, 32)[low] == 0).all()
