"""The logits that a layer under set_routing chooses its experts from, beyond the size where they come from the tensor cores.

Wr is in two BF16 pieces there, off by 2^-16 of a weight (2^-8 of 2^-8), and its products with BF16 tokens are exact; 2 C / 16 additions of 16 products
to an FP32 sum, truncated at worst, are within C / 4 * 2^-24 of the sum of the products' sizes, the exact kernel's C additions within C * 2^-24, and that sum
is at most |x| |w|.  The documented bound, (1.5 C 2^-24 + 2^-16) |x| max |w|, is above all of it; the bias adds 2^-24 of itself and of the sum.
"""
import pytest
import torch

from mgpt_b200 import MoELayer
from tests.test_routing_gpu import _reference

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("n,C,E,size", [(4096, 2048, 64, 1.0), (13000, 256, 128, 1.0), (13000, 256, 128, 40.0), (30011, 520, 33, 3.0)])
def test_logits(n, C, E, size):
    g = torch.Generator(device="cuda").manual_seed(C)
    layer = MoELayer(C, 64, E, 4, mode="bf16")
    wr = torch.randn(C, E, device="cuda", generator=g) * C ** -0.5          # FP32: no BF16 numbers
    br = torch.randn(1, E, device="cuda", generator=g) * 0.1
    rest = [torch.randn(p.shape, device="cuda", generator=g) * 0.05 for p in layer.get_parameters()[2:]]
    layer.load_parameters([p.cpu().numpy() for p in (wr, br, *rest)])
    bias = torch.randn(E, device="cuda", generator=g) * 0.05
    how = dict(score="sigmoid", bias=bias, renormalise=True)
    layer.set_routing(**how)
    x = (torch.randn(n, C, device="cuda", generator=g) * size).bfloat16()
    layer.forward(x)
    z = layer.workspace_view("logits", torch.float32, (n, E))
    exact = x.double() @ wr.double() + br.double()
    lengths = x.double().norm(dim=1, keepdim=True) * wr.double().norm(dim=0).max()
    bound = (1.5 * C * U + 2.0 ** -16) * lengths + 4 * U * (lengths + br.abs().max())
    assert ((z.double() - exact).abs() <= bound).all()
    idx = layer.workspace_view("top_idx", torch.int32, (n, 4))
    assert torch.equal(idx.cpu().long(), _reference(z, 4, **how)[0])        # chosen from these logits
