"""Forward-only calls of the layers whose products run on the CUDA cores: the same y as the training forward."""
import pytest
import torch

from mgpt_b200 import MoELayer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode,gemm_impl", [("fp32", 0), ("bf16", 1)])
@pytest.mark.parametrize("n", [1, 9, 260])
def test_inference_equals_forward(mode, gemm_impl, n):
    layer = MoELayer(64, 128, 16, 4, mode=mode, gemm_impl=gemm_impl)
    g = torch.Generator().manual_seed(1)
    layer.load_parameters([torch.randn(p.shape, generator=g).numpy() * 0.2 for p in layer.get_parameters()])
    x = torch.randn(n, 64, generator=g).cuda()
    y = layer.forward(x)
    layer._ws = None                                # a workspace of the inference size, not the larger one of training
    assert torch.equal(layer.forward_inference(x), y)
    layer.check_status()
