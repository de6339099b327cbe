"""The norms where every group of warps takes several tokens: a ring that is filled again, forward and backward, for every number of warps."""
import pytest
import torch

import tests.test_residual_norm_gpu as small

pytestmark = pytest.mark.gpu
B, F = torch.bfloat16, torch.float32


# warps per token, BF16: 1 1 2 4 4 8 8, no ring; FP32: 1 2 4 8 8, no ring
@pytest.mark.parametrize("n,C,dtype,per", [(20000, 264, B, 0), (21001, 512, B, 1000), (12007, 1000, B, 0), (6001, 2048, B, 97), (5003, 1032, B, 0), (3000, 2056, B, 0), (2999, 4096, B, 300),
                                           (1501, 4104, B, 0), (20000, 136, F, 0), (11000, 512, F, 1), (7000, 1024, F, 0), (5000, 2048, F, 613), (3000, 2056, F, 0), (1300, 8200, F, 0)])
def test_several_tokens_per_group(n, C, dtype, per):
    small.test_forward_and_backward(n, C, dtype, per)
