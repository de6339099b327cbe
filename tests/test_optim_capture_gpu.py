"""An optimiser step's number, rates and random bits are the call's own: a graph would repeat them with every replay."""
import pytest
import torch

from mgpt_b200 import AdamW, MoeError

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_is_not_captured(bits):
    w, g = torch.ones(5000, device="cuda"), torch.full((5000,), 1e-3, device="cuda")
    other = w.clone()
    opt, want = AdamW([w], [g], state_bits=bits), AdamW([other], [g], state_bits=bits)
    for t in (1, 2):
        want.step(t)
    opt.step(1)
    torch.cuda.synchronize()
    with pytest.raises(MoeError, match="captur"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step(2)
    opt.step(2)                                                 # outside it is what it was
    assert torch.equal(w, other) and torch.equal(opt.m.float(), want.m.float()) and torch.equal(opt.v.float(), want.v.float())
