"""The status word of the head loss: found under every name of its device."""
import pytest
import torch

import mgpt_b200
from mgpt_b200 import MoeError

pytestmark = pytest.mark.gpu


def _args(n=20, C=64, V=100):
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w = (torch.randn(k, C, device="cuda", generator=g).bfloat16() for k in (n, V))
    return x, w, torch.randint(0, V, (n,), device="cuda", generator=g, dtype=torch.int32)


@pytest.mark.parametrize("name", [None, "cuda", "cuda:0", 0, torch.device("cuda"), torch.device("cuda", 0)])
def test_every_name_of_the_device(name):
    x, w, t = _args()
    t[3] = 100
    mgpt_b200.head_loss(x, w, t)
    with pytest.raises(MoeError, match="beyond the vocabulary"):
        mgpt_b200.check_status(name)
    mgpt_b200.check_status(name)


def test_a_first_call_in_a_graph_is_refused_and_leaves_nothing(monkeypatch):
    """The status word is made by a device's first call, cleared and waited for: neither can be part of a capture."""
    from mgpt_b200 import training
    monkeypatch.setattr(training, "_status", {})
    x, w, t = _args()
    torch.cuda.synchronize()
    with pytest.raises(MoeError, match="captur"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            mgpt_b200.head_loss(x, w, t)
    assert not training._status
    want, lse = mgpt_b200.head_loss(x, w, t)                    # this makes it
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _ = mgpt_b200.head_loss(x, w, t)
    graph.replay()
    mgpt_b200.check_status()
    assert torch.equal(loss, want)
