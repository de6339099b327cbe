"""The layer under set_routing: routing, outputs and all gradients against the formulas in 64 bits, in every way the layer is called.

Bars as for the layer's own routing: rel-L2 1e-5 in FP32 mode, 2e-2 in BF16 mode; the choice of experts is that of the logits that the
layer's router left in the workspace.
"""
import pytest
import torch

import mgpt_b200
from mgpt_b200 import MoeError, MoELayer
from tests.test_routing_gpu import _reference

pytestmark = pytest.mark.gpu


def _layer(C, H, E, k, mode, seed=0, gemm_impl=0):
    g = torch.Generator().manual_seed(seed)
    layer = MoELayer(C, H, E, k, mode=mode, gemm_impl=gemm_impl)
    layer.load_parameters([(torch.randn(p.shape, generator=g) * (p.shape[0] ** -0.5 if p.shape[0] > 1 else 0.1)).bfloat16().float().numpy() for p in layer.get_parameters()])
    return layer


def _formula(layer, x, idx, how, dy=None):
    """y (and the gradients) in 64 bits, the choice given."""
    P = [p.detach().double().requires_grad_(dy is not None) for p in layer.get_parameters()]
    x = x.double().requires_grad_(dy is not None)
    z = x @ P[0] + P[1]
    s = torch.sigmoid(z) if how["score"] == "sigmoid" else torch.softmax(z, 1)
    w = s.gather(1, idx)
    w = how.get("scale", 1.0) * (w / (w.sum(1, keepdim=True) + 1e-20) if how.get("renormalise") else w)
    y = torch.zeros_like(x)
    for e in range(layer.E):
        tok, j = torch.nonzero(idx == e, as_tuple=True)
        Wg, bg, Wu, bu, Wd, bd = P[2 + 6 * e: 8 + 6 * e]
        if len(tok):
            r = x[tok]
            out = (torch.nn.functional.silu(r @ Wg + bg) * (r @ Wu + bu)) @ Wd + bd
            y = y.index_add(0, tok, w[tok, j, None] * out)
    if dy is None:
        return y
    grads = torch.autograd.grad(y, [x] + P, dy.double(), allow_unused=True)
    return y.detach(), grads[0], [torch.zeros_like(p) if g is None else g for p, g in zip(P, grads[1:])]


def _rel(got, want):
    return float((got.double() - want).norm() / want.norm().clamp(min=1e-12))


def _idx(layer, n, how, k):
    z = layer.workspace_view("logits", torch.float32, (n, layer.E))
    want, w, _, _ = _reference(z, k, **how)
    idx = layer.workspace_view("top_idx", torch.int32, (n, k))
    assert torch.equal(idx.cpu().long(), want)
    assert (layer.workspace_view("top_p", torch.float32, (n, k)).cpu().double() - w).abs().max() < 1e-5
    return idx.long().clone()


WAYS = [dict(score="sigmoid", renormalise=True, scale=2.5, bias=True, groups=4, top_groups=2), dict(score="softmax", renormalise=True), dict(score="softmax"),
        dict(score="sigmoid", bias=True)]


@pytest.mark.parametrize("mode,dtype,gemm_impl", [("fp32", torch.float32, 0), ("bf16", torch.bfloat16, 0), ("bf16", torch.float32, 0), ("bf16", torch.bfloat16, 1)])
@pytest.mark.parametrize("n,C,H,E,k", [(5, 64, 128, 8, 2), (300, 128, 256, 8, 3), (333, 64, 72, 12, 4), (200, 40, 64, 6, 2)])
@pytest.mark.parametrize("way", range(len(WAYS)))
def test_forward_and_backward(mode, dtype, gemm_impl, n, C, H, E, k, way):
    how = dict(WAYS[way])
    if E % how.get("groups", 1):
        how.update(groups=3)
    g = torch.Generator(device="cuda").manual_seed(n)
    if how.pop("bias", False):
        how["bias"] = torch.randn(E, device="cuda", generator=g) * 0.1
    layer = _layer(C, H, E, k, mode, gemm_impl=gemm_impl)
    layer.set_routing(**how)
    x, dy = (torch.randn(n, C, device="cuda", generator=g).bfloat16().to(dtype) for _ in range(2))
    layer.zero_grad()
    y = layer.forward(x)
    idx = _idx(layer, n, how, k)
    dx = layer.backward(dy)
    want_y, want_dx, want = _formula(layer, x, idx, how, dy)
    bar = 1e-5 if mode == "fp32" else 2e-2
    assert _rel(y, want_y) < bar and _rel(dx, want_dx) < bar
    for i, (p, w) in enumerate(zip(layer.get_parameters(), want)):
        if float(w.norm()) > 0:
            assert _rel(p.grad, w) < bar, i
    counts = torch.bincount(idx.reshape(-1), minlength=E).tolist()
    assert layer.get_expert_counts() == counts
    layer.check_status()


@pytest.mark.parametrize("mode,dtype", [("fp32", torch.float32), ("bf16", torch.bfloat16)])
def test_other_calls_route_alike(mode, dtype):
    """Recompute with the saved routing, inference, the block's calls: the same choice, and the same bits where the arithmetic is the same."""
    n, C, H, E, k = 260, 64, 128, 16, 4
    bias = torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 0.1
    how = dict(score="sigmoid", bias=bias, groups=4, top_groups=3, renormalise=True, scale=1.5)
    layer = _layer(C, H, E, k, mode)
    layer.set_routing(**how)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(n, C, device="cuda", generator=g).to(dtype) for _ in range(2))
    layer.zero_grad()
    y = layer.forward(x)
    dx = layer.backward(dy)
    grads = [p.grad.clone() for p in layer.get_parameters()]
    layer.zero_grad()
    layer.forward(x)
    saved = layer.save_routing()
    layer._ws.zero_()                                                   # the arena is someone else's in between
    again = torch.empty_like(y)
    layer.recompute_into(x, again, saved)
    assert torch.equal(again, y)
    assert torch.equal(layer.backward(dy), dx)
    for a, p in zip(grads, layer.get_parameters()):
        assert _rel(p.grad, a.double()) < 1e-5
    assert torch.equal(layer.forward_inference(x), y)
    scale = torch.ones(C, device="cuda")
    out = layer.block_forward(x, scale)
    u = layer.block_input().clone()
    assert _rel(out, x.double() + layer.forward(u).double()) < (1e-5 if mode == "fp32" else 2e-2)
    # a bias changed in place is seen by the next call
    before = layer.forward(x).clone()
    bias.neg_()
    assert not torch.equal(layer.forward(x), before)
    _idx(layer, n, how, k)
    # and the reference's routing comes back
    layer.set_routing()
    plain = _layer(C, H, E, k, mode)
    assert torch.equal(layer.forward(x), plain.forward(x))


def test_tensor_core_router():
    """Enough work for the first pass on the tensor cores: experts are chosen from its logits."""
    n, C, H, E, k = 13000, 256, 64, 128, 4
    how = dict(score="sigmoid", bias=torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 0.05, groups=8, top_groups=4, renormalise=True)
    layer = _layer(C, H, E, k, "bf16")
    layer.set_routing(**how)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(n, C, device="cuda", generator=g).bfloat16() for _ in range(2))
    layer.zero_grad()
    y = layer.forward(x)
    idx = _idx(layer, n, how, k)
    z = layer.workspace_view("logits", torch.float32, (n, E))
    exact = x.double() @ layer.get_parameters()[0].double() + layer.get_parameters()[1].double()
    assert float((z.double() - exact).abs().max()) < 1e-4
    dx = layer.backward(dy)
    want_y, want_dx, want = _formula(layer, x, idx, how, dy)
    assert _rel(y, want_y) < 2e-2 and _rel(dx, want_dx) < 2e-2
    for i in (0, 1, 2, 3, 6, 7):
        assert _rel(layer.get_parameters()[i].grad, want[i]) < 2e-2, i


def test_tokens_without_experts_of_their_own():
    """A router bias of minus infinity takes experts out; a NaN among the tokens stays in its own row."""
    layer = _layer(64, 64, 8, 3, "bf16")
    layer.set_routing("softmax", renormalise=True)
    layer.get_parameters()[1][0, 3:] = -float("inf")
    x = torch.randn(70, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    y = layer.forward(x)
    assert torch.isfinite(y).all() and layer.get_expert_counts() == [70, 70, 70, 0, 0, 0, 0, 0]
    layer.get_parameters()[1][0, 2:] = -float("inf")
    y = layer.forward(x)                                                # the third place has weight 0
    assert torch.isfinite(y).all() and layer.get_expert_counts() == [70, 70, 70, 0, 0, 0, 0, 0]
    assert (layer.workspace_view("top_p", torch.float32, (70, 3))[:, 2] == 0).all()
    dx = layer.backward(x)
    assert torch.isfinite(dx).all()
    x[5, 7] = float("nan")
    y = layer.forward(x)
    assert torch.isnan(y[5]).all() and torch.isfinite(y[[0, 4, 6, 69]]).all()
    layer.check_status()


def test_a_step_in_a_graph():
    layer = _layer(128, 128, 16, 2, "bf16")
    bias = torch.zeros(16, device="cuda")
    layer.set_routing("sigmoid", bias=bias, renormalise=True)
    x = torch.randn(512, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    y = layer.forward(x)
    layer.backward(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy = layer.forward(x)
        gdx = layer.backward(x)
    bias.copy_(torch.randn(16, device="cuda") * 0.2)
    layer.zero_grad()
    graph.replay()
    torch.cuda.synchronize()
    got = gy.clone(), gdx.clone()
    y = layer.forward(x)
    assert torch.equal(y, got[0]) and torch.equal(layer.backward(x), got[1])


def test_refusals():
    layer = _layer(64, 64, 8, 2, "bf16")
    for bad in (dict(score="relu"), dict(score="sigmoid", groups=3), dict(score="sigmoid", groups=8, top_groups=1), dict(score="softmax", bias=torch.zeros(7, device="cuda")),
                dict(score="softmax", scale=float("nan"))):
        with pytest.raises(MoeError):
            layer.set_routing(**bad)
    x = torch.randn(4, 64, device="cuda").bfloat16()
    layer.forward(x)
    layer.set_routing("sigmoid")
    with pytest.raises(MoeError):
        layer.backward(x)                                               # of a forward under the other routing
    assert mgpt_b200.MoELayer is MoELayer
