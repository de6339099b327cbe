"""Routing, kept activations and the layer together: a model's step, and the layer cut at its exchange points.

The step's gradients are compared with those of the same step on whole activations.  What was kept is off by 2^-8 of a group's largest value at
most, about 2^-8 / sqrt(3) / 2 of a value in the mean; a gradient of the norm before the head, or of the embedding, is a sum of products with
such values: 1e-2 of its norm is above that and the BF16 roundings that both steps have alike.
"""
import ctypes as ct
import importlib.util
import os

import pytest
import torch

import mgpt_b200
from mgpt_b200 import MoELayer, _lib
from tests.test_layer_routing_gpu import _formula, _idx, _layer, _rel

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_lm.py")


@pytest.fixture(scope="module")
def lm():
    spec = importlib.util.spec_from_file_location("train_lm", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("routing", [None, "softmax", "sigmoid"])
def test_gradients_of_a_step_from_what_was_kept(lm, routing):
    tokens, targets = lm.batch(16, 64, 1000, 5)
    grads = []
    for bits in (16, 8):
        model = lm.Model(blocks=2, routing=routing, kept_bits=bits)
        loss = model.step(tokens, targets, lr=0.0)
        grads.append((float(loss), [g.clone() for g in model.grads], [b.clone() for b in model.bias if b is not None]))
    assert grads[0][0] == grads[1][0]                                   # the forward pass is the same
    whole = torch.cat([g.reshape(-1) for g in grads[0][1]]).double()
    kept = torch.cat([g.reshape(-1) for g in grads[1][1]]).double()
    assert 0 < _rel(kept, whole) < 1e-2
    for b in grads[0][2]:
        assert (b == 0).all()


@pytest.mark.parametrize("routing", ["softmax", "sigmoid"])
def test_a_gradient_against_differences(lm, routing):
    """The loss at embeddings moved along the gradient, against the gradient's square: the tolerance of the step without these."""
    tokens, targets = lm.batch(16, 64, 1000, 5)
    model = lm.Model(blocks=1, routing=routing, kept_bits=8)
    base = model.embed.clone()
    model.step(tokens, targets, lr=0.0)
    grad = model.d_embed.clone()
    size = grad.norm()
    s = 0.02 * base.norm() / size
    ends = []
    for sign in (1, -1):
        model.embed.copy_(base + sign * s * grad)
        model.head.copy_(model.embed)
        ends.append(float(model.step(tokens, targets, lr=0.0)))
    want = float(2 * s * size ** 2)
    assert abs(ends[0] - ends[1] - want) <= 0.15 * want


def test_it_runs_and_moves_the_bias(lm):
    losses = lm.train(steps=12, routing="sigmoid", kept_bits=8)
    assert len(losses) == 12 and all(v == v and abs(v) < 100 for v in losses)
    model = lm.Model(routing="sigmoid")
    model.step(*lm.batch(16, 64, 1000, 1))
    torch.cuda.synchronize()
    assert all(float(b.abs().max()) == pytest.approx(1e-3) for b in model.bias)


def test_router_of_ones_own_and_the_experts_plan():
    """A router's product, route, the plan over its indices: the counts agree, and every row is an expert's that the token chose."""
    n, E, k = 700, 64, 6
    g = torch.Generator(device="cuda").manual_seed(0)
    logits, bias = torch.randn(n, E, device="cuda", generator=g), torch.randn(E, device="cuda", generator=g) * 0.05
    counts = torch.zeros(E, dtype=torch.int32, device="cuda")
    idx, w = mgpt_b200.route(logits, k, score="sigmoid", bias=bias, groups=8, top_groups=4, renormalise=True, counts=counts)
    lib = _lib.load()
    R, cap = n * k, (n * k + E * 127) // 128 * 128
    i32 = dict(dtype=torch.int32, device="cuda")
    out = dict(counts=torch.empty(E, **i32), offsets=torch.empty(E, **i32), padded=torch.empty(E + 1, **i32), tile=torch.empty(cap // 128, **i32), tiles=torch.empty(1, **i32),
               map=torch.empty(R, **i32), pos=torch.empty(R, **i32), row=torch.empty(cap, **i32), status=torch.zeros(1, **i32))
    size = lib.mgpt_moe_op_plan_scratch_bytes(R, E)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    p = {k_: v.data_ptr() for k_, v in out.items()}
    _lib.check(lib.mgpt_moe_op_plan(idx.data_ptr(), R, E, p["counts"], p["offsets"], p["padded"], p["tile"], p["tiles"], p["map"], p["pos"], p["row"], cap, p["status"],
                                    scratch.data_ptr(), size, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out["counts"], counts) and int(out["status"]) == 0
    expert_of_row = torch.bucketize(out["pos"], out["padded"][1:], right=True)
    assert torch.equal(expert_of_row.view(n, k).int(), idx)


@pytest.mark.parametrize("mode,dtype", [("fp32", torch.float32), ("bf16", torch.bfloat16)])
def test_the_layer_cut_at_its_exchange_points(mode, dtype):
    """The routing side of an expert-parallel layer under set_routing: rows out, rows back, and the gradient, beside the whole layer's."""
    n, C, H, E, k = 333, 64, 128, 8, 3
    bias = torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 0.1
    how = dict(score="sigmoid", bias=bias, groups=4, top_groups=2, renormalise=True, scale=1.5)
    whole = _layer(C, H, E, k, mode)
    whole.set_routing(**how)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(n, C, device="cuda", generator=g).to(dtype) for _ in range(2))
    whole.zero_grad()
    y = whole.forward(x)
    dx = whole.backward(dy)
    side = _layer(C, H, E, k, mode)                                     # routes; its own experts stay idle
    side.set_routing(**how)
    experts = MoELayer(C, H, E, 1, mode=mode)
    experts.load_parameters([p.detach().cpu().numpy() for p in whole.get_parameters()])
    side.zero_grad()
    experts.zero_grad()
    lib, st, io = _lib.load(), torch.cuda.current_stream().cuda_stream, 1 if dtype == torch.bfloat16 else 0

    def view(layer, ws, count, name, t):
        off, size = ct.c_size_t(), ct.c_size_t()
        _lib.check(lib.mgpt_moe_workspace_view(layer._h, count, name.encode(), ct.byref(off), ct.byref(size)))
        return ws[off.value: off.value + size.value].view(t)

    size = lib.mgpt_moe_stage_workspace_bytes(side._h, n, 1)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    cap = view(side, ws, n, "row_src", torch.int32).numel()
    rows = torch.zeros(cap, C, dtype=dtype, device="cuda")
    _lib.check(lib.mgpt_moe_route(side._h, x.data_ptr(), n, io, ws.data_ptr(), size, rows.data_ptr(), st))
    counts = view(side, ws, n, "counts", torch.int32).clone()
    used = int(((counts + 127) // 128 * 128).sum())
    size2 = lib.mgpt_moe_stage_workspace_bytes(experts._h, used, 0)
    ws2 = torch.zeros(size2, dtype=torch.uint8, device="cuda")
    out, back, d_rows, d_in = (torch.zeros_like(rows) for _ in range(4))
    _lib.check(lib.mgpt_moe_experts_forward(experts._h, rows.data_ptr(), counts.data_ptr(), 1, used, out.data_ptr(), ws2.data_ptr(), size2, st))
    y2, dx2 = torch.empty_like(y), torch.empty_like(y)
    _lib.check(lib.mgpt_moe_combine(side._h, out.data_ptr(), y2.data_ptr(), io, ws.data_ptr(), size, st))
    _lib.check(lib.mgpt_moe_combine_backward(side._h, out.data_ptr(), dy.data_ptr(), io, d_rows.data_ptr(), ws.data_ptr(), size, st))
    _lib.check(lib.mgpt_moe_experts_backward(experts._h, d_rows.data_ptr(), d_in.data_ptr(), ws2.data_ptr(), size2, st))
    _lib.check(lib.mgpt_moe_route_backward(side._h, x.data_ptr(), d_in.data_ptr(), dx2.data_ptr(), io, ws.data_ptr(), size, st))
    bar = 1e-5 if mode == "fp32" else 1e-2
    assert _rel(y2, y.double()) < bar and _rel(dx2, dx.double()) < bar
    for i in (0, 1):
        assert _rel(side.get_parameters()[i].grad, whole.get_parameters()[i].grad.double()) < bar


@pytest.mark.parametrize("chunks", [1, 2])
@pytest.mark.parametrize("mode,dtype", [("fp32", torch.float32), ("bf16", torch.bfloat16)])
def test_the_expert_parallel_layer_with_one_rank(mode, dtype, chunks):
    from mgpt_b200.ep import ExpertParallelMoE
    n, C, H, E, k = 333, 64, 128, 8, 3
    bias = torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 0.1
    how = dict(bias=bias, groups=4, top_groups=2, renormalise=True, scale=1.5)
    whole = _layer(C, H, E, k, mode)
    ep = ExpertParallelMoE(C, H, E, k, mode=mode, n_chunks=chunks)
    ep.load_parameters([p.detach() for p in whole.get_parameters()])
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(n, C, device="cuda", generator=g).to(dtype) for _ in range(2))
    bar = 1e-5 if mode == "fp32" else 1e-2
    for score in ("sigmoid", "softmax", None):
        for layer in (whole, ep):
            layer.set_routing(score, **(how if score else {}))
            layer.zero_grad()
        y, y2 = whole.forward(x), ep.forward(x)
        dx, dx2 = whole.backward(dy), ep.backward(dy)
        assert _rel(y2, y.double()) < bar and _rel(dx2, dx.double()) < bar
        for p, q in zip(whole.get_parameters(), ep.get_parameters()):
            assert _rel(q.grad, p.grad.double()) < bar


@pytest.mark.parametrize("mode,dtype", [("fp32", torch.float32), ("bf16", torch.bfloat16)])
def test_the_blocks_glue(mode, dtype):
    n, C, H, E, k = 150, 64, 128, 8, 2
    how = dict(score="sigmoid", renormalise=True, scale=2.0)
    layer = _layer(C, H, E, k, mode)
    layer.set_routing(**how)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dout = (torch.randn(n, C, device="cuda", generator=g).to(dtype) for _ in range(2))
    scale = 1 + 0.1 * torch.randn(C, device="cuda", generator=g)
    layer.zero_grad()
    y = layer.block_forward(x, scale, eps=1e-5)
    idx = _idx(layer, n, how, k)
    d_scale = torch.zeros_like(scale)
    dx = layer.block_backward(scale, dout, d_scale)
    leaf = x.double().requires_grad_()
    u = leaf / torch.sqrt((leaf * leaf).mean(1, keepdim=True) + 1e-5) * scale.double()
    want_u, du, _ = _formula(layer, u.detach(), idx, how, dout)
    want_dx = torch.autograd.grad(u, leaf, du)[0] + dout.double()
    bar = 1e-5 if mode == "fp32" else 2e-2
    assert _rel(y, x.double() + want_u) < bar and _rel(dx, want_dx) < bar


@pytest.mark.parametrize("n", [300, 5000])
def test_a_routers_bias_gradient_is_the_same_every_time(n):
    layer = _layer(128, 64, 24, 4, "bf16")
    layer.set_routing("softmax")
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(n, 128, device="cuda", generator=g).bfloat16() for _ in range(2))
    seen = []
    for _ in range(3):
        layer.zero_grad()
        layer.forward(x)
        layer.backward(dy)
        seen.append(layer.get_parameters()[1].grad.clone())
    assert torch.equal(seen[0], seen[1]) and torch.equal(seen[0], seen[2])
    dz = layer.workspace_view("dlogits", torch.float32, (n, 24)).double()
    assert ((seen[0].double() - dz.sum(0)).abs() <= (n / 2 + 64) * 2.0 ** -24 * dz.abs().sum(0)).all()
