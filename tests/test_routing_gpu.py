"""Routing to experts and its gradient against the formulas in 64 bits.

The indices must be those of 64 bits.  Weights, with u = 2^-24: exp is within 4u, a softmax's sum of E terms within (E/32 + 8)u and its argument
within |z - max| u, a quotient within 3u, the sum over k weights within k u: 64u of the value for these sizes (E to 512, |z| to 20).  Sums of
gradients have terms that cancel: 64u of the terms' sizes.  BF16 results add 2^-8 of themselves.
"""
import math

import pytest
import torch

import mgpt_b200
from mgpt_b200 import MoeError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TINY = 1e-20


def _reference(z, k, score="softmax", bias=None, groups=1, top_groups=None, group_top=2, renormalise=False, scale=1.0):
    """Indices and weights by the definition, on the CPU in 64 bits, token by token where something is out."""
    z = z.double().cpu()
    n, E = z.shape
    b = torch.zeros(E, dtype=torch.float64) if bias is None else bias.double().cpu()
    out = ~(z > -math.inf) | ~(b > -math.inf)
    clean = torch.where(z > -math.inf, z, -math.inf)
    if score == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-clean))
        bad = torch.isnan(z).any(1)
    else:
        top = clean.amax(1, keepdim=True)
        e = torch.where(clean > -math.inf, torch.exp(clean - top), 0.0)
        s = e / e.sum(1, keepdim=True).clamp(min=1e-300)
        bad = (~(z < math.inf)).any(1)
    c = torch.where(out, -math.inf, s + b)
    order = torch.where(out, -math.inf, z) if bias is None else c
    top_groups = groups if top_groups is None else top_groups
    size = E // groups
    inside = torch.ones(n, groups, dtype=torch.bool)
    if top_groups < groups:
        two = c.view(n, groups, size).sort(dim=2, descending=True).values[:, :, :group_top]
        total = torch.where(two > -math.inf, two, 0.0).sum(2)
        total = torch.where(two[:, :, 0] > -math.inf, total, -math.inf)
        best = total.sort(stable=True, dim=1, descending=True).indices[:, :top_groups]
        inside = torch.zeros(n, groups, dtype=torch.bool).scatter_(1, best, True)
    inside = inside.repeat_interleave(size, 1)
    # in order: the experts inside that are not out, then the others inside by index, then nothing
    low = torch.where(inside, torch.where(order == -math.inf, -1e300, order), -math.inf)
    idx = low.sort(stable=True, dim=1, descending=True).indices[:, :k]
    g = torch.where(out, 0.0, s).gather(1, idx)
    w = scale * (g / (g.sum(1, keepdim=True) + TINY) if renormalise else g)
    return idx, torch.where(bad[:, None], math.nan, w), s, bad


def _logits(n, E, dtype=torch.float32, seed=0, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, E, device="cuda", generator=g) * std).to(dtype)


def _bias(E, seed=1, std=0.05):
    return torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * std


def _check(z, k, counts=True, **how):
    seen = torch.full((z.shape[-1],), 3, dtype=torch.int32, device="cuda") if counts else None
    idx, w = mgpt_b200.route(z, k, counts=seen, **how)
    want, want_w, _, bad = _reference(z, k, **how)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32 and idx.shape == w.shape == (z.shape[0], k)
    ok = ~bad
    assert torch.equal(idx.cpu().long()[ok], want[ok])
    assert ((w.cpu().double() - want_w)[ok].abs() <= 64 * U * want_w[ok].abs() + 1e-37).all()
    assert torch.isnan(w.cpu()[bad]).all()
    assert (idx >= 0).all() and (idx < z.shape[1]).all()
    assert (idx.sort(1).values.diff(dim=1) > 0).all()
    if counts:
        assert torch.equal(seen.cpu().long() - 3, torch.bincount(idx.cpu().reshape(-1).long(), minlength=z.shape[1]))
    return idx, w


SHAPES = [(1, 1, 1, 1, 1), (5, 2, 2, 1, 1), (33, 7, 3, 1, 1), (100, 8, 8, 4, 2), (1, 9, 4, 3, 2), (257, 16, 2, 1, 1), (64, 24, 5, 8, 4), (31, 32, 32, 1, 1),
          (129, 33, 6, 3, 2), (1000, 64, 4, 1, 1), (77, 64, 8, 16, 5), (50, 65, 7, 5, 3), (200, 128, 8, 8, 3), (65, 155, 6, 5, 3), (40, 160, 6, 8, 3), (300, 256, 8, 8, 4),
          (7, 257, 9, 1, 1), (129, 384, 12, 32, 10), (19, 510, 32, 30, 7), (130, 512, 32, 16, 2), (3, 512, 1, 2, 1)]


@pytest.mark.parametrize("n,E,k,groups,top_groups", SHAPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(n, E, k, groups, top_groups, score):
    k = min(k, E, top_groups * (E // groups))
    for i, dtype in enumerate((torch.float32, torch.bfloat16)):
        z = _logits(n, E, dtype, seed=n + E + i)
        for bias in (None, _bias(E, seed=E)):
            _check(z, k, score=score, bias=bias, groups=groups, top_groups=top_groups, renormalise=i == 0, scale=2.5 if i == 0 else 1.0, group_top=1 + i)


def test_many_tokens_more_than_the_grid_holds():
    z = _logits(40001, 64, seed=5)
    _check(z, 6, score="sigmoid", bias=_bias(64), groups=8, top_groups=3, renormalise=True)
    _check(z, 6)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(8, 2), (64, 8), (256, 8), (155, 5)])
def test_equal_scores_go_by_index(score, E, groups):
    z = torch.randint(-2, 3, (200, E), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).float()
    z[0] = 0.0
    z[1] = -0.0
    z[2, ::2] = -0.0                                                    # equal to 0
    z[2, 1::2] = 0.0
    bias = torch.randint(0, 2, (E,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).float() * 0.25
    for b in (None, torch.zeros(E, device="cuda"), bias):
        for top_groups in (groups, groups // 2):
            _check(z, 4, score=score, bias=b, groups=groups, top_groups=top_groups)


@pytest.mark.parametrize("E", [16, 256])
def test_scores_closer_than_fp32(E):
    """Biases that make scores equal up to a few 1e-9, and logits one unit in the last place apart."""
    g = torch.Generator(device="cuda").manual_seed(7)
    z = torch.randn(300, E, device="cuda", generator=g)
    z[:, 1::2] = torch.nextafter(z[:, ::2], torch.full_like(z[:, ::2], 9.0))
    for score in ("sigmoid", "softmax"):
        _check(z, 5, score=score, bias=torch.zeros(E, device="cuda"), renormalise=True)
        _check(z, 5, score=score, bias=torch.zeros(E, device="cuda"), groups=E // 2, top_groups=E // 4) if E == 16 else None
        _check(z, 5, score=score)
    z[:, 3::8] = z[:, 0::8]                                             # equal ones, and a better one behind them
    for k in (1, 2, 3, 4):
        _check(z, k)
        _check(z, k, score="sigmoid", bias=torch.zeros(E, device="cuda"))
    z[:, :] = 1.0
    z[:, E - 1] = torch.nextafter(z[:, E - 1], z[:, E - 1] + 1)
    z[1, E - 1] = 1e9
    z[2, : E // 2] = -1e9
    z[3, 5] = math.inf
    for k in (1, 2, 3, 4):
        _check(z, k, score="sigmoid")
        _check(z, k, score="sigmoid", bias=torch.zeros(E, device="cuda"))
        _check(z[:3], k)
        _check(z[:3], k, bias=torch.zeros(E, device="cuda"))
    z = torch.linspace(18.0, 30.0, E, device="cuda").repeat(4, 1)       # sigmoids that are 1 in FP32
    _check(z, 5, score="sigmoid", bias=torch.zeros(E, device="cuda"))
    _check(z.flip(1), 5, score="sigmoid")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(8, 4), (64, 8), (255, 5), (512, 16)])
def test_experts_that_are_out(score, E, groups):
    z = _logits(64, E, seed=11)
    z[0] = -math.inf                                                    # nothing is left
    z[1, 1:] = -math.inf                                                # one is
    z[2, : E // 2] = -math.inf
    z[3, ::2] = -math.inf
    z[4] = torch.finfo(torch.float32).min                               # a mask of the lowest number: not out, but last
    z[5, 1:] = torch.finfo(torch.float32).min
    z[6, 3] = math.nan
    z[7] = math.nan
    z[8, E - 1] = math.inf
    z[9, 2], z[9, 3] = math.nan, -math.inf
    b = _bias(E)
    masked = b.clone()
    masked[1], masked[E - 2] = -math.inf, math.nan
    low = b.clone()
    low[::3] = torch.finfo(torch.float32).min
    high = b.clone()
    high[5] = high[2] = math.inf                                        # chosen first
    for top_groups in (groups, 2):
        for bias in (None, b, masked, low, high):
            _check(z, 3, score=score, bias=bias, groups=groups, top_groups=top_groups, renormalise=True, group_top=2)
            _check(z, 2, score=score, bias=bias, groups=groups, top_groups=top_groups, group_top=1)
    idx, w = mgpt_b200.route(z[:1], 3, score=score, renormalise=True)
    assert idx.tolist() == [[0, 1, 2]] and (w == 0).all()


def test_shapes_strides_and_streams():
    z = _logits(60, 33, torch.bfloat16)
    idx, w = mgpt_b200.route(z.view(3, 4, 5, 33), 4)
    assert idx.shape == w.shape == (3, 4, 5, 4)
    one, w1 = mgpt_b200.route(z[7], 4)                                  # one token, not on a 16-byte boundary
    assert torch.equal(one, idx.view(60, 4)[7]) and torch.equal(w1, w.view(60, 4)[7])
    empty, we = mgpt_b200.route(z[:0], 4)
    assert empty.shape == we.shape == (0, 4)
    assert mgpt_b200.route_backward(z[:0], empty, we).shape == (0, 33)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, w2 = mgpt_b200.route(z.view(3, 4, 5, 33), 4)
        d = mgpt_b200.route_backward(z.view(3, 4, 5, 33), other, w2)
    side.synchronize()
    assert torch.equal(other, idx) and torch.equal(w2, w) and torch.equal(d, mgpt_b200.route_backward(z.view(3, 4, 5, 33), idx, w))


def _grad_reference(z, idx, dw, score, renormalise, scale, out=None):
    z = z.double().requires_grad_()
    s = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)
    g = s.gather(1, idx.long())
    if out is not None:
        g = torch.where(out[idx.long()], 0.0, g)
    w = scale * (g / (g.sum(1, keepdim=True) + TINY) if renormalise else g)
    return torch.autograd.grad(w, z, dw.double())[0], s.detach()


@pytest.mark.parametrize("n,E,k,groups,top_groups", SHAPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_backward(n, E, k, groups, top_groups, score):
    k = min(k, E, top_groups * (E // groups))
    for dtype in (torch.float32, torch.bfloat16):
        z = _logits(n, E, dtype, seed=n + E)
        dw = torch.randn(n, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(E))
        for renormalise in (False, True):
            how = dict(score=score, renormalise=renormalise, scale=1.7)
            idx, _ = mgpt_b200.route(z, k, groups=groups, top_groups=top_groups, **how)
            got = mgpt_b200.route_backward(z, idx, dw, **how)
            want, s = _grad_reference(z, idx, dw, **how)
            g = s.gather(1, idx.long())
            S = g.sum(1, keepdim=True) if renormalise else torch.ones_like(g[:, :1])
            size = s * 1.7 * (dw.abs().double().amax(1, keepdim=True)) * 2 / S * (1 if renormalise else k)
            bound = 64 * U * size + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) * want.abs() + 1e-37
            assert got.dtype == dtype and ((got.double() - want).abs() <= bound).all()
            if score == "sigmoid":
                chosen = torch.zeros_like(want, dtype=torch.bool).scatter_(1, idx.long(), True)
                assert (got[~chosen] == 0).all()


def test_backward_against_differences():
    z = _logits(6, 24, seed=2).double()
    for score in ("softmax", "sigmoid"):
        for renormalise in (False, True):
            how = dict(score=score, renormalise=renormalise, scale=2.0)
            idx, _ = mgpt_b200.route(z.float(), 5, **how)
            dw = torch.randn(6, 5, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
            got = mgpt_b200.route_backward(z.float(), idx, dw, **how)

            def value(v):                               # the weights' sum against dw, with the choice held
                s = torch.sigmoid(v) if score == "sigmoid" else torch.softmax(v, 1)
                g = s.gather(1, idx.long())
                return (2.0 * (g / g.sum(1, keepdim=True) if renormalise else g) * dw.double()).sum()

            base = z.float().double()
            for e in range(24):
                step = torch.zeros_like(base)
                step[:, e] = 1e-4
                for i in range(6):
                    one = torch.zeros_like(base)
                    one[i] = step[i]
                    diff = (value(base + one) - value(base - one)) / 2e-4      # (off by h^2/6 of the third derivative, and 1e-12)
                    assert abs(float(got[i, e]) - float(diff)) < 1e-6


def test_backward_of_experts_that_are_out():
    z = _logits(5, 16, seed=9)
    z[0, 2:] = -math.inf                                                # two left of three
    z[1] = -math.inf
    bias = torch.zeros(16, device="cuda")
    bias[4:] = -math.inf
    dw = torch.ones(5, 6, device="cuda") + torch.arange(6, device="cuda")
    for score in ("softmax", "sigmoid"):
        for renormalise in (False, True):
            how = dict(score=score, renormalise=renormalise)
            idx, w = mgpt_b200.route(z, 6, bias=bias, **how)
            got = mgpt_b200.route_backward(z, idx, dw, bias=bias, **how)
            assert torch.isfinite(got).all() and (got[1] == 0).all() and (got[z == -math.inf] == 0).all()
            want, _ = _grad_reference(z[2:], idx[2:], dw[2:], out=bias == -math.inf, scale=1.0, **how)
            assert (got[2:].double() - want).abs().max() < 1e-5 * 2 ** -3
    z[3, 7] = math.nan
    idx, w = mgpt_b200.route(z, 6)
    assert torch.isnan(w[3]).all() and torch.isfinite(w[2]).all()
    got = mgpt_b200.route_backward(z, idx, dw)
    assert torch.isnan(got[3]).all() and torch.isfinite(got[[0, 1, 2, 4]]).all()


def test_backward_with_indices_of_ones_own():
    """An index outside the experts has no gradient; one that is repeated counts as often."""
    z = _logits(2, 8, seed=4)
    idx = torch.tensor([[3, -1, 8, 2 ** 31 - 1], [5, 5, 1, -2 ** 31]], dtype=torch.int32, device="cuda")
    dw = torch.tensor([[1.0, 2.0, 3.0, 4.0], [1.0, 0.5, 2.0, 7.0]], device="cuda")
    got = mgpt_b200.route_backward(z, idx, dw, score="sigmoid")
    s = torch.sigmoid(z.double())
    d = s * (1 - s)
    want = torch.zeros_like(d)
    want[0, 3], want[1, 5], want[1, 1] = d[0, 3], 1.5 * d[1, 5], 2 * d[1, 1]
    assert ((got.double() - want).abs() <= 32 * U * want.abs()).all()
    p = torch.softmax(z.double(), 1)
    dense = torch.zeros_like(p)
    dense[0, 3], dense[1, 5], dense[1, 1] = 1.0, 1.5, 2.0
    want = p * (dense - (p * dense).sum(1, keepdim=True))
    got = mgpt_b200.route_backward(z, idx, dw, score="softmax")
    assert ((got.double() - want).abs() <= 64 * U * p * 4).all()


def test_calls_in_a_graph():
    z = _logits(500, 64, seed=1)
    bias = _bias(64)
    counts = torch.zeros(64, dtype=torch.int32, device="cuda")
    dw = torch.randn(500, 6, device="cuda")
    how = dict(score="sigmoid", renormalise=True)
    idx, w = mgpt_b200.route(z, 6, bias=bias, groups=8, top_groups=4, **how)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gi, gw = mgpt_b200.route(z, 6, bias=bias, groups=8, top_groups=4, counts=counts, **how)
        gd = mgpt_b200.route_backward(z, gi, dw, **how)
    for seed in (3, 4):
        z.copy_(_logits(500, 64, seed=seed))
        counts.zero_()
        graph.replay()
        idx, w = mgpt_b200.route(z, 6, bias=bias, groups=8, top_groups=4, **how)
        assert torch.equal(gi, idx) and torch.equal(gw, w) and torch.equal(gd, mgpt_b200.route_backward(z, idx, dw, **how))
        assert int(counts.sum()) == 3000


def test_refusals():
    z = _logits(4, 16)
    for bad in (dict(top_k=0), dict(top_k=17), dict(top_k=33), dict(top_k=4, groups=3), dict(top_k=4, groups=0), dict(top_k=4, groups=4, top_groups=5), dict(top_k=4, groups=4, top_groups=0),
                dict(top_k=5, groups=4, top_groups=1), dict(top_k=2, score="tanh"), dict(top_k=2, group_top=3), dict(top_k=2, scale=math.inf), dict(top_k=2, bias=torch.zeros(15, device="cuda")),
                dict(top_k=2, bias=torch.zeros(16, device="cuda", dtype=torch.bfloat16)), dict(top_k=2, counts=torch.zeros(16, device="cuda")), dict(top_k=2, groups=2 ** 40)):
        with pytest.raises(MoeError):
            mgpt_b200.route(z, **bad)
    for tensor in (z.half(), z.t(), z.cpu(), torch.zeros(3, 0, device="cuda"), torch.zeros(2, 513, device="cuda")):
        with pytest.raises(MoeError):
            mgpt_b200.route(tensor, 1)
    idx, w = mgpt_b200.route(z, 2)
    for args in ((z, idx.long(), w), (z, idx[:3], w), (z, idx, w.double()), (z, idx, w[:, :1]), (z, idx[0], w)):
        with pytest.raises(MoeError):
            mgpt_b200.route_backward(*args)
