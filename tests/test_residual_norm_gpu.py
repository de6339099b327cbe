"""The norms around a block, its gate and the skip connection, and all gradients, against the formulas in 64 bits.

Bounds, with u = 2^-24: a value goes through at most about 40 roundings to FP32 (the sums over a row are taken 16 to 64 at a time in
each thread and then pairwise, and count for 24 of them), each of which is at most u of the sizes of the terms; sums over n tokens
add n/2 + 64 roundings of the sum of the terms' sizes.  BF16 results add 2^-8 of themselves.
"""
import pytest
import torch

import mgpt_b200
from mgpt_b200 import MoeError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-5


def _inputs(n, C, dtype, per, post=True, gate=True, pre=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)                                             # noqa: E731
    x, h, dy, du = ((r(n, C) * s).to(dtype) for s in (2.0, 0.7, 1.0, 1.0))
    rows = -(-n // per) if per else 1
    a = dict(post_scale=1 + 0.1 * r(C) if post else None, gate=0.5 * r(rows, C) if gate else None, pre_scale=1 + 0.1 * r(C) if pre else None,
             alpha=0.8, eps=EPS, tokens_per_gate=per)
    return x, h, dy, du if pre else None, a


def _reference(x, h, dy, du, a):
    n, C = x.shape
    d = {k: v.double().requires_grad_() for k, v in (("x", x), ("h", h), ("post", a["post_scale"]), ("gate", a["gate"]), ("pre", a["pre_scale"])) if v is not None}
    per = a["tokens_per_gate"] or max(n, 1)
    hn = d["h"]
    if "post" in d:
        hn = hn / torch.sqrt((hn * hn).mean(1, keepdim=True) + EPS) * d["post"]
    if "gate" in d:
        hn = hn * d["gate"][torch.arange(n, device="cuda") // per]
    y = a["alpha"] * d["x"] + hn
    u = y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS) * d["pre"] if "pre" in d else None
    outs, ups = ((y, u), (dy.double(), du.double())) if u is not None else ((y,), (dy.double(),))
    grads = dict(zip(d, torch.autograd.grad(outs, list(d.values()), ups)))
    return y.detach(), None if u is None else u.detach(), grads


def _near(got, want, k, what, row_max=True):
    """|got - want| within k roundings of the row's largest value (terms of that size cancel in it), and BF16's of the value."""
    size = want.abs().amax(-1, keepdim=True) if row_max else want.abs()
    bound = k * U * size + (2.0 ** -8 if got.dtype == torch.bfloat16 else 0.0) * want.abs() + 1e-30
    over = (got.double() - want).abs() - bound
    assert not over.isnan().any() and (over <= 0).all(), f"{what}: {float(over.max()):.3g} over"


CASES = [(1, 8, torch.float32, 0), (3, 64, torch.bfloat16, 2), (8, 1024, torch.bfloat16, 0), (1021, 320, torch.float32, 256), (777, 1000, torch.bfloat16, 100),
         (300, 2048, torch.bfloat16, 0), (300, 2056, torch.float32, 7), (33, 4096, torch.bfloat16, 1), (33, 4104, torch.bfloat16, 0), (20, 8200, torch.float32, 3),
         (9, 16384, torch.bfloat16, 0), (5000, 264, torch.bfloat16, 5000), (2500, 40, torch.float32, 3)]


@pytest.mark.parametrize("n,C,dtype,per", CASES)
def test_forward_and_backward(n, C, dtype, per):
    x, h, dy, du, a = _inputs(n, C, dtype, per, seed=n + C)
    y, u, stats = mgpt_b200.residual_norm(x, h, **a)
    want_y, want_u, g = _reference(x, h, dy, du, a)
    _near(y, want_y, 40, "y")
    _near(u, want_u, 40, "u")
    grads = {k: torch.randn_like(v) for k, v in (("post", a["post_scale"]), ("gate", a["gate"]), ("pre", a["pre_scale"]))}
    before = {k: v.double() for k, v in grads.items()}
    dx, dh = mgpt_b200.residual_norm_backward(x, h, stats, dy, du, d_post_scale=grads["post"], d_gate=grads["gate"], d_pre_scale=grads["pre"], **a)
    _near(dx, g["x"], 80, "dx")
    _near(dh, g["h"], 160, "dh")                                    # (terms that cancel to a value are a few times the row's largest)
    # sizes of the terms of the sums over tokens: |D h_hat| and |du y_hat| are of the order of sqrt(n) times the sums themselves
    for k in grads:
        size = (n ** 0.5 + 1) * (g[k].abs().mean() + g[k].abs()) * 4
        over = (grads[k].double() - before[k] - g[k]).abs() - ((n / 2 + 64) * U * size + 4 * U * before[k].abs())
        assert (over <= 0).all(), f"d_{k}: {float(over.max()):.3g} over"


@pytest.mark.parametrize("post,gate,pre", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)])
def test_parts_that_are_absent(post, gate, pre):
    x, h, dy, du, a = _inputs(70, 136, torch.float32, 20 if gate else 0, post, gate, pre, seed=2)
    y, u, stats = mgpt_b200.residual_norm(x, h, **a)
    want_y, want_u, g = _reference(x, h, dy, du, a)
    _near(y, want_y, 40, "y")
    assert (u is None) == (not pre)
    if pre:
        _near(u, want_u, 40, "u")
    grads = {k: torch.zeros_like(a[n]) for k, n in (("post", "post_scale"), ("gate", "gate"), ("pre", "pre_scale")) if a[n] is not None}
    dx, dh = mgpt_b200.residual_norm_backward(x, h, stats, dy, du, d_post_scale=grads.get("post"), d_gate=grads.get("gate"), d_pre_scale=grads.get("pre"), **a)
    _near(dx, g["x"], 80, "dx")
    _near(dh, g["h"], 160, "dh")
    for k, v in grads.items():
        assert (v.double() - g[k]).norm() <= 200 * U * g[k].norm()
    # without the parameters' gradients
    again = mgpt_b200.residual_norm_backward(x, h, stats, dy, du, **a)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dh)


def test_rows_of_zeros_and_rows_that_are_not_finite():
    x, h, dy, du, a = _inputs(40, 64, torch.float32, 0)
    want = mgpt_b200.residual_norm(x, h, **a)
    x[3] = h[3] = 0
    h[7, 5] = float("nan")
    h[9, 0] = float("inf")
    y, u, stats = mgpt_b200.residual_norm(x, h, **a)
    assert not y[3].any() and not u[3].any()
    fine = torch.ones(40, dtype=torch.bool, device="cuda")
    fine[[3, 7, 9]] = False
    assert torch.equal(y[fine], want[0][fine]) and torch.equal(u[fine], want[1][fine])
    assert y[7].isnan().all() and y[9].isnan().any()
    dx, dh = mgpt_b200.residual_norm_backward(x, h, stats, dy, du, **a)
    assert dx[3].isfinite().all() and dh[3].isfinite().all() and dx[fine].isfinite().all()


def test_large_residuals_without_a_second_norm():
    """x near the largest number: y is finite, and the gradients, in which x is not, are what they are with a small x."""
    n, C = 9, 512
    x, h, dy, _, a = _inputs(n, C, torch.float32, 4, pre=False, seed=8)
    h.abs_()
    a["gate"].fill_(1.0)
    x.fill_(1e38)
    y, _, stats = mgpt_b200.residual_norm(x, h, **a)
    assert y.isfinite().all()
    _, _, g = _reference(x, h, dy, None, a)
    dx, dh = mgpt_b200.residual_norm_backward(x, h, stats, dy, **a)
    _near(dx, g["x"], 80, "dx")
    _near(dh, g["h"], 160, "dh")


def test_gradients_against_differences():
    """In 64 bits: the loss <y, dy> + <u, du> at parameters +- s of a direction, against the gradients' products with it."""
    n, C, per = 12, 64, 5
    x, h, dy, du, a = _inputs(n, C, torch.float32, per, seed=5)
    _, _, stats = mgpt_b200.residual_norm(x, h, **a)
    grads = [torch.zeros_like(a[k]) for k in ("post_scale", "gate", "pre_scale")]
    dx, dh = mgpt_b200.residual_norm_backward(x, h, stats, dy, du, d_post_scale=grads[0], d_gate=grads[1], d_pre_scale=grads[2], **a)
    g = torch.Generator(device="cuda").manual_seed(3)
    at = [v.double() for v in (x, h, a["post_scale"], a["gate"], a["pre_scale"])]

    def loss(v):
        X, H, po, ga, pr = v
        y = a["alpha"] * X + ga[torch.arange(n, device="cuda") // per] * H / torch.sqrt((H * H).mean(1, keepdim=True) + EPS) * po
        u = y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS) * pr
        return float((y * dy.double()).sum() + (u * du.double()).sum())

    s = 1e-5
    for i, grad in enumerate([dx, dh, *grads]):
        way = torch.randn(grad.shape, device="cuda", dtype=torch.float64, generator=g)
        up, down = (loss([v + (sign * s * way if i == j else 0) for j, v in enumerate(at)]) for sign in (1, -1))
        diff, got = (up - down) / (2 * s), float((grad.double() * way).sum())
        assert abs(diff - got) <= 1e-5 * float((grad.double() * way).abs().sum())      # 160 u, and s^2 of the third derivatives


def test_same_call_same_bits_and_any_stream():
    x, h, dy, du, a = _inputs(3000, 520, torch.bfloat16, 700, seed=6)

    def run():
        y, u, stats = mgpt_b200.residual_norm(x, h, **a)
        g = [torch.zeros_like(a[k]) for k in ("post_scale", "gate", "pre_scale")]
        return y, u, stats, *mgpt_b200.residual_norm_backward(x, h, stats, dy, du, d_post_scale=g[0], d_gate=g[1], d_pre_scale=g[2], **a), *g

    first = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = run()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_refusals():
    x, h, dy, du, a = _inputs(10, 64, torch.bfloat16, 0)
    _, _, stats = mgpt_b200.residual_norm(x, h, **a)
    norm, back = mgpt_b200.residual_norm, mgpt_b200.residual_norm_backward
    for bad in (lambda: norm(x.cpu(), h, **a), lambda: norm(x, h.float(), **a), lambda: norm(x, h[:5], **a), lambda: norm(x.half(), h.half(), **a),
                lambda: norm(x, h.T.contiguous().T, **a), lambda: norm(x, h, **{**a, "post_scale": a["post_scale"].bfloat16()}),
                lambda: norm(x, h, **{**a, "gate": a["gate"].repeat(2, 1)}), lambda: norm(x, h, **{**a, "tokens_per_gate": 3}),
                lambda: norm(x, h, **{**a, "tokens_per_gate": -1}), lambda: norm(x[:, :12].contiguous(), h[:, :12].contiguous()),
                lambda: back(x, h, stats[:, :5], dy, du, **a), lambda: back(x, h, stats, dy, None, **a), lambda: back(x, h, stats, dy.float(), du, **a),
                lambda: back(x, h, stats, dy, du, d_post_scale=torch.zeros(32, device="cuda"), **a),
                lambda: back(x, h, stats, dy, du, **{**a, "post_scale": None}, d_post_scale=torch.zeros(64, device="cuda"))):
        with pytest.raises(MoeError):
            bad()
    y, u, _ = norm(x[:0], h[:0], **a)
    assert y.shape == u.shape == (0, 64)
    y3, _, _ = norm(x.view(2, 5, 64), h.view(2, 5, 64), **{**a, "gate": a["gate"].view(64)})
    assert torch.equal(y3.view(10, 64), norm(x, h, **a)[0])
