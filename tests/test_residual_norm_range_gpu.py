"""The norms of rows whose squares no longer fit FP32: the values are finite, and so are the results, to the bounds of ordinary rows.

Such a row is summed again at 2^-72 of its size: two more roundings of a result, and up to 2^-22 of a root that is itself below FP32's smallest
normal number.  Both are within the 40 roundings (160 for dh) that the ordinary rows' bounds count.
"""
import pytest
import torch

import mgpt_b200
from tests.test_residual_norm_gpu import EPS, U, _inputs, _near, _reference

pytestmark = pytest.mark.gpu


def _sized(n, lo, hi):
    """A factor per token, powers of two from 2^lo to 2^hi."""
    return torch.exp2(torch.linspace(lo, hi, n, device="cuda").round())[:, None]


@pytest.mark.parametrize("n,C,dtype,per", [(40, 64, torch.float32, 0), (40, 512, torch.bfloat16, 7), (40, 1024, torch.float32, 0), (40, 2048, torch.bfloat16, 0), (33, 3000, torch.float32, 5),
                                           (33, 4104, torch.bfloat16, 0), (20, 8200, torch.float32, 3), (9, 16384, torch.bfloat16, 0)])
@pytest.mark.parametrize("big", ["h", "x", "both"])
def test_rows_whose_squares_overflow(n, C, dtype, per, big):
    x, h, dy, du, a = _inputs(n, C, dtype, per, seed=n + C)
    if big != "x":
        h = (h.float() * _sized(n, 50, 120)).to(dtype)
    if big != "h":
        x = (x.float() * _sized(n, 120, 50)).to(dtype)
    assert x.isfinite().all() and h.isfinite().all()
    y, u, stats = mgpt_b200.residual_norm(x, h, **a)
    want_y, want_u, g = _reference(x, h, dy, du, a)
    _near(y, want_y, 40, "y")
    _near(u, want_u, 40, "u")
    grads = {k: torch.zeros_like(a[p]) for k, p in (("post", "post_scale"), ("gate", "gate"), ("pre", "pre_scale"))}
    dx, dh = mgpt_b200.residual_norm_backward(x, h, stats, dy, du, d_post_scale=grads["post"], d_gate=grads["gate"], d_pre_scale=grads["pre"], **a)
    _near(dx, g["x"], 80, "dx")
    _near(dh, g["h"], 160, "dh")
    for k in grads:
        size = (n ** 0.5 + 1) * (g[k].abs().mean() + g[k].abs()) * 4
        over = (grads[k].double() - g[k]).abs() - (n / 2 + 64) * U * size
        assert (over <= 0).all(), f"d_{k}: {float(over.max()):.3g} over"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_large_value_in_a_row_and_other_rows(dtype):
    """The row's other values are what they are beside it; rows without one have the bits that they have alone."""
    x, h, _, _, a = _inputs(50, 320, dtype, 0, seed=3)
    want = mgpt_b200.residual_norm(x, h, **a)
    h2 = h.clone()
    h2[::7, 5] = 3e25
    y, u, stats = mgpt_b200.residual_norm(x, h2, **a)
    ref_y, ref_u, _ = _reference(x, h2, x, x, a)
    _near(y, ref_y, 40, "y")
    _near(u, ref_u, 40, "u")
    other = torch.arange(50, device="cuda") % 7 != 0
    assert torch.equal(y[other], want[0][other]) and torch.equal(u[other], want[1][other]) and torch.equal(stats[:, other], want[2][:, other])


@pytest.mark.parametrize("post,gate,pre", [(1, 0, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
def test_parts_that_are_absent(post, gate, pre):
    x, h, _, _, a = _inputs(30, 136, torch.float32, 0, post, gate, pre, seed=2)
    x, h = x * _sized(30, 100, 40), h * _sized(30, 40, 100)
    y, u, _ = mgpt_b200.residual_norm(x, h, **a)
    want_y, want_u, _ = _reference(x, h, x, x if pre else None, a)
    _near(y, want_y, 40, "y")
    if pre:
        _near(u, want_u, 40, "u")


def test_infinities_spoil_their_own_element_only():
    """1/sqrt of an infinite sum is 0: an infinity in h makes its own element NaN, one in y its own element of u."""
    x, h, _, _, a = _inputs(20, 64, torch.float32, 0, seed=4)
    h[3, 7], x[5, 9] = float("inf"), float("-inf")
    y, u, _ = mgpt_b200.residual_norm(x, h, **a)
    r = torch.where(h.isinf().any(1, keepdim=True), 0.0, 1.0 / torch.sqrt(h.square().mean(1, keepdim=True) + EPS))
    bad = torch.zeros_like(h, dtype=torch.bool)
    bad[3, 7] = True
    plain = a["alpha"] * x + a["gate"] * (h * r * a["post_scale"])
    assert torch.equal(y.isnan(), bad) and y[5, 9] == float("-inf")
    assert torch.equal(y.isfinite(), plain.isfinite())
    assert u[3].isnan().all() and u[5, 9].isnan() and (u[5, :9] == 0).all() and (u[5, 10:] == 0).all()
