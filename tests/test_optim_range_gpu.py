"""8-bit moments of elements far below the largest of their block: a small gradient beside a large one, a gradient that comes rarely, one
that has stopped, one that jumps.

Bound of an update, in units of lr.  Let M and S be what the codes of m and of the root of v stand for, um and us their units.  A root that is not
zero is rounded down to no less than half of itself (from two steps of 2^-9 to one; more bits above) and never to zero, m is rounded up by
no more than an eighth of itself or one step of 2^-9 um.  So M/S <= 2 * (9/8) |m|/root + um/us, and um/us <= 2 max|m| / max root.  The
next update is (0.9 M + 0.1 |g|) / sqrt(0.999 S^2 + 0.001 g^2) <= 0.9005 M/S + 3.2.  With the factor of the bias corrections, at most 1 here,
and |m|/root below R (the largest exact update so far, in the same units): at most 0.9005 (2.25 + 2) R + 3.2 < 4 R + 3.2.
"""
import numpy as np
import pytest
import torch

from mgpt_b200 import AdamW

pytestmark = pytest.mark.gpu
BLOCK = 256


def _gradients(kind, ratio, n, steps):
    """Every second element is `ratio` times its neighbours' size."""
    g = torch.Generator(device="cuda").manual_seed(7)
    small = torch.arange(n, device="cuda") % 2 == 1
    size = torch.where(small, ratio, 1.0)
    for t in range(steps):
        z = torch.randn(n, device="cuda", generator=g)
        coin = torch.rand(n, device="cuda", generator=g)
        if kind == "steady":
            yield z * size
        elif kind == "rare":
            yield z * size * ((coin < 0.02) | ~small)
        elif kind == "stops":
            yield z * size * ((t < 50) | ~small)
        else:
            yield z * size * torch.where(coin < 1e-3, 1e4, 1.0)


@pytest.mark.parametrize("kind,ratio", [("steady", 1e-4), ("steady", 1e-5), ("steady", 1e-6), ("rare", 1e-3), ("rare", 1e-5), ("stops", 1e-5), ("jumps", 1.0), ("jumps", 1e-3)])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
def test_updates_stay_in_proportion(kind, ratio, grad):
    n, steps = 64 * BLOCK, 200
    w, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda", dtype=grad)
    m, v = torch.zeros(n, device="cuda", dtype=torch.float64), torch.zeros(n, device="cuda", dtype=torch.float64)
    opt = AdamW([w], [g], state_bits=8, weight_decay=0.0, seed=5)
    exact = torch.zeros((), device="cuda", dtype=torch.float64)
    moved = torch.zeros(n, dtype=torch.bool, device="cuda")
    for t, x in enumerate(_gradients(kind, ratio, n, steps), 1):
        g.copy_(x)
        w.zero_()
        opt.step(t, lr=1.0)
        d = g.double()
        m, v = 0.9 * m + 0.1 * d, 0.999 * v + 0.001 * d * d
        exact = torch.maximum(exact, ((m / (1 - 0.9 ** t)) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)).abs().max())
        moved |= g != 0
        assert float(w.abs().max()) <= 4.0 * float(exact) + 3.2, f"step {t}: an update of {float(w.abs().max()):.4g} lr, exact moments {float(exact):.3g}"
        assert torch.equal(opt.v.float() > 0, moved), f"step {t}: a root that is not zero is kept as zero"


def test_a_root_of_its_block_s_smallest_step():
    """Roots on either side of the smallest code, 2^-9 units: above it rounding is stochastic and unbiased, below it the code is 2^-9; zero is zero."""
    n = 400 * BLOCK
    g = torch.zeros(n, device="cuda")
    unit = 2.0 ** -7                                            # of the root: the block's largest is 1 (sqrt(0.001) g)
    roots = torch.tensor([2.0 ** -20, 2.0 ** -11, 0.999 * 2.0 ** -9, 1.25 * 2.0 ** -9, 1.75 * 2.0 ** -9, 2.5 * 2.0 ** -9], device="cuda") * unit
    at = g.view(-1, BLOCK)
    at[:, 0] = 1.01 / 0.001 ** 0.5
    at[:, 1:7] = roots / 0.001 ** 0.5
    opt = AdamW([torch.zeros(n, device="cuda")], [g], state_bits=8, weight_decay=0.0, seed=2)
    opt.step(1, lr=0.0)
    assert (opt.v_scale == unit).all()
    codes = opt.v.float().view(-1, BLOCK).double().cpu().numpy() * 2 ** 9
    assert (codes[:, 1:4] == 1).all() and not codes[:, 7:].any()
    for i, want, low in ((4, 1.25, 1), (5, 1.75, 1), (6, 2.5, 2)):
        assert set(codes[:, i]) <= {low, low + 1}
        assert abs(codes[:, i].mean() - want) <= 5 * 0.5 / np.sqrt(len(codes))       # 5 standard deviations of at most a half
