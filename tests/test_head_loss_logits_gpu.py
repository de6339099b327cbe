"""The gradients' logits are the loss's: the same sums, so that exp(z - lse) is off by the roundings of z and lse alone.

Bound of a certain token's gradient, with u = 2^-24.  Its target's logit z is hundreds above all others: p = 1 and dz = 0, up to
  lse       z + log of a sum of one term, exp of (z log2(e) rounded once, subtracted from z log2(e)): u|z|, and the sum's rounding u|lse|
  p         exp of z - lse by the same rounding: u|lse|, and 2 ulp of the exponential
which is 4 u |lse| + 16 u of d_loss with the rounding of dz to BF16.  (One accumulator over 2048 channels, cut off after every
16 products, ends some 2e-6 of z below the sum of its parts: 8e-4 of d_loss at z = 400.)
"""
import pytest
import torch

import mgpt_b200
from tests.test_head_loss_gpu import U, _check, _inputs, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,C", [(60, 512), (60, 640), (300, 1024), (300, 1600), (300, 2048), (520, 4096)])
def test_certain_tokens_have_no_gradient(n, C):
    V = 1500
    g = torch.Generator().manual_seed(C)
    w = (torch.randn(V, C, generator=g) * (1.5 / C ** 0.5)).bfloat16().cuda()
    t = torch.randperm(V, generator=g)[:n].int().cuda()
    x = (180.0 * w[t.long()].float()).bfloat16().float()
    d = (0.5 + torch.rand(n, generator=g)).cuda()
    z = x.double() @ w.double().T
    top = z.gather(1, t.long()[:, None])[:, 0]
    z.scatter_(1, t.long()[:, None], float("-inf"))
    assert (top - z.amax(1) > 100).all()
    loss, lse = mgpt_b200.head_loss(x, w, t)
    assert (loss.double() <= 4 * U * top).all()
    dw = torch.zeros(V, C, device="cuda")
    dx, _ = mgpt_b200.head_loss_backward(x, w, t, lse, d, dw)
    bound = (d.double() * (4 * U * top + 16 * U))[:, None] * 1.01
    over = dx.double().abs() - bound * w[t.long()].double().abs()
    assert (over <= 1e-30).all(), f"dx: {float((dx.double().abs() / w[t.long()].double().abs()).amax() / 1):.3g} of d_loss, bound {float(bound.max()):.3g}"
    over = dw[t.long()].double().abs() - bound * x.double().abs()
    assert (over <= 1e-30).all(), "dw"
    rest = torch.ones(V, dtype=torch.bool, device="cuda")
    rest[t.long()] = False
    assert dw[rest].abs().max() <= 1e-30


@pytest.mark.parametrize("n,C,V,size", [(200, 512, 1000, 100), (200, 1024, 1000, 100), (300, 1600, 3001, 30), (513, 2048, 1700, 100)])
def test_gradients_at_large_logits(n, C, V, size):
    x, w, t, d = _inputs(n, C, V, seed=6)
    x = x * size
    r = _reference(x, w, t, d)
    loss, lse = mgpt_b200.head_loss(x, w, t)
    _check(loss, r["loss"], r["err"], "loss")
    dx, dw = mgpt_b200.head_loss_backward(x, w, t, lse, d)
    _check(dx, r["dx"], r["ex"] + 2.0 ** -8 * r["dx"].abs(), "dx")
    _check(dw, r["dw"], r["ew"] + 2.0 ** -8 * r["dw"].abs(), "dw")
