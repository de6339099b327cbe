"""Offsets beyond 32 bits: more than 2^31 logits, and more than 2^31 kept values.  The last rows against the same rows by themselves."""
import pytest
import torch

import mgpt_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_many_logits(score):
    n, E, k = (1 << 22) + 1001, 512, 4
    z = torch.empty(n, E, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    bias = torch.linspace(-0.1, 0.1, E, device="cuda") if score == "sigmoid" else None
    how = dict(score=score, renormalise=True)
    idx, w = mgpt_b200.route(z, k, bias=bias, **how)
    dw = torch.ones(n, k, device="cuda") * torch.arange(k, device="cuda")
    dz = mgpt_b200.route_backward(z, idx, dw, **how)
    for rows in (slice(0, 300), slice(n - 1500, n)):
        part = z[rows].clone()
        i, v = mgpt_b200.route(part, k, bias=bias, **how)
        assert torch.equal(i, idx[rows]) and torch.allclose(v, w[rows], rtol=1e-6, atol=0)
        assert torch.equal(mgpt_b200.route_backward(part, i, dw[rows].clone(), **how), dz[rows])


@pytest.mark.parametrize("C", [2048, 2056])
def test_much_that_is_kept(C):
    n = (1 << 20) + 77
    x = torch.empty(n, C, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    kept = mgpt_b200.keep8(x)
    back = mgpt_b200.restore8(kept)
    y, _, stats, (x8, h8) = mgpt_b200.residual_norm(x, x, keep=True)
    assert torch.equal(x8.values, kept.values) and torch.equal(h8.exponents, kept.exponents)
    dx, dh = mgpt_b200.residual_norm_backward(x8, h8, stats, x)
    for rows in (slice(0, 100), slice(n - 100, n)):
        part = x[rows].clone()
        k = mgpt_b200.keep8(part)
        assert torch.equal(k.values, kept.values[rows]) and torch.equal(k.exponents, kept.exponents[rows]) and torch.equal(mgpt_b200.restore8(k), back[rows])
        assert torch.equal(dx[rows], part) and torch.equal(dh[rows], part)          # alpha 1, nothing normalised
