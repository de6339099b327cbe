"""Whose logits hold a NaN (softmax: or +inf) has weights of NaN, and experts as documented all the same: those that are out last, whatever the
other tokens of the call are."""
import math

import pytest
import torch

import mgpt_b200
from tests.test_routing_gpu import _bias, _logits, _reference

pytestmark = pytest.mark.gpu


def _expected(z, k, score, bias=None, groups=1, top_groups=None, **how):
    """With logits of +inf a softmax's scores are 1 / m for the m of them and 0 for the others, the limit of m large ones: logits of 0 and about -1e4 have
    those scores in 64 bits.  (Without a bias the order is that of the logits.)"""
    z = z.double()
    if score == "softmax" and (bias is not None or top_groups not in (None, groups)):
        finite = torch.where(z == math.inf, 0.0, torch.where(z > -math.inf, z - 1e4, z))
        z = torch.where((z == math.inf).any(1, keepdim=True), finite, z)
    return _reference(z, k, score=score, bias=bias, groups=groups, top_groups=top_groups, **how)[0]


def _rows(n, E, dtype, seed):
    """Tokens of all kinds, every other one as usual."""
    z = _logits(n, E, dtype, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    kind = torch.arange(n, device="cuda") % 16
    some = torch.rand(n, E, device="cuda", generator=g)
    one = torch.zeros(n, E, dtype=torch.bool, device="cuda")
    one[torch.arange(n), torch.randint(0, E, (n,), device="cuda", generator=g)] = True
    nan, inf = torch.tensor(math.nan, dtype=dtype, device="cuda"), torch.tensor(math.inf, dtype=dtype, device="cuda")

    def put(k, where, value):
        z[:] = torch.where((kind == k)[:, None] & where, value, z)

    put(1, one, nan)
    put(3, some < 0.5, nan)
    put(5, some < 2.0, nan)
    put(7, one, nan)
    put(7, some < 0.3, -inf)
    put(9, one, inf)
    put(11, some < 0.2, inf)
    put(11, one, nan)
    put(13, ~one, nan)
    put(14, some < 2.0, -inf)                                           # beside them: nothing left, and all alike
    put(15, some < 2.0, torch.zeros_like(inf))
    return z


def _check(z, k, **how):
    idx, w = mgpt_b200.route(z, k, **how)
    want = _expected(z, k, **how)
    assert torch.equal(idx.cpu().long(), want)
    bad = torch.isnan(z).any(1) | ((z == math.inf).any(1) if how["score"] == "softmax" else False)
    assert torch.equal(torch.isnan(w).all(1), bad) and not torch.isnan(w[~bad]).any()
    return idx


SHAPES = [(64, 2, 1, 1, 1), (100, 8, 3, 1, 1), (100, 16, 3, 4, 2), (65, 33, 4, 1, 1), (97, 64, 4, 1, 1), (97, 64, 6, 8, 3), (80, 155, 6, 5, 3), (80, 256, 8, 8, 4), (33, 512, 12, 16, 5),
          (3000, 128, 8, 1, 1), (3000, 128, 8, 8, 4), (5000, 64, 4, 1, 1)]


@pytest.mark.parametrize("n,E,k,groups,top_groups", SHAPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_choice(n, E, k, groups, top_groups, score, dtype):
    z = _rows(n, E, dtype, seed=E)
    for bias in (None, _bias(E, seed=E)):
        _check(z, k, score=score, bias=bias, groups=groups, top_groups=top_groups, renormalise=True)


@pytest.mark.parametrize("E", [8, 64, 128, 256])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_choice_does_not_depend_on_the_other_tokens(score, E):
    """A token with a NaN alone, beside usual ones and beside one with nothing left."""
    z = _logits(40, E, seed=E)
    z[::4, 1] = math.nan
    for bias in (None, _bias(E, seed=3)):
        how = dict(score=score, bias=bias)
        alone = torch.cat([mgpt_b200.route(z[i:i + 1], 3, **how)[0] for i in range(40)])
        assert torch.equal(mgpt_b200.route(z, 3, **how)[0], alone)
        beside = z.clone()
        beside[1::4] = -math.inf
        idx = mgpt_b200.route(beside, 3, **how)[0]
        rows = torch.arange(40, device="cuda") % 4 != 1
        assert torch.equal(idx[rows], alone[rows]) and (idx[::4] != 1).all()
        counts = torch.zeros(E, dtype=torch.int32, device="cuda")
        mgpt_b200.route(beside, 3, counts=counts, **how)
        assert torch.equal(counts, torch.bincount(idx.flatten().long(), minlength=E).int())
