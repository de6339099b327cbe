"""The gradient of routing where its terms nearly cancel: one chosen expert, an expert far ahead of the others, equal gradients of the weights.

The formula in 64 bits is written in differences, as autograd of the quotient cancels there too.  With g the chosen scores, t = 1e-20, S = sum g + t,
A = sum dw g, T_j = sum_i g_i (dw_j - dw_i) and, for a softmax, rest = the sum of the scores that were not chosen (1 - sum g):

    renormalised:  dg_j = scale / S^2 (T_j + t dw_j);    softmax: dz_j = p_j scale / S^2 (T_j + t (T_j + dw_j rest)),  others -p_e scale t A / S^2
    as they are:   dg_j = scale dw_j;                    softmax: dz_j = p_j scale (T_j + dw_j rest),                  others -p_e scale A

Bounds, u = 2^-24: a score is within (4 + d) u, d the distance of its logit from the largest (the exponential's argument is rounded; a sigmoid's is
exact), a softmax's sum of E terms within 24 u, sums over k chosen within k u <= 12 u, differences and products within a few u: (64 + 4 d) u of
the sum of the terms' sizes.  BF16 results add 2^-8 of themselves.
"""
import pytest
import torch

import mgpt_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TINY = 1e-20


def _formula(z, idx, dw, score, renormalise, scale):
    """The gradient and the sum of its terms' sizes."""
    z, dw, idx = z.double(), dw.double(), idx.long()
    s = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)
    g = s.gather(1, idx)
    diff = dw[:, :, None] - dw[:, None, :]
    T, T_size = (g[:, None, :] * diff).sum(2), (g[:, None, :] * diff.abs()).sum(2)
    A, A_size = (dw * g).sum(1, keepdim=True), (dw * g).abs().sum(1, keepdim=True)
    S = g.sum(1, keepdim=True) + TINY
    over = scale / S if renormalise else torch.full_like(S, scale)
    if score == "sigmoid":
        chosen, size = (((T + TINY * dw) / S, (T_size + TINY * dw.abs()) / S) if renormalise else (dw, dw.abs()))
        one = g * torch.sigmoid(-z).gather(1, idx)
        zero = torch.zeros_like(z)
        return zero.scatter(1, idx, over * chosen * one), zero.scatter(1, idx, over * size * one)
    rest = s.scatter(1, idx, 0.0).sum(1, keepdim=True)
    if renormalise:
        chosen, size = (T + TINY * (T + dw * rest)) / S, (T_size + TINY * (dw.abs() + A_size)) / S
        other, other_size = -TINY * A / S, TINY * A_size / S
    else:
        chosen, size = T + dw * rest, T_size + dw.abs() * rest
        other, other_size = -A, A_size
    return s * over * other.expand_as(s).scatter(1, idx, chosen), s * over * other_size.expand_as(s).scatter(1, idx, size)


def _check(z, k, dw, score, renormalise, scale=1.7):
    how = dict(score=score, renormalise=renormalise, scale=scale)
    idx, _ = mgpt_b200.route(z, k, **how)
    got = mgpt_b200.route_backward(z, idx, dw, **how)
    want, size = _formula(z, idx, dw, **how)
    spread = (z.double().amax(1, keepdim=True) - z.double()).amax(1, keepdim=True) if score == "softmax" else 0.0
    bound = (64 + 4 * spread) * U * size + (2.0 ** -8 if z.dtype == torch.bfloat16 else 0.0) * want.abs() + 1e-37
    assert got.dtype == z.dtype and ((got.double() - want).abs() <= bound).all()


def _dw(n, k, seed=5):
    return torch.randn(n, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


SCORES = ["softmax", "sigmoid"]
TYPES = [torch.float32, torch.bfloat16]
# renormalised or not
WAYS = [True, False]


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("renormalise", WAYS)
@pytest.mark.parametrize("n,E", [(1, 1), (33, 7), (257, 64), (64, 155), (5000, 128), (9, 512)])
def test_one_chosen_expert(score, dtype, renormalise, n, E):
    z = (torch.randn(n, E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)) * 3.0).to(dtype)
    _check(z, 1, _dw(n, 1), score, renormalise)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("renormalise", WAYS)
@pytest.mark.parametrize("E,k", [(2, 2), (8, 2), (24, 5), (64, 8), (155, 6), (256, 12)])
def test_one_expert_ahead(score, dtype, renormalise, E, k):
    """By 0 to 60: the others' share goes from half to 1e-26."""
    n = 61
    g = torch.Generator(device="cuda").manual_seed(E)
    z = torch.randn(n, E, device="cuda", generator=g) * 0.5 - 3.0
    ahead = torch.randint(0, E, (n,), device="cuda", generator=g)
    z[torch.arange(n), ahead] = z.amax(1) + torch.arange(n, device="cuda")
    if score == "sigmoid":                                              # (sigmoids are ahead of each other below zero)
        z = z - z.amax(1, keepdim=True)
    z = z.to(dtype)
    _check(z, k, _dw(n, k), score, renormalise)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("renormalise", WAYS)
def test_equal_gradients_of_the_weights(score, dtype, renormalise):
    """No difference is left: renormalised weights have the gradient of the 1e-20, others that of what was not chosen."""
    z = _dw(300, 40, seed=2) * 2.0
    z[:100, 3] += 25.0
    z[100:200, 30:] = -50.0
    z = z.to(dtype)
    for k in (1, 4, 30):
        dw = _dw(300, 1).expand(300, k).contiguous()
        _check(z, k, dw, score, renormalise)


@pytest.mark.parametrize("renormalise", WAYS)
def test_sigmoids_about_the_constant_beside_their_sum(renormalise):
    """Sums of scores from 1e-13 to 1e-26, about 1e-20 and below it."""
    z = -30.0 - _dw(200, 16, seed=3).abs() - torch.arange(200, device="cuda")[:, None] * 0.15
    _check(z, 4, _dw(200, 4), "sigmoid", renormalise)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("ahead", [9.0, 12.0, 15.0])
def test_against_differences(score, ahead):
    """Steps of 1e-4 in 64 bits: off by h^2 / 6 of the third derivative, 2e-9 of the gradient, and by 1e-16 / h."""
    z = _dw(4, 6, seed=8) * 0.3 - 8.0
    z[:, 2] = z.amax(1) + ahead
    if score == "sigmoid":
        z = z - z.amax(1, keepdim=True)
    dw = _dw(4, 2)
    for renormalise in WAYS:
        how = dict(score=score, renormalise=renormalise, scale=1.0)
        idx, _ = mgpt_b200.route(z, 2, **how)
        got = mgpt_b200.route_backward(z, idx, dw, **how)

        def value(v):
            s = torch.sigmoid(v) if score == "sigmoid" else torch.softmax(v, 1)
            g = s.gather(1, idx.long())
            return ((g / (g.sum(1, keepdim=True) + TINY) if renormalise else g) * dw.double()).sum(1)

        for e in range(6):
            step = torch.zeros(4, 6, dtype=torch.float64, device="cuda")
            step[:, e] = 1e-4
            diff = (value(z.double() + step) - value(z.double() - step)) / 2e-4
            assert ((got[:, e].double() - diff).abs() <= 2e-5 * diff.abs() + 2e-11).all(), (renormalise, e)


def test_repeated_experts():
    """An expert that is named twice counts twice, and what is not an expert not at all, where one is far ahead too."""
    z = _dw(3, 8, seed=4)
    z[1, 5] += 12.0
    z[2, 5] += 20.0
    idx = torch.tensor([[5, 5, 1, 9]], dtype=torch.int32, device="cuda").expand(3, 4).contiguous()
    dw = torch.tensor([[1.0, 0.5, 2.0, 7.0]], device="cuda").expand(3, 4).contiguous()
    p = torch.softmax(z.double(), 1)
    p5, p1 = p[:, 5:6], p[:, 1:2]
    got = mgpt_b200.route_backward(z, idx, dw).double()
    rest = p.clone()
    rest[:, 5] = rest[:, 1] = 0.0
    rest = rest.sum(1, keepdim=True)
    A = 1.5 * p5 + 2.0 * p1
    want = -p * A
    want[:, 5:6], want[:, 1:2] = p5 * (p1 * (1.5 - 2.0) + 1.5 * rest), p1 * (p5 * (2.0 - 1.5) + 2.0 * rest)
    size = p * A
    size[:, 5:6], size[:, 1:2] = p5 * (p1 * 0.5 + 1.5 * rest), p1 * (p5 * 0.5 + 2.0 * rest)
    assert ((got - want).abs() <= (64 + 4 * 24) * U * size).all()
    got = mgpt_b200.route_backward(z, idx, dw, renormalise=True).double()
    S = 2.0 * p5 + p1
    want, size = torch.zeros_like(p), torch.full_like(p, 1e-19)
    # entries 5, 5, 1: each of 5's differs from the other by 0.5, which cancels between them
    want[:, 5:6], want[:, 1:2] = p5 / S ** 2 * p1 * (1.0 - 2.0 + 0.5 - 2.0), p1 / S ** 2 * p5 * (1.0 + 1.5)
    size[:, 5:6], size[:, 1:2] = p5 / S ** 2 * (p1 * 2.5 + p5 * 1.0), p1 / S ** 2 * p5 * 2.5
    assert ((got - want).abs() <= (64 + 4 * 24) * U * size + 1e-19).all()


def test_gradients_of_a_row_sum_to_zero():
    """Renormalised weights do not change when all chosen scores grow alike: for a softmax a row's gradients cancel, however far one expert is ahead."""
    z = _dw(200, 32, seed=6)
    z[:, 7] += torch.arange(200, device="cuda") * 0.15
    idx, _ = mgpt_b200.route(z, 4, renormalise=True)
    d = mgpt_b200.route_backward(z, idx, _dw(200, 4), renormalise=True).double()
    assert (d.sum(1).abs() <= (128 + 8 * 35) * U * d.abs().sum(1)).all()
