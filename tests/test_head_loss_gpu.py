"""Softmax cross entropy of a vocabulary product and its gradients against the formulas in 64 bits.

Bounds, element by element, with u = 2^-24:
  logits      products of BF16 values are exact; a sum of C of them in FP32, rounded or cut off after every 16 and joined in
              parts of 512, is off by at most (C/16 + 2) * 2u of the sum of their sizes
  loss, lse   twice a logit's, and a few u of the largest logit and of the logarithm
  dz          d_loss times what twice a logit's error does to p (relative), and BF16's rounding: 2^-8 of dz (of the largest
              |d_loss| where tokens have one each: the operand is kept over it, its own rounding is relative all the same)
  dx, dw      the bound of dz summed against |w|, |x|; FP32 sums of K terms: (K/16 + 64) * 2u of the sizes; BF16 results: 2^-8 of themselves
"""
import numpy as np
import pytest
import torch

import mgpt_b200
from mgpt_b200 import MoeError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _inputs(n, C, V, ignored=0.0, seed=0, sharp=3.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, C, generator=g) * (1.5 / C ** 0.5)).bfloat16()
    t = torch.randint(0, V, (n,), generator=g, dtype=torch.int32)
    x = torch.randn(n, C, generator=g) + sharp * torch.rand(n, 1, generator=g) * w[t.long()].float()
    x = x.bfloat16().to(dtype)
    t[torch.rand(n, generator=g) < ignored] = -100
    d = torch.rand(n, generator=g) / max(n, 1)
    return x.cuda(), w.cuda(), t.cuda(), d.cuda()


def _reference(x, w, t, d=None):
    """Losses, gradients and their bounds, in 64 bits."""
    V, C = w.shape
    keep = (t >= 0) & (t < V)
    x, w, lab = x[keep].bfloat16().double(), w.double(), t[keep].long()
    z = x @ w.T
    dz_logit = (C / 16 + 2) * 2 * U * (x.abs() @ w.abs().T)
    rows = torch.arange(len(lab), device=x.device)
    lse = torch.logsumexp(z, 1) if len(lab) else z.new_zeros(0)
    top = z.abs().amax(1) if len(lab) else lse
    err = 2 * dz_logit.amax(1) + 16 * U * (top + lse.abs() + 1) if len(lab) else lse
    out = dict(keep=keep, lse=lse, loss=lse - z[rows, lab], err=err)
    if d is not None:
        d = d[keep].double()
        p = torch.exp(z - lse[:, None])
        dz = p.clone()
        dz[rows, lab] -= 1
        dz = dz * d[:, None]
        e = (2.0 ** -8) * dz.abs() + d[:, None].abs() * p * (dz_logit + err[:, None] + 16 * U * (1 + lse.abs()[:, None]))
        out.update(dx=dz @ w, dw=dz.T @ x, ex=e @ w.abs() + (V / 16 + 64) * 2 * U * (dz.abs() @ w.abs()), ew=e.T @ x.abs() + (len(lab) / 16 + 64) * 2 * U * (dz.abs().T @ x.abs()))
    return out


def _check(got, want, bound, what):
    over = (got.double() - want).abs() - bound
    assert not over.isnan().any() and (over <= 1e-30).all(), f"{what}: {float(over.max()):.3g} over its bound at {int(over.argmax())}"


SHAPES = [(1, 8, 1), (1, 64, 1000), (2, 64, 2), (16, 512, 3200), (127, 72, 255), (128, 64, 256), (129, 136, 257), (255, 1000, 511), (256, 512, 513), (257, 520, 1023),
          (300, 1032, 769), (513, 2048, 300), (700, 264, 5021)]


@pytest.mark.parametrize("n,C,V", SHAPES)
@pytest.mark.parametrize("ignored", [0.0, 0.4])
def test_loss_and_gradients(n, C, V, ignored):
    x, w, t, d = _inputs(n, C, V, ignored, seed=n + C)
    r = _reference(x, w, t, d)
    loss, lse = mgpt_b200.head_loss(x, w, t)
    k = r["keep"]
    assert not loss[~k].any() and not lse[~k].any()
    _check(loss[k], r["loss"], r["err"], "loss")
    _check(lse[k], r["lse"], r["err"], "lse")
    dx, dw = mgpt_b200.head_loss_backward(x, w, t, lse, d)
    assert not dx[~k].any()
    _check(dx[k], r["dx"], r["ex"] + 2.0 ** -8 * r["dx"].abs(), "dx")
    _check(dw, r["dw"], r["ew"] + 2.0 ** -8 * r["dw"].abs(), "dw")
    mgpt_b200.check_status()


@pytest.mark.parametrize("n,C,V,piece", [(300, 264, 5021, 0), (300, 264, 5021, 7 * 512 * 256 * 2), (40, 64, 9000, 3 * 256 * 256 * 2), (700, 520, 2100, 1 << 30)])
def test_pieces_of_the_vocabulary(n, C, V, piece):
    """Any number of pieces, a last one that is smaller, and slices of pieces where the tokens are few."""
    x, w, t, d = _inputs(n, C, V, 0.1, seed=3)
    r = _reference(x, w, t, d)
    _, lse = mgpt_b200.head_loss(x, w, t)
    dx, dw = mgpt_b200.head_loss_backward(x, w, t, lse, d, piece_bytes=piece)
    _check(dx[r["keep"]], r["dx"], r["ex"] + 2.0 ** -8 * r["dx"].abs(), "dx")
    _check(dw, r["dw"], r["ew"] + 2.0 ** -8 * r["dw"].abs(), "dw")


def test_fp32_tokens_and_added_gradients():
    n, C, V = 333, 200, 1500
    x, w, t, d = _inputs(n, C, V, 0.2, seed=9, dtype=torch.float32)
    x += 1e-3 * torch.randn_like(x)                                 # values that BF16 has not: rounded to it
    r = _reference(x, w, t, d)
    loss, lse = mgpt_b200.head_loss(x, w, t)
    _check(loss[r["keep"]], r["loss"], r["err"], "loss")
    before = torch.randn(V, C, device="cuda")
    dw = before.clone()
    dx, got = mgpt_b200.head_loss_backward(x, w, t, lse, d, dw)
    assert got is dw and dx.dtype == torch.float32
    _check(dx[r["keep"]], r["dx"], r["ex"] + 8 * U * r["dx"].abs(), "dx")
    _check(dw, before.double() + r["dw"], r["ew"] + 8 * U * (before.double().abs() + r["dw"].abs()), "dw")


def test_every_token_ignored_and_no_token():
    x, w, t, d = _inputs(50, 64, 700)
    t.fill_(-1)
    x.fill_(float("nan"))
    loss, lse = mgpt_b200.head_loss(x, w, t)
    assert not loss.any() and not lse.any()
    dw = torch.full_like(w, float("nan"))
    dx, _ = mgpt_b200.head_loss_backward(x, w, t, lse, d, dw)
    assert not dx.any() and not dw.any()
    f = torch.ones(700, 64, device="cuda")
    mgpt_b200.head_loss_backward(x, w, t, lse, d, f)
    assert (f == 1).all()
    none = mgpt_b200.head_loss(x[:0], w, t[:0])
    assert none[0].shape == none[1].shape == (0,)
    dx, dw = mgpt_b200.head_loss_backward(x[:0], w, t[:0], none[1], d[:0])
    assert dx.shape == (0, 64) and not dw.any()
    mgpt_b200.check_status()


def test_what_ignored_tokens_hold_is_not_looked_at():
    x, w, t, d = _inputs(300, 136, 900, 0.5, seed=4)
    skip = t < 0
    want = mgpt_b200.head_loss(x, w, t)
    grads = mgpt_b200.head_loss_backward(x, w, t, want[1], d)
    x[skip], d[skip] = float("nan"), float("inf")
    lse = want[1].clone()
    lse[skip] = float("nan")
    got = mgpt_b200.head_loss(x, w, t)
    again = mgpt_b200.head_loss_backward(x, w, t, lse, d)
    assert all(torch.equal(a, b) for a, b in zip(want + grads, got + again))


def test_a_token_that_is_not_finite_spoils_itself_only():
    x, w, t, d = _inputs(300, 136, 900, seed=5)
    want = mgpt_b200.head_loss(x, w, t)
    x[17, 3] = float("nan")
    got = mgpt_b200.head_loss(x, w, t)
    others = torch.arange(300, device="cuda") != 17
    assert got[0][17].isnan() and torch.equal(got[0][others], want[0][others])
    dx, _ = mgpt_b200.head_loss_backward(x, w, t, got[1], d)
    assert dx[17].isnan().all() and dx[others].isfinite().all()


def test_large_logits():
    """Logits of some hundreds: no exponential overflows, certain tokens have loss 0."""
    x, w, t, d = _inputs(200, 512, 1000, seed=6)
    x = x * 300
    r = _reference(x, w, t, d)
    loss, lse = mgpt_b200.head_loss(x, w, t)
    _check(loss, r["loss"], r["err"], "loss")
    dx, dw = mgpt_b200.head_loss_backward(x, w, t, lse, d)
    assert dx.isfinite().all() and dw.isfinite().all()


def test_targets_beyond_the_vocabulary_are_reported_and_take_no_part():
    x, w, t, d = _inputs(100, 64, 300, seed=7)
    loss, _ = mgpt_b200.head_loss(x, w, t)
    bad = t.clone()
    bad[5], bad[50] = 300, 2 ** 31 - 1
    got, _ = mgpt_b200.head_loss(x, w, bad)
    with pytest.raises(MoeError, match="beyond the vocabulary"):
        mgpt_b200.check_status()
    mgpt_b200.check_status()                                        # reported once
    loss[5] = loss[50] = 0
    assert torch.equal(got, loss)


def test_tokens_do_not_depend_on_their_neighbours():
    x, w, t, _ = _inputs(900, 264, 3000, seed=8)
    whole, _ = mgpt_b200.head_loss(x, w, t)
    for a, b in ((0, 1), (255, 257), (13, 700)):
        part, _ = mgpt_b200.head_loss(x[a:b].contiguous(), w, t[a:b].contiguous())
        assert torch.equal(part, whole[a:b])


def test_gradient_against_differences():
    """Losses of x +- h v in 64 bits against <dx, v>: what they differ by is the bound of dx and the third derivative's share."""
    n, C, V = 60, 64, 400
    x, w, t, _ = _inputs(n, C, V, seed=10)
    d = torch.ones(n, device="cuda")
    _, lse = mgpt_b200.head_loss(x, w, t)
    dx, _ = mgpt_b200.head_loss_backward(x, w, t, lse, d)
    r = _reference(x, w, t, d)
    v = torch.randn(n, C, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(1))
    h = 1e-4

    def losses(s):
        z = (x.double() + s * v) @ w.double().T
        return torch.logsumexp(z, 1) - z[torch.arange(n, device="cuda"), t.long()]

    diff = (losses(h) - losses(-h)) / (2 * h)
    zv = (v @ w.double().T).abs().amax(1)
    bound = ((r["ex"] + 2.0 ** -8 * r["dx"].abs()) * v.abs()).sum(1) + h * h * zv ** 3 * 2 + 1e-9
    assert ((dx.double() * v).sum(1) - diff).abs().le(bound).all()


def test_same_call_same_bits_and_any_stream():
    x, w, t, d = _inputs(777, 264, 5021, 0.3, seed=11)
    first = mgpt_b200.head_loss(x, w, t)
    grads = mgpt_b200.head_loss_backward(x, w, t, first[1], d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = mgpt_b200.head_loss(x, w, t)
        more = mgpt_b200.head_loss_backward(x, w, t, again[1], d)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first + grads, again + more))


def test_calls_in_a_graph():
    x, w, t, d = _inputs(300, 136, 900, 0.3, seed=12)
    want = mgpt_b200.head_loss(x, w, t)
    want += mgpt_b200.head_loss_backward(x, w, t, want[1], d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mgpt_b200.head_loss(x, w, t)
        got += mgpt_b200.head_loss_backward(x, w, t, got[1], d)
    for g in got:
        g.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals():
    x, w, t, d = _inputs(32, 64, 100)
    lse = torch.zeros(32, device="cuda")
    for bad in (lambda: mgpt_b200.head_loss(x.cpu(), w, t), lambda: mgpt_b200.head_loss(x, w.float(), t), lambda: mgpt_b200.head_loss(x, w, t.long()),
                lambda: mgpt_b200.head_loss(x[:, :32], w, t), lambda: mgpt_b200.head_loss(x.T.contiguous().T, w, t), lambda: mgpt_b200.head_loss(x, w.T.contiguous().T, t),
                lambda: mgpt_b200.head_loss(x, w, t[:31]), lambda: mgpt_b200.head_loss(x.half(), w, t), lambda: mgpt_b200.head_loss(x, w, t.cpu()),
                lambda: mgpt_b200.head_loss_backward(x, w, t, lse.double(), d), lambda: mgpt_b200.head_loss_backward(x, w, t, lse, d[:5]),
                lambda: mgpt_b200.head_loss_backward(x, w, t, lse, d, torch.zeros(100, 32, device="cuda")),
                lambda: mgpt_b200.head_loss_backward(x, w, t, lse, d, torch.zeros(100, 64, device="cuda", dtype=torch.float16)),
                lambda: mgpt_b200.head_loss(torch.zeros(32 * 64 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(32, 64), w, t),
                lambda: mgpt_b200.head_loss(torch.zeros(32, 60, device="cuda", dtype=torch.bfloat16), torch.zeros(100, 60, device="cuda", dtype=torch.bfloat16), t)):
        with pytest.raises(MoeError):
            bad()
    assert np.isfinite(mgpt_b200.head_loss(x.view(4, 8, 64), w, t.view(4, 8))[0].cpu().numpy()).all()


@pytest.mark.parametrize("C", [8, 64, 128, 256, 384, 512, 520, 1024, 1600])
def test_many_tiles_per_pair_of_sms(C):
    """Hundreds of tiles per pair, at widths where the products hide the exponentials and where they do not: warps that share a row
    may be an item apart.  Every call gives the same bits, and they are right."""
    n, V = 2100, 20011
    x, w, t, d = _inputs(n, C, V, 0.02, seed=C)
    first = mgpt_b200.head_loss(x, w, t)
    grads = mgpt_b200.head_loss_backward(x, w, t, first[1], d)
    for _ in range(6):
        again = mgpt_b200.head_loss(x, w, t)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        more = mgpt_b200.head_loss_backward(x, w, t, again[1], d)
        assert torch.equal(grads[0], more[0]) and torch.equal(grads[1], more[1])
    mgpt_b200.check_status()
    some = torch.arange(0, n, 7, device="cuda")
    r = _reference(x[some], w, t[some])
    _check(first[0][some][r["keep"]], r["loss"], r["err"], "loss")
    _check(first[1][some][r["keep"]], r["lse"], r["err"], "lse")
