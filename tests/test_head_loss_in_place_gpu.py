"""Tokens that are read where they lie (BF16, a multiple of 16 channels, none ignored, whole tiles or many of them), and the same tokens from the packed
copy, which one more token that is ignored makes the call take: the same bits, and the right ones."""
import pytest
import torch

import mgpt_b200
from tests.test_head_loss_gpu import _check, _inputs, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,C,V", [(512, 512, 1500), (512, 1040, 1500), (768, 512, 777), (768, 1040, 1500), (2100, 64, 1500), (2100, 1024, 1500), (2049, 528, 1000), (2303, 16, 300),
                                   (2560, 2048, 1100)])
def test_in_place_and_packed(n, C, V):
    x, w, t, d = _inputs(n, C, V, seed=n + C)
    r = _reference(x, w, t, d)
    loss, lse = mgpt_b200.head_loss(x, w, t)
    _check(loss, r["loss"], r["err"], "loss")
    _check(lse, r["lse"], r["err"], "lse")
    dx, dw = mgpt_b200.head_loss_backward(x, w, t, lse, d)
    _check(dx, r["dx"], r["ex"] + 2.0 ** -8 * r["dx"].abs(), "dx")
    _check(dw, r["dw"], r["ew"] + 2.0 ** -8 * r["dw"].abs(), "dw")
    for at in (n, 300):                                         # behind the others, and among them
        def more(a, v):
            return torch.cat([a[:at], torch.full_like(a[:1], v), a[at:]])

        kept = torch.arange(n + 1, device="cuda") != at
        loss1, lse1 = mgpt_b200.head_loss(more(x, float("nan")), w, more(t, -100))
        dx1, dw1 = mgpt_b200.head_loss_backward(more(x, float("nan")), w, more(t, -100), lse1, more(d, float("inf")))
        assert torch.equal(loss1[kept], loss) and torch.equal(lse1[kept], lse) and not loss1[at] and not lse1[at]
        assert torch.equal(dx1[kept], dx) and torch.equal(dw1, dw) and not dx1[at].any()
    mgpt_b200.check_status()


@pytest.mark.parametrize("n", [2, 100, 130, 256])
def test_one_tile_whose_ignored_tokens_are_read(n):
    """What they hold stays in their own rows."""
    x, w, t, _ = _inputs(n, 200, 900, seed=n)
    want = mgpt_b200.head_loss(x, w, t)
    out = torch.arange(n, device="cuda") % 3 == 1
    x[out], t[out] = float("nan"), -1
    loss, lse = mgpt_b200.head_loss(x, w, t)
    assert torch.equal(loss[~out], want[0][~out]) and torch.equal(lse[~out], want[1][~out]) and not loss[out].any() and not lse[out].any()
