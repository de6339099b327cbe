"""What routing and the kept activations refuse, through the C ABI: before any CUDA call, so without a GPU."""
import ctypes as ct
import math

import pytest
import torch

from mgpt_b200 import Kept8, MoeError, _lib, keep8, restore8, route, route_backward
from tests.test_abi import lib  # noqa: F401

EINVAL = 1
P = 1 << 20                         # an address on every boundary that is asked for; never followed


def _routing(score=1, groups=4, top_groups=2, group_top=2, renormalise=1, scale=1.0, bias=P):
    return _lib.Routing(score, groups, top_groups, group_top, renormalise, scale, bias)


def _route(lib, logits=P, io=0, n=4, E=64, k=6, idx=P, w=P, counts=P, r=None, **how):
    r = ct.byref(_routing(**how)) if r is None else r
    return lib.mgpt_moe_op_route(logits, io, n, E, k, r, idx, w, counts, None)


def _route_bwd(lib, logits=P, io=0, idx=P, dw=P, n=4, E=64, k=6, dz=P, **how):
    return lib.mgpt_moe_op_route_backward(logits, io, idx, dw, n, E, k, ct.byref(_routing(**how)), dz, None)


BAD = [dict(n=-1), dict(E=0), dict(E=516), dict(k=0), dict(k=33), dict(E=4, k=5, groups=1, top_groups=1), dict(io=2), dict(logits=None), dict(logits=P + 2), dict(score=2), dict(score=-1),
       dict(groups=0), dict(groups=-4), dict(groups=3), dict(groups=64), dict(top_groups=0), dict(top_groups=5), dict(group_top=0), dict(group_top=3),
       dict(groups=32, top_groups=2, k=5), dict(scale=math.nan), dict(scale=math.inf), dict(bias=P + 2), dict(n=1 << 29, k=4)]


@pytest.mark.parametrize("bad", BAD + [dict(idx=None), dict(w=None), dict(idx=P + 1), dict(w=P + 2), dict(counts=P + 2), dict(io=1, logits=P + 1)])
def test_route_refuses(lib, bad):  # noqa: F811
    assert _route(lib, **bad) == EINVAL
    assert lib.mgpt_moe_last_error()


@pytest.mark.parametrize("bad", BAD + [dict(idx=None), dict(dw=None), dict(dz=None), dict(idx=P + 1), dict(dw=P + 2), dict(dz=P + 2), dict(io=1, dz=P + 1)])
def test_route_backward_refuses(lib, bad):  # noqa: F811
    assert _route_bwd(lib, **bad) == EINVAL


def test_no_tokens_are_no_work(lib):  # noqa: F811
    assert _route(lib, n=0, logits=None, idx=None, w=None) == 0
    assert _route_bwd(lib, n=0, logits=None, idx=None, dw=None, dz=None) == 0
    assert lib.mgpt_moe_op_keep8(None, 1, 0, 64, None, None, None) == 0
    assert lib.mgpt_moe_op_restore8(None, None, 0, 64, None, 1, None) == 0


def test_null_routing(lib):  # noqa: F811
    assert lib.mgpt_moe_op_route(P, 0, 4, 64, 6, None, P, P, None, None) == EINVAL
    assert lib.mgpt_moe_set_routing(None, ct.byref(_routing())) == EINVAL


@pytest.mark.parametrize("bad", [dict(C=60), dict(C=0), dict(n=-1), dict(n=(1 << 30) + 1), dict(io=2), dict(x=None), dict(v=None), dict(e=None), dict(x=P + 8), dict(v=P + 4)])
def test_keep_and_restore_refuse(lib, bad):  # noqa: F811
    a = dict(x=P, io=1, n=4, C=64, v=P, e=P, **{}) | bad
    assert lib.mgpt_moe_op_keep8(a["x"], a["io"], a["n"], a["C"], a["v"], a["e"], None) == EINVAL
    assert lib.mgpt_moe_op_restore8(a["v"], a["e"], a["n"], a["C"], a["x"], a["io"], None) == EINVAL


@pytest.mark.parametrize("bad", [dict(x=None), dict(h=P + 8), dict(xv=None), dict(hv=None), dict(xe=None), dict(he=None), dict(xv=P + 4), dict(hv=P + 4), dict(xe=P + 2), dict(he=P + 1), dict(C=12), dict(io=3), dict(u=None)])
def test_residual_norm_keep_refuses(lib, bad):  # noqa: F811
    a = dict(x=P, h=P, io=1, C=64, u=P, xv=P, xe=P, hv=P, he=P) | bad
    assert lib.mgpt_moe_op_residual_norm_keep(a["x"], a["h"], a["io"], P, P, 0, P, 1.0, 1e-5, 4, a["C"], P, a["u"], P, a["xv"], a["xe"], a["hv"], a["he"], None) == EINVAL


@pytest.mark.parametrize("bad", [dict(xv=None), dict(hv=None), dict(xe=None), dict(he=None), dict(xv=P + 4), dict(hv=P + 4), dict(xe=P + 1), dict(he=P + 2), dict(C=12), dict(dy=None), dict(du=None), dict(dx=None), dict(ws=None)])
def test_residual_norm_backward_kept_refuses(lib, bad):  # noqa: F811
    a = dict(xv=P, xe=P, hv=P, he=P, C=64, dy=P, du=P, dx=P, ws=P) | bad
    assert lib.mgpt_moe_op_residual_norm_backward_kept(a["xv"], a["xe"], a["hv"], a["he"], 1, P, P, 0, P, 1.0, 4, a["C"], P, a["dy"], a["du"], a["dx"], P, P, P, P, a["ws"], 1 << 30, None) == EINVAL


def test_no_cpu_path():
    x = torch.zeros(2, 32)
    for call in (lambda: route(x, 2), lambda: route_backward(x, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2)), lambda: keep8(x),
                 lambda: restore8(Kept8(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8), torch.float32))):
        with pytest.raises(MoeError, match="CUDA"):
            call()
