"""What the head loss, the residual norm and the optimiser refuse, through the C ABI: before any CUDA call, so without a GPU."""
import ctypes as ct
import os
import subprocess
import sys

import pytest
import torch

from mgpt_b200 import MoeError, _lib, training
from tests.test_abi import lib  # noqa: F401

EINVAL, ENOMEM = 1, 4
P = 1 << 20                         # an address on every boundary that is asked for; never followed


def _loss(lib, x=P, io=1, w=P, targets=P, n=4, C=64, V=100, loss=P, lse=P, status=P, ws=P, size=1 << 40):
    return lib.mgpt_moe_op_head_loss(x, io, w, targets, n, C, V, loss, lse, status, ws, size, None)


def _loss_bwd(lib, x=P, io=1, w=P, targets=P, lse=P, d_loss=P, n=4, C=64, V=100, dx=P, dw=P, dw_dtype=1, status=P, ws=P, size=1 << 40):
    return lib.mgpt_moe_op_head_loss_backward(x, io, w, targets, lse, d_loss, n, C, V, dx, dw, dw_dtype, status, ws, size, None)


@pytest.mark.parametrize("bad", [dict(C=60), dict(C=0), dict(V=0), dict(n=-1), dict(io=2), dict(x=None), dict(w=None), dict(targets=None), dict(loss=None),
                                 dict(lse=None), dict(status=None), dict(x=P + 8), dict(w=P + 2), dict(ws=None), dict(ws=P + 16), dict(n=1 << 30, V=1 << 30)])
def test_head_loss_refuses(lib, bad):  # noqa: F811
    assert _loss(lib, **bad) == EINVAL
    assert lib.mgpt_moe_last_error()


@pytest.mark.parametrize("bad", [dict(C=60), dict(V=-3), dict(n=-1), dict(io=7), dict(dw_dtype=2), dict(dw=None), dict(dx=None), dict(lse=None), dict(d_loss=None),
                                 dict(x=P + 4), dict(dx=P + 8), dict(dw=P + 8), dict(ws=P + 128), dict(status=None)])
def test_head_loss_backward_refuses(lib, bad):  # noqa: F811
    assert _loss_bwd(lib, **bad) == EINVAL


def test_head_loss_workspaces(lib):  # noqa: F811
    n, C, V = 1000, 264, 50021
    size = lib.mgpt_moe_op_head_loss_workspace_bytes(n, C, V)
    assert size > 0 and _loss(lib, n=n, C=C, V=V, size=size - 1) == ENOMEM
    one = lib.mgpt_moe_op_head_loss_backward_workspace_bytes(n, C, V, 0)
    all_ = lib.mgpt_moe_op_head_loss_backward_workspace_bytes(n, C, V, 1 << 60)
    tile = 1024 * 256 * 2                                                       # dz of 256 vocabulary rows, tokens up to whole tiles
    assert all_ - one == (196 - 1) * tile                                       # 196 of them in this vocabulary
    assert _loss_bwd(lib, n=n, C=C, V=V, size=one - 1) == ENOMEM
    assert lib.mgpt_moe_op_head_loss_workspace_bytes(n, 12, V) == 0             # no such shape


def test_head_loss_without_tokens_is_no_work(lib):  # noqa: F811
    assert _loss(lib, n=0, x=None, targets=None, loss=None, lse=None, ws=None, size=0) == 0
    assert _loss_bwd(lib, n=0, x=None, targets=None, ws=None, size=0, dw_dtype=0) == 0


def test_sizes_of_workspaces_without_tokens():
    """A caller asks for the size before it looks at the number of tokens.  In a process of its own: a division by zero ends it."""
    code = ("from mgpt_b200 import _lib; lib = _lib.load(); "
            "print([lib.mgpt_moe_op_head_loss_backward_workspace_bytes(0, C, V, p) for C, V, p in ((1024, 50021, 512 << 20), (8, 1, 0), (264, 300, 1 << 60))], "
            "lib.mgpt_moe_op_head_loss_workspace_bytes(0, 64, 100), lib.mgpt_moe_op_residual_norm_backward_workspace_bytes(0, 64, 3))")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and r.stdout.split() == "[0, 0, 0] 0 0".split(), (r.returncode, r.stdout, r.stderr)


def _norm(lib, x=P, h=P, io=1, post=P, gate=P, per=0, pre=P, n=4, C=64, y=P, u=P, stats=P):
    return lib.mgpt_moe_op_residual_norm(x, h, io, post, gate, per, pre, 1.0, 1e-5, n, C, y, u, stats, None)


def _norm_bwd(lib, x=P, h=P, io=1, post=P, gate=P, per=0, pre=P, n=4, C=64, stats=P, dy=P, du=P, dx=P, dh=P, dpost=P, dgate=P, dpre=P, ws=P, size=1 << 30):
    return lib.mgpt_moe_op_residual_norm_backward(x, h, io, post, gate, per, pre, 1.0, n, C, stats, dy, du, dx, dh, dpost, dgate, dpre, ws, size, None)


@pytest.mark.parametrize("bad", [dict(C=12), dict(C=16392), dict(C=0), dict(n=-1), dict(per=-1), dict(io=3), dict(x=None), dict(h=None), dict(y=None), dict(stats=None),
                                 dict(u=None), dict(pre=None), dict(x=P + 8), dict(h=P + 2), dict(y=P + 8), dict(u=P + 8), dict(post=P + 4), dict(gate=P + 8), dict(pre=P + 4)])
def test_residual_norm_refuses(lib, bad):  # noqa: F811
    assert _norm(lib, **bad) == EINVAL


@pytest.mark.parametrize("bad", [dict(C=12), dict(n=-2), dict(per=-1), dict(dy=None), dict(du=None), dict(pre=None), dict(post=None), dict(gate=None), dict(dx=None),
                                 dict(dh=None), dict(stats=None), dict(dy=P + 8), dict(dh=P + 8), dict(ws=None), dict(ws=P + 4)])
def test_residual_norm_backward_refuses(lib, bad):  # noqa: F811
    assert _norm_bwd(lib, **bad) == EINVAL


def test_residual_norm_workspace(lib):  # noqa: F811
    size = lib.mgpt_moe_op_residual_norm_backward_workspace_bytes(1000, 64, 10)
    assert size >= 100 * 2 * 64 * 4                                             # two sums for every gate row at least
    assert _norm_bwd(lib, n=1000, per=10, size=size - 1) == ENOMEM
    assert _norm(lib, n=0, x=None, h=None, y=None, u=None, stats=None, pre=None) == 0


def test_optimiser_refuses(lib):  # noqa: F811
    h = ct.c_void_p()

    def create(bits=8, n=1, **kw):
        t = (_lib.OptimTensor * 1)(_lib.OptimTensor(**{**dict(w=P, grad=P, w_bf16=None, n=10, weight_decay=0.0, grad_dtype=0), **kw}))
        return lib.mgpt_moe_optim_create(0, t, n, bits, ct.byref(h))

    for bad in (dict(bits=16), dict(n=0), dict(n=-1), dict(w=None), dict(grad=None), dict(grad_dtype=5), dict(w=P + 2), dict(grad=P + 1), dict(w_bf16=P + 1)):
        if "n" in bad:
            assert create(n=bad["n"]) == EINVAL
        else:
            assert create(**bad) == EINVAL
        assert not h.value
    t = (_lib.OptimTensor * 3)(*[_lib.OptimTensor(P, P, None, n, 0.0, 0) for n in (1, 256, 257)])
    assert lib.mgpt_moe_optim_blocks(t, 3) == 1 + 1 + 2
    assert lib.mgpt_moe_optim_step(None, P, P, P, P, 1e-3, 0.9, 0.999, 1e-8, 1, None, 0, None, None) == EINVAL


class _OnDevice(torch.Tensor):
    """A tensor that says it is on a GPU, for calls that end before anything touches its memory."""
    is_cuda, device = property(lambda s: True), property(lambda s: torch.device("cuda", 0))


class _Records:
    """Stands for the library: keeps what its functions get, as the C types that they take."""

    def __init__(self, lib):
        self._lib, self.got = lib, {}

    def __getattr__(self, name):
        types = getattr(self._lib, name).argtypes

        def call(*args):
            self.got[name] = [t(a).value if t in (ct.c_int, ct.c_size_t) else a for t, a in zip(types, args)]
            return 0
        return call


@pytest.fixture
def recorded(lib, monkeypatch):  # noqa: F811
    r, empty = _Records(lib), torch.empty
    monkeypatch.setattr(training._lib, "load", lambda: r)
    monkeypatch.setattr(training.torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(training, "_stream", lambda device: None)
    monkeypatch.setattr(training.torch, "empty", lambda *a, device=None, **kw: empty(*a, **kw))
    return r


def _on_device(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(_OnDevice)


@pytest.mark.parametrize("per,rows,passed", [(0, 1, 0), (3, 4, 3), (10, 1, 10), (11, 1, None), (2 ** 31 - 1, 1, None), (2 ** 31, 1, None), (2 ** 32 + 3, 1, None), (2 ** 70 + 1, 1, None)])
def test_tokens_per_gate_that_int_does_not_hold(recorded, per, rows, passed):
    """Python's numbers are cut to 32 bits on their way into C: a gate of one row would be read as one of four."""
    x, h, gate = _on_device(10, 16), _on_device(10, 16), _on_device(rows, 16)
    stats = training.residual_norm(x, h, gate=gate, tokens_per_gate=per)[2]
    training.residual_norm_backward(x, h, stats.as_subclass(_OnDevice), x, gate=gate, d_gate=_on_device(rows, 16), tokens_per_gate=per)
    for name, at in (("mgpt_moe_op_residual_norm", 5), ("mgpt_moe_op_residual_norm_backward", 5), ("mgpt_moe_op_residual_norm_backward_workspace_bytes", 2)):
        got = recorded.got[name][at]
        assert got == passed if passed is not None else got == 0 or got >= 10, name


class _Huge:
    """Only the sizes of a tensor."""
    dtype, is_cuda, device = torch.bfloat16, True, torch.device("cuda", 0)

    def __init__(self, *shape, dtype=torch.bfloat16):
        self.shape, self.dtype = torch.Size(shape), dtype

    def numel(self):
        return self.shape.numel()

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return P


@pytest.mark.parametrize("n,V,C", [(2 ** 32 + 4, 100, 8), (2 ** 31, 100, 8), (4, 2 ** 32 + 100, 8), (4, 100, 2 ** 32 + 8)])
def test_sizes_that_int_does_not_hold(recorded, n, V, C):
    x, w, t, f = _Huge(n, C), _Huge(V, C), _Huge(n, dtype=torch.int32), _Huge(n, dtype=torch.float32)
    for call in (lambda: training.head_loss(x, w, t), lambda: training.head_loss_backward(x, w, t, f, f)):
        with pytest.raises(MoeError, match="out of range"):
            call()
    if V == 100:
        stats = _Huge(2, n, dtype=torch.float32)
        for call in (lambda: training.residual_norm(x, x), lambda: training.residual_norm_backward(x, x, stats, x)):
            with pytest.raises(MoeError, match="out of range"):
                call()
    assert not recorded.got
