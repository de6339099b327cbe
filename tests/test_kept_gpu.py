"""Activations kept in 8 bits: the format bit for bit against its definition in 64 bits, and the norms' gradients from them.

The norms with kept x and h do the arithmetic of the calls on tensors: their results are compared bit for bit with those of the tensors that
:func:`restore8` gives, whose own accuracy is tested against 64 bits elsewhere, and with the formulas in 64 bits here.
"""
import math

import pytest
import torch

import mgpt_b200
from mgpt_b200 import Kept8, MoeError

pytestmark = pytest.mark.gpu
EPS = 1e-5
U = 2.0 ** -24


def _power(e):
    """2^e to the last bit (torch's power of a tensor is not, on the device)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _definition(x):
    """Whole numbers and exponents of [n, C], in 64 bits."""
    n, C = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -C % 32)).view(n, -1, 32)
    largest = x.abs().amax(2)
    finite = torch.isfinite(x).all(2)
    e = torch.full_like(largest, -126.0)
    for k in range(-126, 121):                                          # the least power that will do
        e = torch.where(torch.round(largest / 2.0 ** k) > 127.0, float(k + 1), e)
    q = torch.round(x / _power(e)[:, :, None]).clamp(-127.0, 127.0)     # (2^121 at most: 64 * 2^122 is no FP32 number)
    return torch.where(finite[:, :, None], q, 0.0).view(n, -1)[:, :C], torch.where(finite, e + 127, 255.0), finite


def _x(n, C, dtype, seed=0, wide=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    sizes = torch.exp(torch.randn(C, device="cuda", generator=g) * 2.0) if wide else 1.0
    return (torch.randn(n, C, device="cuda", generator=g) * sizes).to(dtype)


SHAPES = [(1, 8), (3, 24), (1, 40), (5, 32), (2, 64), (17, 72), (100, 96), (3, 1000), (1, 1024), (65, 1032), (7, 2048), (300, 264), (9, 4104), (2, 16384), (5001, 40), (4097, 256)]


@pytest.mark.parametrize("n,C", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_kept_and_restored(n, C, dtype):
    x = _x(n, C, dtype, seed=n + C)
    kept = mgpt_b200.keep8(x)
    q, e, _ = _definition(x)
    assert kept.shape == x.shape and kept.dtype == dtype and kept.exponents.shape == (n, -(-C // 32)) and kept.nbytes == n * (C + -(-C // 32))
    assert torch.equal(kept.values.double(), q) and torch.equal(kept.exponents.double(), e)
    unit = _power(e - 127.0).repeat_interleave(32, 1)[:, :C]
    for to in (None, torch.float32, torch.bfloat16):
        back = mgpt_b200.restore8(kept, to)
        assert back.dtype == (to or dtype) and torch.equal(back.double(), q * unit)
    assert ((q * unit - x.double()).abs() <= unit / 2).all()            # half a unit
    again = mgpt_b200.keep8(mgpt_b200.restore8(kept))
    assert torch.equal(mgpt_b200.restore8(again), mgpt_b200.restore8(kept))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_ends_of_the_range(dtype):
    top = torch.finfo(dtype).max
    x = torch.zeros(12, 64, dtype=dtype, device="cuda")
    x[0, 3], x[0, 40] = top, -top
    x[1] = 2.0 ** -126                                                  # the smallest normal number
    x[2] = 2.0 ** -133                                                  # below it
    x[3, 5] = 2.0 ** -119
    x[4, 0], x[4, 1], x[4, 2] = 127.0, 0.5, 1.5                         # halves go to even
    x[5, 0], x[5, 1] = 127.5, 1.0                                       # would round to 128: the next power
    x[6, 0], x[6, 33] = math.nan, 1.0
    x[7, 31], x[7, 32] = math.inf, -math.inf
    x[8, 0], x[8, 1] = 255.0, -255.0
    x[9] = -0.0
    x[10, 0], x[10, 1] = 254.0, -1.0
    kept = mgpt_b200.keep8(x)
    q, e, finite = _definition(x)
    assert torch.equal(kept.exponents.double(), e)
    inside = finite.repeat_interleave(32, 1)
    assert torch.equal(kept.values.double()[inside], q[inside])
    back = mgpt_b200.restore8(kept)
    assert torch.isnan(back[~inside]).all() and torch.isfinite(back[inside]).all()
    assert (back[0, 3].double() - top).abs() <= 2.0 ** 121 and back[0, 0] == 0     # 127 units for just under 128: one unit, by arithmetic


def test_nothing_beside_it_is_written():
    x = _x(33, 72, torch.bfloat16)
    values, exponents = torch.full((35, 72), 77, dtype=torch.int8, device="cuda"), torch.full((35, 3), 77, dtype=torch.uint8, device="cuda")
    from mgpt_b200 import _lib
    lib = _lib.load()
    _lib.check(lib.mgpt_moe_op_keep8(x.data_ptr(), 1, 33, 72, values[1:].data_ptr(), exponents[1:].data_ptr(), torch.cuda.current_stream().cuda_stream))
    kept = mgpt_b200.keep8(x)
    assert torch.equal(values[1:34], kept.values) and torch.equal(exponents[1:34], kept.exponents)
    assert (values[[0, 34]] == 77).all() and (exponents[[0, 34]] == 77).all()
    out = torch.full((35, 72), 5.0, device="cuda")
    _lib.check(lib.mgpt_moe_op_restore8(kept.values.data_ptr(), kept.exponents.data_ptr(), 33, 72, out[1:].data_ptr(), 0, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[1:34], mgpt_b200.restore8(kept, torch.float32)) and (out[[0, 34]] == 5).all()


def _args(n, C, per, post=True, gate=True, pre=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)                                             # noqa: E731
    rows = -(-n // per) if per else 1
    return dict(post_scale=1 + 0.1 * r(C) if post else None, gate=0.5 * r(rows, C) if gate else None, pre_scale=1 + 0.1 * r(C) if pre else None,
                alpha=0.8, eps=EPS, tokens_per_gate=per)


def _grads(a):
    return {f"d_{k}": torch.zeros_like(a[k]) for k in ("post_scale", "gate", "pre_scale") if a[k] is not None}


CASES = [(1, 8, torch.float32, 0), (3, 64, torch.bfloat16, 2), (8, 1024, torch.bfloat16, 0), (1021, 320, torch.float32, 256), (777, 1000, torch.bfloat16, 100),
         (300, 2048, torch.bfloat16, 0), (300, 2056, torch.float32, 7), (33, 4096, torch.bfloat16, 1), (33, 4104, torch.bfloat16, 0), (20, 8200, torch.float32, 3),
         (9, 16384, torch.bfloat16, 0), (9, 16376, torch.float32, 0), (5000, 264, torch.bfloat16, 5000), (2500, 40, torch.float32, 3), (700, 1032, torch.float32, 0)]


@pytest.mark.parametrize("n,C,dtype,per", CASES)
def test_norms_keep_and_take(n, C, dtype, per):
    a = _args(n, C, per, seed=n)
    x, h = _x(n, C, dtype, seed=1), _x(n, C, dtype, seed=2)
    dy, du = _x(n, C, dtype, seed=3, wide=False), _x(n, C, dtype, seed=4, wide=False)
    y, u, stats = mgpt_b200.residual_norm(x, h, **a)
    ky, ku, kstats, (x8, h8) = mgpt_b200.residual_norm(x, h, keep=True, **a)
    assert torch.equal(y, ky) and torch.equal(u, ku) and torch.equal(stats, kstats)
    for kept, t in ((x8, x), (h8, h)):
        want = mgpt_b200.keep8(t)
        assert isinstance(kept, Kept8) and torch.equal(kept.values, want.values) and torch.equal(kept.exponents, want.exponents)
    g, gk = _grads(a), _grads(a)
    xr, hr = mgpt_b200.restore8(x8), mgpt_b200.restore8(h8)
    dx, dh = mgpt_b200.residual_norm_backward(xr, hr, stats, dy, du, **g, **a)
    kdx, kdh = mgpt_b200.residual_norm_backward(x8, h8, stats, dy, du, **gk, **a)
    assert torch.equal(dx, kdx) and torch.equal(dh, kdh)
    for k in g:
        assert torch.equal(g[k], gk[k])


@pytest.mark.parametrize("post,gate,pre", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)])
def test_parts_that_are_absent(post, gate, pre):
    n, C = 70, 136
    a = _args(n, C, 20 if gate else 0, post, gate, pre)
    x, h, dy = (_x(n, C, torch.bfloat16, seed=s) for s in (1, 2, 3))
    du = _x(n, C, torch.bfloat16, seed=4) if pre else None
    y, u, stats, (x8, h8) = mgpt_b200.residual_norm(x, h, keep=True, **a)
    assert (u is None) == (not pre)
    g, gk = _grads(a), _grads(a)
    want = mgpt_b200.residual_norm_backward(mgpt_b200.restore8(x8), mgpt_b200.restore8(h8), stats, dy, du, **g, **a)
    got = mgpt_b200.residual_norm_backward(x8, h8, stats, dy, du, **gk, **a)
    assert all(torch.equal(p, q) for p, q in zip(want, got)) and all(torch.equal(g[k], gk[k]) for k in g)


def test_gradients_are_the_formulas_at_what_was_kept():
    """Against 64 bits: about 40 roundings in a value and 160 where terms of the row's size cancel, each at most 2^-24 of the row's largest."""
    n, C = 203, 1032
    a = _args(n, C, 50, seed=5)
    x, h = _x(n, C, torch.float32, seed=1, wide=False), _x(n, C, torch.float32, seed=2, wide=False)
    dy, du = _x(n, C, torch.float32, seed=3, wide=False), _x(n, C, torch.float32, seed=4, wide=False)
    _, _, stats, (x8, h8) = mgpt_b200.residual_norm(x, h, keep=True, **a)
    g = _grads(a)
    dx, dh = mgpt_b200.residual_norm_backward(x8, h8, stats, dy, du, **g, **a)

    def definition(t):
        q, e, _ = _definition(t)
        return q * _power(e - 127.0).repeat_interleave(32, 1)[:, :C]

    gate = a["gate"].double()[torch.arange(n, device="cuda") // 50]
    post, pre = a["post_scale"].double(), a["pre_scale"].double()
    r1 = 1 / torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + EPS)
    yy = 0.8 * x.double() + gate * (h.double() * r1 * post)
    r2 = 1 / torch.sqrt((yy ** 2).mean(1, keepdim=True) + EPS)
    hh = definition(h) * r1
    yh = (0.8 * definition(x) + gate * hh * post) * r2
    d = du.double() * pre
    D = dy.double() + r2 * (d - yh * (d * yh).mean(1, keepdim=True))
    e = D * gate * post
    want = dict(dx=(0.8 * D, dx), dh=(r1 * (e - hh * (e * hh).mean(1, keepdim=True)), dh))
    for k, (w, got) in want.items():
        assert ((got.double() - w).abs() <= 160 * U * w.abs().amax(1, keepdim=True)).all(), k
    rows = torch.arange(n, device="cuda") // 50
    sums = dict(d_post_scale=D * gate * hh, d_pre_scale=du.double() * yh)
    for k, terms in sums.items():
        assert ((g[k].double() - terms.sum(0)).abs() <= (n / 2 + 128) * U * terms.abs().sum(0)).all(), k
    terms = D * hh * post
    d_gate = torch.zeros_like(a["gate"], dtype=torch.float64).index_add_(0, rows, terms)
    assert ((g["d_gate"].double() - d_gate).abs() <= (n / 2 + 128) * U * torch.zeros_like(d_gate).index_add_(0, rows, terms.abs())).all()


def test_a_value_that_is_not_finite_shows_in_the_gradients():
    x, h, dy = (_x(4, 64, torch.bfloat16, seed=s) for s in (1, 2, 3))
    x[1, 40] = math.inf
    _, _, stats, (x8, h8) = mgpt_b200.residual_norm(x, h, keep=True, pre_scale=torch.ones(64, device="cuda"))
    dx, dh = mgpt_b200.residual_norm_backward(x8, h8, stats, dy, dy, pre_scale=torch.ones(64, device="cuda"))
    assert torch.isnan(dx[1]).any() and torch.isfinite(dx[[0, 2, 3]]).all() and torch.isfinite(dh[[0, 2, 3]]).all()


def test_shapes_streams_and_graphs():
    x = _x(30, 64, torch.bfloat16).view(2, 3, 5, 64)
    kept = mgpt_b200.keep8(x)
    assert kept.values.shape == x.shape and kept.exponents.shape == (2, 3, 5, 2)
    one = mgpt_b200.keep8(x[1, 2, 4])
    assert torch.equal(one.values, kept.values[1, 2, 4]) and torch.equal(one.exponents, kept.exponents[1, 2, 4])
    nothing = mgpt_b200.keep8(x[:0])
    assert mgpt_b200.restore8(nothing).shape == (0, 3, 5, 64)
    y, u, stats, (x8, h8) = mgpt_b200.residual_norm(x[:0], x[:0], keep=True)
    assert x8.shape == (0, 3, 5, 64) and mgpt_b200.residual_norm_backward(x8, h8, stats, x[:0])[0].shape == (0, 3, 5, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = mgpt_b200.restore8(mgpt_b200.keep8(x))
    side.synchronize()
    assert torch.equal(other, mgpt_b200.restore8(kept))
    graph = torch.cuda.CUDAGraph()
    pre = torch.ones(64, device="cuda")
    with torch.cuda.graph(graph):
        _, _, gs, (gx, gh) = mgpt_b200.residual_norm(x, x, keep=True, pre_scale=pre)
        gd = mgpt_b200.residual_norm_backward(gx, gh, gs, x, x, pre_scale=pre)
        back = mgpt_b200.restore8(gx)
    x.copy_(_x(30, 64, torch.bfloat16, seed=8).view(2, 3, 5, 64))
    graph.replay()
    _, _, s, (x8, h8) = mgpt_b200.residual_norm(x, x, keep=True, pre_scale=pre)
    want = mgpt_b200.residual_norm_backward(x8, h8, s, x, x, pre_scale=pre)
    assert torch.equal(back, mgpt_b200.restore8(x8)) and all(torch.equal(p, q) for p, q in zip(want, gd))


def test_refusals():
    x = _x(4, 64, torch.bfloat16)
    for bad in (x.half(), x.t(), x.cpu(), x[:, :60].contiguous(), torch.zeros(3, 0, device="cuda"), torch.tensor(1.0, device="cuda"), x.view(-1)[4:68].view(1, 64)):
        with pytest.raises(MoeError):
            mgpt_b200.keep8(bad)
    kept = mgpt_b200.keep8(x)
    for bad in (Kept8(kept.values, kept.exponents[:, :1], x.dtype), Kept8(kept.values.short(), kept.exponents, x.dtype), Kept8(kept.values, kept.exponents, torch.float16), x,
                Kept8(kept.values.view(-1)[4:68].view(1, 64), kept.exponents[:1], x.dtype)):
        with pytest.raises(MoeError):
            mgpt_b200.restore8(bad)
    with pytest.raises(MoeError):
        mgpt_b200.restore8(kept, torch.float16)
    _, _, stats, (x8, h8) = mgpt_b200.residual_norm(x, x, keep=True)
    for bad in ((x, h8), (x8, x), (mgpt_b200.keep8(x[:2]), h8), (x8, mgpt_b200.keep8(x[:, :32].contiguous()))):
        with pytest.raises(MoeError):
            mgpt_b200.residual_norm_backward(*bad, stats, x)
