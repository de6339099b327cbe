"""The expert side touches the rows of a call and no others: behind them lie NaN in what it reads and a pattern in what it writes, or no memory at all."""
import math

import pytest
import torch

from mgpt_b200 import MoELayer, _lib

pytestmark = pytest.mark.gpu
BEHIND = 1024                           # rows
MAPPED = 14 << 20                       # bytes


def _rel(got, want):
    return float((got.double() - want).norm() / want.norm().clamp(min=1e-12))


@pytest.mark.parametrize("at_the_end", [False, True])
@pytest.mark.parametrize("mode,gemm_impl", [("fp32", 0), ("bf16", 0), ("bf16", 1)])
@pytest.mark.parametrize("C,H,counts", [(64, 128, [[128, 152, 72, 45]]), (64, 128, [[143, 141, 117, 201]]), (72, 136, [[1, 0, 300, 128]]), (128, 320, [[5, 7], [0, 260], [129, 1]]),
                                        (320, 328, [[700, 520]])])
def test_rows(mode, gemm_impl, C, H, counts, at_the_end):
    E, n_src = len(counts[0]), len(counts)
    g = torch.Generator(device="cuda").manual_seed(C + H)
    layer = MoELayer(C, H, E, 1, mode=mode, gemm_impl=gemm_impl)
    layer.load_parameters([(torch.randn(p.shape, device="cuda", generator=g) * (p.shape[0] ** -0.5 if p.shape[0] > 1 else 0.1)).bfloat16().float().cpu().numpy()
                           for p in layer.get_parameters()])
    dtype = torch.float32 if mode == "fp32" else torch.bfloat16
    real, expert = [], []
    for s in counts:
        for e, c in enumerate(s):
            pad = -(-c // 128) * 128
            real += [True] * c + [False] * (pad - c)
            expert += [e] * pad
    n = len(real)
    real, expert = torch.tensor(real, device="cuda"), torch.tensor(expert, device="cuda")

    def rows(fill):
        if not at_the_end:
            return torch.full((n + BEHIND, C), fill, device="cuda").to(dtype)
        whole = torch.empty(MAPPED, dtype=torch.uint8, device="cuda")       # (an allocation of its own, of whole pages)
        return whole[MAPPED - n * C * dtype.itemsize:].view(dtype).view(n, C)

    x, dy, out, dx = rows(math.nan), rows(math.nan), rows(-7.0), rows(-7.0)
    for t in (x, dy):
        t[:n] = torch.where(real[:, None], torch.randn(n, C, device="cuda", generator=g), 0.0).to(dtype)
    seg = torch.tensor(counts, dtype=torch.int32, device="cuda")
    lib, h, stream = layer.lib, layer._h, layer._stream()
    ws = torch.empty(int(lib.mgpt_moe_stage_workspace_bytes(h, n, 0)), dtype=torch.uint8, device="cuda")
    layer.zero_grad()
    _lib.check(lib.mgpt_moe_experts_forward(h, x.data_ptr(), seg.data_ptr(), n_src, n, out.data_ptr(), ws.data_ptr(), ws.numel(), stream))
    _lib.check(lib.mgpt_moe_experts_backward(h, dy.data_ptr(), dx.data_ptr(), ws.data_ptr(), ws.numel(), stream))
    layer.check_status()
    assert (out[n:] == -7.0).all() and (dx[n:] == -7.0).all() and torch.isnan(x[n:]).all() and torch.isnan(dy[n:]).all()
    P = [p.detach().double().requires_grad_() for p in layer.get_parameters()]
    leaf = x[:n].double().requires_grad_()
    y = torch.zeros(n, C, dtype=torch.float64, device="cuda")
    for e in range(E):
        Wg, bg, Wu, bu, Wd, bd = P[2 + 6 * e: 8 + 6 * e]
        at = torch.nonzero((expert == e) & real)[:, 0]
        r = leaf[at]
        y = y.index_add(0, at, (torch.nn.functional.silu(r @ Wg + bg) * (r @ Wu + bu)) @ Wd + bd)
    grads = torch.autograd.grad(y, [leaf] + P[2:], dy[:n].double(), allow_unused=True)
    bar = 1e-5 if mode == "fp32" else 2e-2
    assert _rel(out[:n][real], y.detach()[real]) < bar and _rel(dx[:n][real], grads[0][real]) < bar
    for i, (p, w) in enumerate(zip(layer.get_parameters()[2:], grads[1:])):
        if w is not None and float(w.norm()) > 0:
            assert _rel(p.grad, w) < bar, i
        assert torch.isfinite(p.grad).all()
