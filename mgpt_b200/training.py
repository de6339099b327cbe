"""The rest of a training step around the layer, over the C ABI: the loss of a language model's head, the norms around a
block with its gate and skip connection, and AdamW over many tensors.

As in :mod:`mgpt_b200.moe_layer`, torch is used for device memory and streams only.  Every call enqueues its work on the
current stream and returns; wrong arguments raise :class:`MoeError` before anything is enqueued.
"""
from __future__ import annotations

import ctypes as ct

import numpy as np
import torch

from . import _lib
from ._lib import IO_BF16, IO_F32, MoeError

PIECE_BYTES = 512 << 20         # of the vocabulary's gradient rows that are worked on at a time
STATE_BLOCK = 256               # elements that share a scale of the 8-bit moments

_DTYPES = {torch.float32: IO_F32, torch.bfloat16: IO_BF16}
_F32, _BF16, _I32, _EITHER = (torch.float32,), (torch.bfloat16,), (torch.int32,), (torch.float32, torch.bfloat16)
_TENSOR = np.dtype([("w", "u8"), ("grad", "u8"), ("w_bf16", "u8"), ("n", "i8"), ("weight_decay", "f4"), ("grad_dtype", "i4")])      # mgpt_moe_optim_tensor
_INT_MAX = 2 ** 31 - 1          # ctypes cuts larger numbers to 32 bits without a word
_status = {}


def _need(ok, what):
    if not ok:
        raise MoeError(what)


def _device(t: torch.Tensor) -> torch.device:
    if not t.is_cuda:
        raise MoeError("mgpt_b200: tensors must be on a CUDA device; there is no CPU path")
    device = t.device
    if device.index != torch.cuda.current_device():
        raise MoeError(f"tensors are on {device}, the current device is cuda:{torch.cuda.current_device()}")
    return device


def _check(t, name, shape, dtypes, device):
    """The address of a contiguous tensor of this shape, one of these types, on this device."""
    if t.dtype in dtypes and t.shape == shape and t.is_contiguous() and t.device == device:
        return t.data_ptr()
    raise MoeError(f"{name}: expected a contiguous {tuple(shape)} tensor of {' or '.join(str(d) for d in dtypes)} on {device}, "
                   f"got {tuple(t.shape)} of {t.dtype} on {t.device}" + ("" if t.is_contiguous() else ", not contiguous"))


def _optional(t, name, shape, dtypes, device):
    return None if t is None else _check(t, name, shape, dtypes, device)


# (the stream's handle without the object around it: 2 us less per call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream(device):
    return _raw_stream(device.index)


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _status_word(device):
    s = _status.get(device)
    if s is None:
        _need(not torch.cuda.is_current_stream_capturing(), "head loss: a device's first call, which makes its status word, cannot be captured in a graph")
        s = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()     # cleared before any stream writes to it
        _status[device] = s
    return s


def check_status(device=None) -> None:
    """Raises :class:`MoeError` if a call of :func:`head_loss` or :func:`head_loss_backward` on this device recorded an error
    since the last check (a target beyond the vocabulary, a bounded wait that ran out).  Synchronises the device."""
    device = torch.device("cuda" if device is None else device)
    if device.index is None:                                # ("cuda" is no tensor's device: theirs have a number)
        device = torch.device(device.type, torch.cuda.current_device())
    s = _status.get(device)
    if s is None:
        return
    torch.cuda.synchronize(device)
    bits = int(s.item())
    if bits:
        s.zero_()
        torch.cuda.synchronize(device)
        what = []
        if bits & 32:
            what.append("a target is beyond the vocabulary (it took no part)")
        if bits & ~32:
            what.append("a bounded wait ran out: results are incomplete")
        raise MoeError(f"head loss status {bits}: " + "; ".join(what))


# ---- the loss of a language model's head ------------------------------------------------------------------------------
def _head_args(x, weight, targets):
    device, dtype, shape, matrix = _device(x), x.dtype, x.shape, weight.shape
    if dtype not in _DTYPES or not shape or len(matrix) != 2 or not matrix[0] or not matrix[1] or shape[-1] != matrix[1]:
        raise MoeError(f"head loss: x is [..., C] of FP32 or BF16, weight [V, C]; got {tuple(shape)} of {dtype}, {tuple(matrix)}")
    V, C = matrix
    n = x.numel() // C
    _need(max(n, C, V) <= _INT_MAX, "head loss: sizes out of range")
    return (device, n, C, V, _check(x, "x", shape, _EITHER, device), _check(weight, "weight", matrix, _BF16, device),
            _check(targets, "targets", shape[:-1], _I32, device))


def head_loss(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor):
    """Cross entropy of ``x @ weight.T`` against ``targets``, token by token, without keeping the logits.

    x: ``[..., C]``, FP32 or BF16; weight: BF16 ``[V, C]``; targets: int32 ``[...]``.  Returns ``(loss, lse)``, FP32
    ``[...]``: ``lse`` is what :func:`head_loss_backward` needs.  Tokens whose target is outside ``[0, V)`` (padding, prompts)
    take no part: loss and lse 0, whatever their x holds, and no work (beyond one tile of 256 tokens); targets ``>= V`` are reported by :func:`check_status`."""
    lib = _lib.load()
    device, n, C, V, xp, wp, tp = _head_args(x, weight, targets)
    loss, lse = torch.empty_like(targets, dtype=torch.float32), torch.empty_like(targets, dtype=torch.float32)
    if n:
        size = lib.mgpt_moe_op_head_loss_workspace_bytes(n, C, V)
        ws = _workspace(size, device)
        _lib.check(lib.mgpt_moe_op_head_loss(xp, _DTYPES[x.dtype], wp, tp, n, C, V, loss.data_ptr(), lse.data_ptr(),
                                             _status_word(device).data_ptr(), ws.data_ptr(), size, _stream(device)))
    return loss, lse


def head_loss_backward(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, d_loss: torch.Tensor,
                       d_weight: torch.Tensor = None, *, piece_bytes: int = PIECE_BYTES):
    """Gradients of :func:`head_loss`: ``(dx, d_weight)``.  ``d_loss``: FP32 ``[...]``, the gradient of each token's loss
    (``1 / tokens`` for the mean).  ``d_weight``: an FP32 ``[V, C]`` tensor is added to, a BF16 one (or none: it is made) is
    written.  ``piece_bytes``: workspace for the piece of the vocabulary that is worked on at a time."""
    lib = _lib.load()
    device, n, C, V, xp, wp, tp = _head_args(x, weight, targets)
    lp = _check(lse, "lse", targets.shape, _F32, device)
    gp = _check(d_loss, "d_loss", targets.shape, _F32, device)
    if d_weight is None:
        d_weight = torch.empty_like(weight)
    dwp = _check(d_weight, "d_weight", (V, C), _EITHER, device)
    dx = torch.empty_like(x)
    size = lib.mgpt_moe_op_head_loss_backward_workspace_bytes(n, C, V, piece_bytes) if n else 0
    ws = _workspace(size, device)
    _lib.check(lib.mgpt_moe_op_head_loss_backward(xp, _DTYPES[x.dtype], wp, tp, lp, gp, n, C, V, dx.data_ptr(), dwp, _DTYPES[d_weight.dtype],
                                                  _status_word(device).data_ptr(), ws.data_ptr(), size, _stream(device)))
    return dx, d_weight


# ---- norms around a block ---------------------------------------------------------------------------------------------
def _norm_args(x, h, post_scale, gate, pre_scale, tokens_per_gate):
    device, dtype, shape = _device(x), x.dtype, x.shape
    if dtype not in _DTYPES or not shape:
        raise MoeError(f"residual norm: unsupported tokens {tuple(shape)} of {dtype}")
    C = shape[-1]
    n = x.numel() // C if C else 0
    _need(max(n, C) <= _INT_MAX, "residual norm: sizes out of range")
    if tokens_per_gate:
        _need(tokens_per_gate > 0, "residual norm: tokens_per_gate must not be negative")
        rows = -(-n // tokens_per_gate)
        tokens_per_gate = min(tokens_per_gate, n)       # (C's int does not hold every number that means one row)
    else:
        rows = 1
    if gate is not None and rows == 1 and gate.dim() == 1 and gate.numel() == C:
        gate = gate.view(1, C)
    types, cols = (dtype,), (C,)
    return (device, n, C, rows, tokens_per_gate, _check(x, "x", shape, types, device), _check(h, "h", shape, types, device), _optional(post_scale, "post_scale", cols, _F32, device),
            _optional(gate, "gate", (rows, C), _F32, device), _optional(pre_scale, "pre_scale", cols, _F32, device))


def residual_norm(x: torch.Tensor, h: torch.Tensor, *, post_scale=None, gate=None, pre_scale=None, alpha: float = 1.0, eps: float = 1e-5,
                  tokens_per_gate: int = 0):
    """``y = alpha*x + gate * rmsnorm(h)*post_scale`` and ``u = rmsnorm(y)*pre_scale``: what follows a block and precedes the
    next one, in one pass.  x, h: ``[..., C]``, both FP32 or both BF16.  Without ``post_scale`` h is not normalised, without
    ``gate`` it is 1, without ``pre_scale`` there is no u (None).  ``gate``: FP32 ``[rows, C]``, a row for every
    ``tokens_per_gate`` consecutive tokens (0: one row, which may be given as ``[C]``).  Returns ``(y, u, stats)``; ``stats`` is
    what :func:`residual_norm_backward` needs."""
    lib = _lib.load()
    device, n, C, _, tokens_per_gate, xp, hp, post, gp, pre = _norm_args(x, h, post_scale, gate, pre_scale, tokens_per_gate)
    y = torch.empty_like(x)
    u = torch.empty_like(x) if pre_scale is not None else None
    stats = torch.empty((2, n), dtype=torch.float32, device=device)
    _lib.check(lib.mgpt_moe_op_residual_norm(xp, hp, _DTYPES[x.dtype], post, gp, tokens_per_gate, pre, alpha, eps, n, C, y.data_ptr(),
                                             None if u is None else u.data_ptr(), stats.data_ptr(), _stream(device)))
    return y, u, stats


def residual_norm_backward(x: torch.Tensor, h: torch.Tensor, stats: torch.Tensor, dy: torch.Tensor, du: torch.Tensor = None, *, post_scale=None,
                           gate=None, pre_scale=None, alpha: float = 1.0, eps: float = 1e-5, tokens_per_gate: int = 0, d_post_scale=None,
                           d_gate=None, d_pre_scale=None):
    """Gradients of :func:`residual_norm`: returns ``(dx, dh)`` and adds to ``d_post_scale``, ``d_gate`` and ``d_pre_scale`` (FP32,
    of the parameters' shapes) where they are given.  ``dy``: the gradient of y by its other uses; ``du``: that of u.  The other
    arguments are those of the forward call (``eps`` is in ``stats`` already)."""
    lib = _lib.load()
    device, n, C, rows, tokens_per_gate, xp, hp, post, gp, pre = _norm_args(x, h, post_scale, gate, pre_scale, tokens_per_gate)
    f32 = _F32
    sp = _check(stats, "stats", (2, n), f32, device)
    dyp, dup = _check(dy, "dy", x.shape, (x.dtype,), device), _optional(du, "du", x.shape, (x.dtype,), device)
    if d_gate is not None and d_gate.dim() == 1 and rows == 1 and d_gate.numel() == C:
        d_gate = d_gate.view(1, C)
    dpost, dgate, dpre = (_optional(d_post_scale, "d_post_scale", (C,), f32, device), _optional(d_gate, "d_gate", (rows, C), f32, device),
                          _optional(d_pre_scale, "d_pre_scale", (C,), f32, device))
    dx, dh = torch.empty_like(x), torch.empty_like(x)
    size = lib.mgpt_moe_op_residual_norm_backward_workspace_bytes(n, C, tokens_per_gate)
    ws = _workspace(size, device)
    _lib.check(lib.mgpt_moe_op_residual_norm_backward(xp, hp, _DTYPES[x.dtype], post, gp, tokens_per_gate, pre, alpha, n, C, sp, dyp, dup,
                                                      dx.data_ptr(), dh.data_ptr(), dpost, dgate, dpre, ws.data_ptr(), size, _stream(device)))
    return dx, dh


# ---- optimiser --------------------------------------------------------------------------------------------------------
class AdamW:
    """AdamW over many tensors in one launch.  ``weights``: FP32 tensors; ``grads``: FP32 or BF16 tensors of the same sizes;
    ``copies`` (optional): BF16 tensors that get the new weights; ``weight_decay``: one number, or one per tensor.

    ``state_bits`` 32 keeps the moments in FP32 (``m``, ``v``); 8 keeps a byte each for m and the root of v (``m``, ``v``:
    float8_e4m3fn, in units of ``m_scale``, ``v_scale``, one power of two per 256 elements; ``v`` stands for sqrt(v)), rounded
    stochastically as ``seed`` and the step say.  An element whose gradients are less than about 2^-17 of its block's largest takes
    smaller steps than it would with exact moments (32 bits keep them).  Every tensor starts on a multiple of 256 elements of the state;
    ``state`` gives buffers of that form to continue from.  The tensors' addresses are taken once, here: a tensor that
    moves needs a new object (with the old one's state)."""

    def __init__(self, weights, grads, *, copies=None, state_bits: int = 8, state=None, weight_decay=0.01, seed: int = 0):
        self.lib = _lib.load()
        self._h = ct.c_void_p()
        self.weights, self.grads = list(weights), list(grads)
        self.copies = list(copies) if copies is not None else [None] * len(self.weights)
        n = len(self.weights)
        _need(n > 0 and len(self.grads) == n and len(self.copies) == n, "AdamW: as many gradients (and copies) as weights, at least one")
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * n
        _need(len(decay) == n, "AdamW: one weight decay, or one per tensor")
        _need(state_bits in (8, 32), "AdamW: state_bits must be 8 or 32")
        self.device, self.state_bits, self.seed = _device(self.weights[0]), state_bits, int(seed) & 0xFFFFFFFF
        table = np.zeros(n, dtype=_TENSOR)
        device, f32, b16 = self.device, torch.float32, torch.bfloat16
        for i, (w, g, c) in enumerate(zip(self.weights, self.grads, self.copies)):
            shape, gd = w.shape, g.dtype
            if not (w.dtype is f32 and (gd is f32 or gd is b16) and g.shape == shape and w.is_contiguous() and g.is_contiguous() and w.device == device == g.device
                    and (c is None or (c.dtype is b16 and c.shape == shape and c.is_contiguous() and c.device == device))):
                for t, name, dtypes in ((w, "weights", _F32), (g, "grads", _EITHER), (c, "copies", _BF16)):
                    _optional(t, f"{name}[{i}]", shape, dtypes, device)
            table[i] = (w.data_ptr(), g.data_ptr(), 0 if c is None else c.data_ptr(), w.numel(), decay[i], _DTYPES[gd])
        table = table.ctypes.data_as(ct.POINTER(_lib.OptimTensor))
        self.blocks = int(self.lib.mgpt_moe_optim_blocks(table, n))
        total, dtype = self.blocks * STATE_BLOCK, torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        if state is None:
            self.m, self.v = torch.zeros(total, dtype=dtype, device=self.device), torch.zeros(total, dtype=dtype, device=self.device)
            self.m_scale, self.v_scale = (torch.ones(self.blocks, device=self.device), torch.ones(self.blocks, device=self.device)) if state_bits == 8 else (None, None)
        else:
            _need(len(state) == (2 if state_bits == 32 else 4), "AdamW: state is (m, v), or (m, v, m_scale, v_scale) for 8 bits")
            self.m, self.v = state[:2]
            self.m_scale, self.v_scale = state[2:] if state_bits == 8 else (None, None)
        self._p = [_check(self.m, "m", (total,), (dtype,), self.device), _check(self.v, "v", (total,), (dtype,), self.device),
                   _optional(self.m_scale, "m_scale", (self.blocks,), _F32, self.device),
                   _optional(self.v_scale, "v_scale", (self.blocks,), _F32, self.device)]
        self.found_nonfinite = torch.zeros(1, dtype=torch.int32, device=self.device)
        torch.cuda.current_stream(self.device).synchronize()       # cleared before a step on any stream reads them
        _lib.check(self.lib.mgpt_moe_optim_create(self.device.index, table, n, state_bits, ct.byref(self._h)))

    def step(self, t: int, lr: float = 3e-4, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8, grad_scale: torch.Tensor = None) -> None:
        """One step; ``t`` counts from 1.  ``grad_scale``: an FP32 tensor of one element that multiplies the gradients.  Elements
        whose gradient is not finite keep their values and set ``found_nonfinite``.  Not for capture in a graph, which would repeat
        ``t``, ``lr`` and the rounding's random bits: refused."""
        _need(self._h.value, "AdamW: closed")
        gs = _optional(grad_scale, "grad_scale", () if grad_scale is not None and grad_scale.dim() == 0 else (1,), _F32, self.device)
        _lib.check(self.lib.mgpt_moe_optim_step(self._h, *self._p, lr, beta1, beta2, eps, int(t), gs, self.seed,
                                                self.found_nonfinite.data_ptr(), _stream(self.device)))

    def close(self) -> None:
        if getattr(self, "_h", None) and self._h.value:
            torch.cuda.synchronize(self.device)              # a step in flight reads the table
            self.lib.mgpt_moe_optim_destroy(self._h)
            self._h = ct.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
