"""Routing to experts from logits, over the C ABI: softmax or sigmoid scores, a bias that balances the experts' load, groups of
experts, the k largest, renormalised weights; and the gradient.

:meth:`mgpt_b200.MoELayer.set_routing` has the layer route so; the calls here are for routers of one's own.  They follow
:mod:`mgpt_b200.training` in streams, checks and errors.
"""
from __future__ import annotations

import ctypes as ct
import functools
from operator import index

import torch

from . import _lib
from ._lib import MoeError
from .training import _DTYPES, _EITHER, _F32, _I32, _INT_MAX, _check, _device, _need, _stream


@functools.lru_cache(maxsize=64)
def _numbers(score, groups, top_groups, group_top, renormalise):
    """The argument's bytes without scale and bias (a copy is quicker made than a new one filled), from plain numbers."""
    _need(score in _lib.SCORES, f"routing: score is 'softmax' or 'sigmoid', got {score!r}")
    numbers = (groups, top_groups, group_top)
    _need(all(-_INT_MAX <= v <= _INT_MAX for v in numbers), "routing: sizes out of range")
    return bytes(_lib.Routing(_lib.SCORES[score], *numbers, int(renormalise), 0.0, None))


def _routing(E, score, bias, groups, top_groups, group_top, renormalise, scale, device):
    try:                        # (the cache must not see what can change, such as a tensor of one number)
        groups, group_top, scale, renormalise = index(groups), index(group_top), float(scale), bool(renormalise)
        top_groups = groups if top_groups is None else index(top_groups)
    except (TypeError, ValueError, OverflowError, RuntimeError) as e:
        raise MoeError(f"routing: {e}") from None
    r = _lib.Routing.from_buffer_copy(_numbers(str(score), groups, top_groups, group_top, renormalise))
    r.scale = scale
    if bias is not None:
        r.bias = _check(bias, "bias", (E,), _F32, device)
    return r


def _set(lib, handle, E, device, score, bias=None, groups=1, top_groups=None, group_top=2, renormalise=False, scale=1.0):
    """Has the layer behind the handle route so (score None: as the reference does)."""
    if score is None:
        _lib.check(lib.mgpt_moe_set_routing(handle, None))
    else:
        r = _routing(E, score, bias, groups, top_groups, group_top, renormalise, scale, device)
        _lib.check(lib.mgpt_moe_set_routing(handle, ct.byref(r)))


def _logits(logits):
    device, shape = _device(logits), logits.shape
    if not shape or not shape[-1] or logits.dtype not in _DTYPES:
        raise MoeError(f"routing: logits are [..., E] of FP32 or BF16, got {tuple(shape)} of {logits.dtype}")
    E = shape[-1]
    n = shape.numel() // E
    _need(n <= _INT_MAX >= E, "routing: sizes out of range")
    return device, n, E, _check(logits, "logits", shape, _EITHER, device)


def route(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor = None, groups: int = 1, top_groups: int = None,
          group_top: int = 2, renormalise: bool = False, scale: float = 1.0, counts: torch.Tensor = None):
    """The experts of every token and their weights: ``(top_idx, weights)``, int32 and FP32 ``[..., top_k]``.

    logits: ``[..., E]``, FP32 or BF16, E up to 512.  With s the ``score`` (``"softmax"`` over the experts, or ``"sigmoid"`` of
    each) and ``c = s + bias`` (``bias``: FP32 ``[E]``, for the order only): of ``groups`` groups of consecutive experts the
    ``top_groups`` (default: all) with the largest sums of their ``group_top`` (1 or 2) largest c stay; chosen are their ``top_k``
    (up to 32) largest c, in falling order, equal ones by index (without a bias: the largest logits).  Weights are ``scale * s``, with ``renormalise``
    over the sum of the chosen s (plus 1e-20).  The choice is that of exact arithmetic on the logits given.

    An expert whose logit or bias is -inf or NaN is out: it is chosen only where fewer than ``top_k`` others are left, by index and with
    weight 0.  A NaN among a token's logits (softmax: or +inf) makes its weights NaN; its experts are chosen as ever (softmax: m logits
    of +inf have the scores 1/m, the others 0).  The indices of a token always differ and
    always lie in ``[0, E)``.  ``counts``: int32 ``[E]``, added to: the tokens that chose each expert, which is what a bias is
    adjusted by (``bias += rate * sign(counts.mean() - counts)``)."""
    lib = _lib.load()
    device, n, E, lp = _logits(logits)
    try:
        top_k = index(top_k)
    except TypeError as e:
        raise MoeError(f"routing: top_k: {e}") from None
    _need(0 < top_k <= E, "routing: top_k is 1 to the number of experts")
    r = _routing(E, score, bias, groups, top_groups, group_top, renormalise, scale, device)
    cp = None if counts is None else _check(counts, "counts", (E,), _I32, device)
    top_idx = torch.empty(*logits.shape[:-1], top_k, dtype=torch.int32, device=device)
    weights = torch.empty_like(top_idx, dtype=torch.float32)
    _lib.check(lib.mgpt_moe_op_route(lp, _DTYPES[logits.dtype], n, E, top_k, ct.byref(r), top_idx.data_ptr(), weights.data_ptr(), cp, _stream(device)))
    return top_idx, weights


def route_backward(logits: torch.Tensor, top_idx: torch.Tensor, d_weights: torch.Tensor, *, score: str = "softmax", bias: torch.Tensor = None,
                   renormalise: bool = False, scale: float = 1.0) -> torch.Tensor:
    """The gradient of the logits (of their type) from that of :func:`route`'s weights (``d_weights``: FP32 ``[..., top_k]``): through
    the chosen scores, and for a softmax through its sum.  ``top_idx`` as :func:`route` gave it, with the same other arguments; ``bias``
    matters only where it takes experts out (-inf, NaN): their weights are constants.  The choice itself has no gradient."""
    lib = _lib.load()
    device, n, E, lp = _logits(logits)
    _need(top_idx.dim() == logits.dim() and top_idx.shape[-1] > 0, "routing: top_idx is [..., top_k]")
    k = top_idx.shape[-1]
    shape = logits.shape[:-1] + (k,)
    ip, dp = _check(top_idx, "top_idx", shape, _I32, device), _check(d_weights, "d_weights", shape, _F32, device)
    r = _routing(E, score, bias, 1, 1, 1, renormalise, scale, device)
    d_logits = torch.empty_like(logits)
    _lib.check(lib.mgpt_moe_op_route_backward(lp, _DTYPES[logits.dtype], ip, dp, n, E, k, ct.byref(r), d_logits.data_ptr(), _stream(device)))
    return d_logits
