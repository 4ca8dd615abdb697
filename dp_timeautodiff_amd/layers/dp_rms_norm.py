"""RMS norm with the residual's addition (K12, include/dpk.h): r = x + residual, y = r / sqrt(mean(r^2) + eps) * weight.

One launch forward and one (plus a short join where few samples have many rows) backward.  Under a GradSampleModule the
backward launch writes the weight's per-sample gradients straight into the arena.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _native
from ..activation8 import Activation8


class _RMSNorm(torch.autograd.Function):
    """(x, residual, weight) -> y, r (r only with a residual), q, e (only with `quantize`).  `sink`: the per-sample gradients'
    destination, with the weight passed detached (unless the engine wants the summed gradients as well); `anchor` keeps the node in the graph when x is data."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, quantize, sink, anchor):
        y, r, rstd, q, e = _native.rms_norm_forward(x, residual, weight, eps, True, quantize)
        ctx.set_materialize_grads(False)
        ctx.sink, ctx.has_residual = sink, residual is not None
        # in 16 bits r is rounded: the weight's gradient, which is not, goes by the sum itself
        parts = (x, residual) if r is None or r.dtype != torch.float32 else (r, None)
        ctx.save_for_backward(*parts, weight, rstd)
        out = (y,) if r is None else (y, r)
        if quantize:
            ctx.mark_non_differentiable(q, e)
            out += (q, e)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr=None, *_):
        r, residual, weight, rstd = ctx.saved_tensors
        if not ctx.has_residual:
            dr = None
        need_x, need_res, need_w = ctx.needs_input_grad[:3]
        if dy is None:  # only r was used: the norm itself has no gradient
            dy = torch.zeros_like(r)
        if ctx.sink is not None:
            with ctx.sink(r.shape[0]) as to:
                dx, _ = _native.rms_norm_backward(r, residual, dy, dr, weight, rstd, need_x or need_res, True, to.window("weight"),
                                                  to.scale, to.accumulate)
            # the summed gradient too, where the engine was asked to leave it to autograd
            dw = _native.rms_norm_backward(r, residual, dy, None, weight, rstd, False, True)[1] if need_w else None
        else:
            dx, dw = _native.rms_norm_backward(r, residual, dy, dr, weight, rstd, need_x or need_res, need_w)
        return dx if need_x else None, dx if need_res else None, dw, None, None, None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
             quantize: bool = False, _sink=None):
    """x [..., C] fp32, bf16 or fp16, residual of the same shape and dtype (or None), weight [C] fp32.

    Returns (y, r) with r = x + residual (x itself without a residual), or (y, r, Activation8) with `quantize`: y also in 8
    bits, without reading y again: in fp32 as compress_activation would hold it, in 16 bits from y before its rounding to them.  The
    8-bit form takes no part in autograd."""
    sink, anchor = _sink if _sink is not None else (None, None)
    if _wants_autograd(anchor, x, residual, weight):
        out = _RMSNorm.apply(x, residual, weight, eps, quantize, sink, anchor)
    else:
        y, r, _, q, e = _native.rms_norm_forward(x, residual, weight, eps, False, quantize)
        out = tuple(t for t in (y, r, q, e) if t is not None)
    y = out[0]
    r = x if residual is None else out[1]
    return (y, r, Activation8(*out[-2:], y.dtype)) if quantize else (y, r)


class DPRMSNorm(nn.Module):
    """RMS norm over the last dimension with the residual's addition: `y, r = norm(x, residual)`."""

    def __init__(self, features: int, eps: float = 1e-6):
        super().__init__()
        if features < 1 or features > _native.RMS_MAX_FEATURES:
            raise ValueError(f"features must be between 1 and {_native.RMS_MAX_FEATURES}")
        self.features, self.eps = features, float(eps)
        self.weight = nn.Parameter(torch.ones(features))
        self.batch_major = False  # True: samples along dimension 0 whatever layout the wrapped model uses
        self._init_runtime()

    def _init_runtime(self):
        object.__setattr__(self, "_dpk_claim", None)  # set by GradSampleModule

    def __deepcopy__(self, memo):
        return _copy_without_runtime(self, memo)

    def extra_repr(self):
        return f"{self.features}, eps={self.eps}"

    def forward(self, x, residual=None, quantize: bool = False):
        claim = _active_claim(self)
        if claim is None:
            return rms_norm(x, self.weight, residual, eps=self.eps, quantize=quantize)
        if x.dim() < 2:
            raise ValueError(f"per-sample gradients need samples along a dimension of their own, got x of shape {tuple(x.shape)}")
        swap = not claim.batch_first and not self.batch_major and x.dim() >= 3  # samples along dimension 1: the kernel wants a sample's rows together
        if swap:
            x, residual = (None if t is None else t.transpose(0, 1).contiguous() for t in (x, residual))
        out = rms_norm(x, claim.parameter(self.weight), residual, eps=self.eps, quantize=quantize, _sink=(claim.sink, claim.anchor))
        if swap:
            back = [t.transpose(0, 1) for t in out[:2]]
            out = (*back, *(Activation8(a.data.transpose(0, 1).contiguous(), a.exponent.transpose(0, 1).contiguous(), a.dtype)
                            for a in out[2:]))
        return out


def _wants_autograd(anchor, *tensors) -> bool:
    """Whether a call has to go through its autograd function: gradients are recorded, or an input carries a forward-mode tangent,
    for which the function raises (it has no jvp; without it the tangent would be lost and read as zero)."""
    tensors = [t for t in tensors if isinstance(t, torch.Tensor)]
    if _has_tangent(*tensors):
        return True
    return torch.is_grad_enabled() and (anchor is not None or any(t.requires_grad for t in tensors))


def _has_tangent(*tensors) -> bool:
    return forward_ad._current_level >= 0 and any(
        isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _active_claim(module):
    """Where a layer's per-sample gradients go, or None outside DP training."""
    claim = module._dpk_claim
    if claim is None or not module.training or not torch.is_grad_enabled() or not claim.enabled():
        return None
    return claim


def _copy_without_runtime(module, memo):
    import copy
    new = module.__class__.__new__(module.__class__)
    nn.Module.__init__(new)
    memo[id(module)] = new
    for k, v in module.__dict__.items():
        if k != "_dpk_claim":
            new.__dict__[k] = copy.deepcopy(v, memo)
    new._init_runtime()
    return new
