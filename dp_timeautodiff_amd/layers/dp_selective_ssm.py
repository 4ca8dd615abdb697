"""Selective state-space layer: short causal convolution (K13) and selective scan (K14), for training, prompts and single tokens.

    dt = softplus(delta + dt_bias);  h_t = exp(-exp(A_log) dt) h_{t-1} + dt B_t u_t;  y = C_t . h_t + D u_t;  out = y silu(z)

Tensors are batch-major: [B, T, channels], fp32, bf16 or fp16, any strides with a contiguous last dimension (column blocks of
a wider projection are read where they lie).  Parameters and scan states are fp32.  `lengths` (int32 [B]) makes the batch a
padded one: rows at and behind a sequence's length are not read, give zeros and take no gradient, and the returned state is that
behind the sequence's own last row.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _native
from .dp_rnn import RNNLinear
from .dp_rms_norm import DPRMSNorm, _active_claim, _copy_without_runtime, _has_tangent, _wants_autograd

_ACTIVATIONS = {None: False, "silu": True}


def _silu(activation) -> bool:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    return _ACTIVATIONS[activation]


def _refuse_tangents(name: str, *tensors):
    if _has_tangent(*tensors):
        raise NotImplementedError(f"{name} is not differentiable: an input carries a forward-mode tangent")


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, want_state, sink, anchor):
        y, out = _native.causal_conv_forward(x, weight, bias, state, lengths, silu, want_state)
        ctx.set_materialize_grads(False)
        ctx.silu, ctx.sink = silu, sink
        ctx.save_for_backward(x, weight, bias, state, lengths)
        return (y, out) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate=None):
        x, weight, bias, state, lengths = ctx.saved_tensors
        need_x, need_w, need_b, need_s = ctx.needs_input_grad[:4]
        if dy is None:
            dy = torch.zeros_like(x)
        args = (x, weight, bias, state, lengths, ctx.silu, dy, dstate, need_s)
        if ctx.sink is not None:
            with ctx.sink(x.shape[0]) as to:
                wins = (to.window("weight"), to.window("bias") if bias is not None else None)
                dx, ds, _ = _native.causal_conv_backward(*args, True, wins, to.scale, to.accumulate)
            # the summed gradients too, where the engine was asked to leave them to autograd
            grads = _native.causal_conv_backward(*args, True)[2] if need_w or need_b else None
        else:
            dx, ds, grads = _native.causal_conv_backward(*args, need_w or need_b)
        dw, db = grads if grads is not None else (None, None)
        return dx if need_x else None, dw, db, ds, None, None, None, None, None


def causal_conv(x, weight, bias=None, *, activation: Optional[str] = "silu", state=None, lengths=None,
                return_state: bool = False, _sink=None):
    """y_t = act(bias + sum_i weight[:, i] x_{t-W+1+i}) per channel; x [B,T,D], weight [D,W] (W up to 4), bias [D].  `state`
    [B,W-1,D] holds the rows before the first (zeros if None).  Returns y, or (y, state behind the sequences)."""
    sink, anchor = _sink if _sink is not None else (None, None)
    silu = _silu(activation)
    if _wants_autograd(anchor, x, weight, bias, state):
        return _CausalConv.apply(x, weight, bias, state, lengths, silu, return_state, sink, anchor)
    y, out = _native.causal_conv_forward(x, weight, bias, state, lengths, silu, return_state)
    return (y, out) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, activation: Optional[str] = "silu"):
    """One token: x [B,D]; `state` [B,W-1,D] is updated in place.  Not differentiable."""
    _refuse_tangents("causal_conv_step", x, state, weight, bias)
    return _native.causal_conv_step(x, state, weight, bias, _silu(activation))


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A_log, B, C, D, z, dt_bias, state, lengths, softplus, want_state, sink, anchor):
        inp = _native.ScanInputs(u, delta, A_log, B, C, D, z, dt_bias, state, lengths, softplus)
        out, hT, kept = _native.selective_scan_forward(inp, True, want_state)
        ctx.set_materialize_grads(False)
        ctx.softplus, ctx.sink = softplus, sink
        ctx.save_for_backward(inp.u, inp.delta, inp.A_log, inp.B, inp.C, inp.D, inp.z, inp.dt_bias, inp.h0, inp.lengths, kept)
        return (out, hT) if want_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dstate=None):
        *operands, kept = ctx.saved_tensors
        inp = _native.ScanInputs.checked(*operands, ctx.softplus)
        need = ctx.needs_input_grad
        need_par = need[2] or need[5] or need[7]
        if dout is None:
            dout = torch.zeros_like(inp.u)
        if ctx.sink is not None:
            with ctx.sink(inp.u.shape[0]) as to:
                wins = (to.window("A_log"), *(to.window(n) if t is not None else None
                                              for n, t in (("D", inp.D), ("dt_bias", inp.dt_bias))))
                du, ddelta, dB, dC, dz, dh0, _ = _native.selective_scan_backward(inp, kept, dout, dstate, need[8], True, wins,
                                                                                 to.scale, to.accumulate)
            # the summed gradients too, where the engine was asked to leave them to autograd
            grads = _native.selective_scan_backward(inp, kept, dout, dstate, False, True)[6] if need_par else None
        else:
            du, ddelta, dB, dC, dz, dh0, grads = _native.selective_scan_backward(inp, kept, dout, dstate, need[8], need_par)
        grads = grads if grads is not None else (None, None, None)
        out = (du, ddelta, grads[0], dB, dC, grads[1], dz, grads[2], dh0)
        return (*(g if n else None for g, n in zip(out, need)), None, None, None, None, None)


def selective_scan(u, delta, A_log, B, C, D=None, z=None, dt_bias=None, *, softplus: bool = True, state=None, lengths=None,
                   return_state: bool = False, _sink=None):
    """u, delta, z [B,T,D]; B, C [B,T,N]; A_log [D,N] (N up to 32), D, dt_bias [D], state [B,D,N] fp32.  D, z, dt_bias and
    state may be None (no skip, no gate, no bias, zeros).  Returns out [B,T,D], or (out, final state [B,D,N])."""
    sink, anchor = _sink if _sink is not None else (None, None)
    if _wants_autograd(anchor, u, delta, A_log, B, C, D, z, dt_bias, state):
        return _SelectiveScan.apply(u, delta, A_log, B, C, D, z, dt_bias, state, lengths, softplus, return_state, sink, anchor)
    inp = _native.ScanInputs(u, delta, A_log, B, C, D, z, dt_bias, state, lengths, softplus)
    out, hT, _ = _native.selective_scan_forward(inp, False, return_state)
    return (out, hT) if return_state else out


def selective_scan_step(u, delta, A_log, B, C, state, D=None, z=None, dt_bias=None, *, softplus: bool = True):
    """One token: u, delta, z [B,D], B, C [B,N]; `state` [B,D,N] is updated in place.  Not differentiable."""
    _refuse_tangents("selective_scan_step", u, delta, A_log, B, C, state, D, z, dt_bias)
    return _native.selective_scan_step(_native.ScanInputs(u, delta, A_log, B, C, D, z, dt_bias, None, None, softplus, step=True),
                                       state)


class DPCausalConv(nn.Module):
    """Depthwise causal convolution over time with its activation; per-sample gradients by K13."""

    def __init__(self, channels: int, width: int = 4, bias: bool = True, activation: Optional[str] = "silu"):
        super().__init__()
        if channels < 1 or not 1 <= width <= _native.CONV_MAX_WIDTH:
            raise ValueError(f"channels must be positive and width between 1 and {_native.CONV_MAX_WIDTH}")
        _silu(activation)
        self.channels, self.width, self.activation = channels, width, activation
        bound = 1.0 / math.sqrt(width)
        self.weight = nn.Parameter(torch.empty(channels, width).uniform_(-bound, bound))
        self.bias = nn.Parameter(torch.empty(channels).uniform_(-bound, bound)) if bias else None
        self._init_runtime()

    def _init_runtime(self):
        object.__setattr__(self, "_dpk_claim", None)  # set by GradSampleModule

    def __deepcopy__(self, memo):
        return _copy_without_runtime(self, memo)

    def forward(self, x, state=None, lengths=None, return_state: bool = False):
        claim = _active_claim(self)
        w, b, sink = self.weight, self.bias, None
        if claim is not None:
            w, b, sink = claim.parameter(w), None if b is None else claim.parameter(b), (claim.sink, claim.anchor)
        return causal_conv(x, w, b, activation=self.activation, state=state, lengths=lengths, return_state=return_state, _sink=sink)

    def step(self, x, state):
        return causal_conv_step(x, state, self.weight, self.bias, activation=self.activation)


class DPSelectiveScan(nn.Module):
    """The scan with its own parameters A_log, D and dt_bias; per-sample gradients by K14."""

    def __init__(self, channels: int, state_size: int = 16, dt_min: float = 1e-3, dt_max: float = 1e-1):
        super().__init__()
        if channels < 1 or not 1 <= state_size <= _native.SCAN_MAX_STATE:
            raise ValueError(f"channels must be positive and state_size between 1 and {_native.SCAN_MAX_STATE}")
        if not 0 < dt_min <= dt_max:
            raise ValueError("expected 0 < dt_min <= dt_max")
        self.channels, self.state_size = channels, state_size
        # decay rates 1 .. N in every channel, step sizes spread evenly over the decades between dt_min and dt_max
        self.A_log = nn.Parameter(torch.arange(1, state_size + 1, dtype=torch.float32).log().repeat(channels, 1))
        self.D = nn.Parameter(torch.ones(channels))
        dt = torch.exp(torch.rand(channels) * (math.log(dt_max) - math.log(dt_min)) + math.log(dt_min))
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))  # softplus of it is dt
        self._init_runtime()

    def _init_runtime(self):
        object.__setattr__(self, "_dpk_claim", None)  # set by GradSampleModule

    def __deepcopy__(self, memo):
        return _copy_without_runtime(self, memo)

    def forward(self, u, delta, B, C, z=None, state=None, lengths=None, return_state: bool = False):
        claim = _active_claim(self)
        par, sink = (self.A_log, self.D, self.dt_bias), None
        if claim is not None:
            par, sink = tuple(claim.parameter(p) for p in par), (claim.sink, claim.anchor)
        return selective_scan(u, delta, par[0], B, C, par[1], z, par[2], state=state, lengths=lengths, return_state=return_state,
                              _sink=sink)

    def step(self, u, delta, B, C, state, z=None):
        return selective_scan_step(u, delta, self.A_log, B, C, state, self.D, z, self.dt_bias)


class SSMState(NamedTuple):
    """What a sequence's later tokens need of its earlier ones."""
    conv: torch.Tensor  # [B, width - 1, channels], the layer's dtype
    scan: torch.Tensor  # [B, channels, state_size] fp32


class DPSelectiveSSM(nn.Module):
    """in_proj -> causal convolution -> (delta, B, C) -> selective scan gated by z -> out_proj, batch-major [B, T, d_model].

    The sequence mixer to put where a DPLSTM / DPGRU stands: all its parameters have per-sample-gradient kernels (the projections
    by K1).  `forward(..., return_state=True)` returns the SSMState that `step` advances token by token."""

    def __init__(self, d_model: int, state_size: int = 16, conv_width: int = 4, expand: int = 2, dt_rank: Optional[int] = None,
                 bias: bool = False):
        super().__init__()
        self.d_model, self.state_size, self.channels = d_model, state_size, expand * d_model
        self.dt_rank = dt_rank if dt_rank is not None else max(1, math.ceil(d_model / 16))
        self.in_proj = SSMLinear(d_model, 2 * self.channels, bias)
        self.conv = DPCausalConv(self.channels, conv_width)
        self.x_proj = SSMLinear(self.channels, self.dt_rank + 2 * state_size, False)
        self.dt_proj = SSMLinear(self.dt_rank, self.channels, False)  # its bias is the scan's dt_bias
        self.scan = DPSelectiveScan(self.channels, state_size)
        self.out_proj = SSMLinear(self.channels, d_model, bias)

    def _split(self, dbc):
        return torch.split(dbc, [self.dt_rank, self.state_size, self.state_size], -1)

    def forward(self, x, state: Optional[SSMState] = None, lengths=None, return_state: bool = False, kept=None):
        """x [B,T,d_model]; `kept`: x in 8 bits, if the caller has it (GradSampleModule(activation_bits=8) stashes that, and refuses
        one of another shape, dtype or device; that it holds the values of this x is the caller's to see to)."""
        xr, z = torch.split(self.in_proj(x, kept), self.channels, -1)
        conv_state, scan_state = state if state is not None else (None, None)
        u = self.conv(xr, conv_state, lengths, return_state)
        if return_state:
            u, conv_state = u
        dt, B, C = self._split(self.x_proj(u))
        y = self.scan(u, self.dt_proj(dt), B, C, z, scan_state, lengths, return_state)
        if return_state:
            y, scan_state = y
        out = self.out_proj(y)
        return (out, SSMState(conv_state, scan_state)) if return_state else out

    def initial_state(self, batch: int, dtype=torch.float32) -> SSMState:
        dev = self.in_proj.weight.device
        return SSMState(torch.zeros(batch, self.conv.width - 1, self.channels, dtype=dtype, device=dev),
                        torch.zeros(batch, self.channels, self.state_size, dtype=torch.float32, device=dev))

    @torch.no_grad()
    def step(self, x, state: SSMState):
        """One token of every sequence: x [B,d_model]; `state` is updated in place."""
        xr, z = torch.split(self.in_proj(x), self.channels, -1)
        u = self.conv.step(xr, state.conv)
        dt, B, C = self._split(self.x_proj(u))
        return self.out_proj(self.scan.step(u, self.dt_proj(dt), B, C, state.scan, z))


class SSMLinear(RNNLinear):
    """A projection of the state-space layer: batch-major whatever layout the wrapped model uses.  `kept` is its input in
    8 bits, where the layer before has written that already; only the engine's stash reads it."""

    def forward(self, x, kept=None):
        return super().forward(x)


class DPSelectiveSSMBlock(nn.Module):
    """Pre-norm residual block: `out, residual = block(x, residual)` with residual := x + residual, out = mixer(norm(residual)).
    The next block (or a final DPRMSNorm) adds `out` to the residual stream; the first call passes residual=None."""

    def __init__(self, d_model: int, state_size: int = 16, conv_width: int = 4, expand: int = 2, eps: float = 1e-6):
        super().__init__()
        self.norm = DPRMSNorm(d_model, eps)
        self.norm.batch_major = True
        self.mixer = DPSelectiveSSM(d_model, state_size, conv_width, expand)

    def forward(self, x, residual=None, lengths=None):
        claim = _active_claim(self.norm)
        if claim is not None and claim.activation_bits == 8:
            # the norm writes the in_proj's stash along with its output
            y, residual, kept = self.norm(x, residual, quantize=True)
            return self.mixer(y, lengths=lengths, kept=kept), residual
        y, residual = self.norm(x, residual)
        return self.mixer(y, lengths=lengths), residual

    @torch.no_grad()
    def step(self, x, state: SSMState, residual=None):
        """One token: x, residual [B,d_model]; `state` is updated in place."""
        y, residual = self.norm(x, residual)
        return self.mixer.step(y, state), residual
