"""Activations held in 8 bits between forward and backward (K15, include/dpk.h).

A DP-SGD step keeps the input of every Linear until the backward pass contracts it with the layer's backprops; in fp32 that
stash is what bounds the physical batch of long sequences after the per-sample-gradient arena.  `compress_activation` keeps a
tensor as one signed byte per element and one exponent byte per 128 neighbours of the last dimension (the scale is a
power of two, so the stored value is the correctly rounded quotient); `restore_activation` gives back the values the bytes
stand for.  The error of an element is at most max|block| / 127 (in a block whose values are under 2^-120, at most 2^-127; in one
with a value from 127 * 2^121 on, at most 2^122).  No finite value restores as inf in the dtype it had.  A block that holds an inf
or NaN restores as NaN.

`GradSampleModule(..., activation_bits=8)` stashes Linear inputs this way.  Clipping bounds whatever gradient comes out, so the
privacy guarantee is untouched; the gradients carry the rounding of the activations.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native


class Activation8(NamedTuple):
    data: torch.Tensor      # int8, the activation's shape
    exponent: torch.Tensor  # uint8 [..., ceil(C / 128)]: k + 127 of the block's scale 2^k, 255 for a block with an inf or NaN
    dtype: torch.dtype      # what was compressed


def compress_activation(x: torch.Tensor) -> Activation8:
    """x [..., C] fp32, bf16 or fp16 on a HIP device."""
    return Activation8(*_native.compress_activation(x), x.dtype)


def restore_activation(a: Activation8, dtype: torch.dtype = None) -> torch.Tensor:
    """The values `a` stands for, in the compressed tensor's dtype or in `dtype`."""
    return _native.restore_activation(a.data, a.exponent, a.dtype if dtype is None else dtype)


def belongs_to(a: Activation8, x: torch.Tensor) -> bool:
    """Whether `a` can be `x` in 8 bits: its shape, dtype and device.  (Not whether it holds x's values.)"""
    return (isinstance(a, Activation8) and a.dtype == x.dtype and a.data.device == x.device == a.exponent.device
            and a.data.shape == x.shape and a.exponent.shape == x.shape[:-1] + (-(-x.shape[-1] // _native.ACT8_BLOCK),))
