"""Layers whose gradients the optimizers step with: linear and layer norm.

Each is one function with a backward pass on hand-written gfx950 kernels
(csrc/tam_linear.hip, csrc/tam_norm.hip); csrc/tam_layers.cpp checks the
arguments and holds the autograd nodes.  Tensors are fp32, bf16 or fp16 on a HIP
device, all of a call of one type (autocast casts nothing here); sums and
statistics are fp32, and every result is rounded to its type once.  Forward-mode
derivatives, a second backward pass and recording by torch.jit.trace or make_fx
raise.  No counterpart in the reference, which has an optimizer only.
"""

import ctypes

import torch

from . import _lib
from .optimizer import _host

_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_ENTRIES = ("tam_linear_workspace", "tam_linear", "tam_linear_backward", "tam_norm_workspace", "tam_norm",
            "tam_norm_backward", "tam_last_error")

_bound = None


def _layers():
    """The host module, with the library's entries bound."""
    global _bound
    if _bound is None:
        lib, mod = _lib.load(), _host()
        mod.bind_layers({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _ENTRIES})
        _bound = mod
    return _bound


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor = None, *, activation: str = None,
           residual: torch.Tensor = None) -> torch.Tensor:
    """act(x @ weight.T + bias) + residual, in one product with its epilogue.

    x (..., inputs), weight (outputs, inputs), bias (outputs), residual (...,
    outputs), all of one dtype; the result is (..., outputs).  activation: None,
    "relu", "gelu" (by erf), "gelu_tanh" or "silu".  A weight kept as (inputs,
    outputs) is passed as its transposed view and read in place.  The backward
    pass gives the gradients of every argument.  Where there is an activation,
    the forward pass keeps its argument z for it, and it hands dy act'(z) to
    the products that make dx and dweight, both rounded to the dtype: in bf16
    these are about 2.4e-3 of their norm off, 1.7e-3 of it their own rounding."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"turboadam_amd.linear: activation must be one of {sorted(k for k in _ACTIVATIONS if k)}, "
                         f"got {activation!r}")
    return (_bound or _layers()).linear(x, weight, bias, residual, _ACTIVATIONS[activation])


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x (..., n) with n at most 32768, weight and bias (n) or None, all of one
    dtype.  The mean and the variance (the mean squared distance from the mean)
    are fp32 sums over a row held in registers, kept in fp32 for the backward
    pass, which gives the gradients of x, weight and bias; those of weight and
    bias are summed over the rows in a fixed order."""
    return (_bound or _layers()).layer_norm(x, weight, bias, eps)
