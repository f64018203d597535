"""Layers whose gradients the optimizers step with: linear and layer norm.

Each is one function with a backward pass on hand-written gfx950 kernels
(csrc/tam_linear.hip, csrc/tam_norm.hip).  Tensors are fp32, bf16 or fp16 on a
HIP device; sums and statistics are fp32, and every result is rounded to its
type once.  No counterpart in the reference, which has an optimizer only.
"""

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_MOST_STRIDE = 1 << 21  # elements of a row stride the kernels take (include/turboadam_amd.h)


def _check(what: str, x, others) -> None:
    """x's and the other tensors' (name, tensor or None) device and dtype."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        got = x.device if isinstance(x, torch.Tensor) else type(x).__name__
        raise RuntimeError(f"turboadam_amd.{what}: tensors must be on an MI355X (HIP) device, got {got}")
    if x.dtype not in _lib.DTYPES:
        raise ValueError(f"turboadam_amd.{what}: x must be float32, bfloat16 or float16, got {x.dtype}")
    for name, t in others:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.device != x.device:
            got = t.device if isinstance(t, torch.Tensor) else type(t).__name__
            raise RuntimeError(f"turboadam_amd.{what}: {name} must be on {x.device} with x, got {got}")
        if t.dtype != x.dtype:
            raise ValueError(f"turboadam_amd.{what}: {name} must be {x.dtype} as x is, got {t.dtype}")


def _plain(t: torch.Tensor) -> torch.Tensor:
    """t as memory holds it: contiguous, its negative bit resolved."""
    return t.resolve_neg().contiguous()


def _rows(t: torch.Tensor, width: int):
    """t as (rows, width) with contiguous rows, and the stride between them."""
    n = math.prod(t.shape[:-1])
    t = t.resolve_neg().reshape(n, width)
    if width != 1 and t.stride(1) != 1 or n > 1 and not width <= t.stride(0) < _MOST_STRIDE:
        t = t.contiguous()
    return t, (t.stride(0) if n > 1 else max(width, 1))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------ linear
def _weight(weight: torch.Tensor):
    """(the weight, its row stride, whether its rows are the inputs): a weight
    stored as (inputs, outputs) and passed as its transpose stays where it is."""
    w = weight.resolve_neg()
    outputs, inputs = w.shape
    if (inputs == 1 or w.stride(1) == 1) and (outputs == 1 or inputs <= w.stride(0) < _MOST_STRIDE):
        return w, (w.stride(0) if outputs > 1 else max(inputs, 1)), 0
    if (outputs == 1 or w.stride(0) == 1) and (inputs == 1 or outputs <= w.stride(1) < _MOST_STRIDE):
        return w, (w.stride(1) if inputs > 1 else max(outputs, 1)), 1
    return w.contiguous(), max(inputs, 1), 0


def _describe(x2, ldx, weight, ldw, in_out, activation):
    d = _lib.TamLinear()
    d.x, d.w = x2.data_ptr(), weight.data_ptr()
    d.rows, d.inputs, d.outputs = x2.shape[0], x2.shape[1], weight.shape[0]
    d.ldx, d.ldw, d.w_in_out = ldx, ldw, in_out
    d.dtype, d.activation = _lib.DTYPES[x2.dtype], activation
    return d


def _run(d, backward: bool, device) -> None:
    lib = _lib.load()
    name = "tam_linear_backward" if backward else "tam_linear"
    with torch.cuda.device(device):
        need = ctypes.c_size_t()
        _lib.check(lib.tam_linear_workspace(ctypes.byref(d), int(backward), ctypes.byref(need)), name)
        ws = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
        _lib.check(getattr(lib, name)(ctypes.byref(d), _ptr(ws), need.value, _lib.stream_of(device)), name)


def _linear_forward(x, weight, bias, residual, activation, keep_z):
    x2, ldx = _rows(x, weight.shape[1])
    w, ldw, in_out = _weight(weight)
    d = _describe(x2, ldx, w, ldw, in_out, activation)
    shape = x.shape[:-1] + (weight.shape[0],)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    z = torch.empty(shape, dtype=x.dtype, device=x.device) if keep_z and activation else None
    bias = None if bias is None else _plain(bias)
    residual = None if residual is None else _plain(residual)
    d.bias, d.residual, d.y, d.z = _ptr(bias), _ptr(residual), y.data_ptr(), _ptr(z)
    _run(d, False, x.device)
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        keep_z = any(ctx.needs_input_grad[:3])
        y, z = _linear_forward(x, weight, bias, residual, activation, keep_z)
        ctx.save_for_backward(x, weight, z)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            x2, ldx = _rows(x, weight.shape[1])
            w, ldw, in_out = _weight(weight)
            d = _describe(x2, ldx, w, ldw, in_out, ctx.activation)
            g = _plain(dy)
            if need_x:
                dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            if need_w:  # laid out as the weight
                shape = (weight.shape[1], weight.shape[0]) if in_out else tuple(weight.shape)
                dw = torch.empty(shape, dtype=x.dtype, device=x.device)
            if need_b:
                db = torch.empty(weight.shape[0], dtype=x.dtype, device=x.device)
            d.dy, d.z, d.dx, d.dw, d.db = g.data_ptr(), _ptr(z), _ptr(dx), _ptr(dw), _ptr(db)
            if dx is not None and weight.shape[1] and not weight.shape[0]:
                dx.zero_()
            _run(d, True, x.device)
            if need_w and in_out:
                dw = dw.t()
        return dx, dw, db, dy if need_r else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor = None, *, activation: str = None,
           residual: torch.Tensor = None) -> torch.Tensor:
    """act(x @ weight.T + bias) + residual, in one product with its epilogue.

    x (..., inputs), weight (outputs, inputs), bias (outputs), residual (...,
    outputs), all of one dtype; the result is (..., outputs).  activation: None,
    "relu", "gelu" (by erf), "gelu_tanh" or "silu".  A weight kept as (inputs,
    outputs) is passed as its transposed view and read in place.  The backward
    pass gives the gradients of every argument; where there is an activation,
    the forward pass keeps its argument, rounded to the dtype, for it."""
    _check("linear", x, (("weight", weight), ("bias", bias), ("residual", residual)))
    if activation not in _ACTIVATIONS:
        raise ValueError(f"turboadam_amd.linear: activation must be one of {sorted(k for k in _ACTIVATIONS if k)}, "
                         f"got {activation!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"turboadam_amd.linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} are not "
                         "(..., inputs) and (outputs, inputs)")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"turboadam_amd.linear: bias must have shape ({weight.shape[0]},), got {tuple(bias.shape)}")
    if residual is not None and residual.shape != x.shape[:-1] + weight.shape[:1]:
        raise ValueError(f"turboadam_amd.linear: residual must have the result's shape "
                         f"{tuple(x.shape[:-1] + weight.shape[:1])}, got {tuple(residual.shape)}")
    act = _ACTIVATIONS[activation]
    if _need(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, act)
    return _linear_forward(x, weight, bias, residual, act, False)[0]


# -------------------------------------------------------------- layer norm
_MOST_NORM = 32768  # elements of a row the kernels take (include/turboadam_amd.h)


def _norm_operands(x, weight, bias, eps):
    d = _lib.TamNorm()
    n = x.shape[-1]
    x2, ldx = _rows(x, n)
    weight = None if weight is None else _plain(weight)
    bias = None if bias is None else _plain(bias)
    d.x, d.w, d.b = x2.data_ptr(), _ptr(weight), _ptr(bias)
    d.rows, d.n, d.ldx, d.dtype, d.eps = x2.shape[0], n, ldx, _lib.DTYPES[x.dtype], eps
    return d, (x2, weight, bias)


def _norm_forward(x, weight, bias, eps, keep):
    lib = _lib.load()
    d, operands = _norm_operands(x, weight, bias, eps)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((d.rows, 2), dtype=torch.float32, device=x.device) if keep else None
    d.y, d.stats = y.data_ptr(), _ptr(stats)
    with torch.cuda.device(x.device):
        _lib.check(lib.tam_norm(ctypes.byref(d), _lib.stream_of(x.device)), "tam_norm")
    del operands
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.eps = eps
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        lib = _lib.load()
        d, operands = _norm_operands(x, weight, None, ctx.eps)
        n, dev = x.shape[-1], x.device
        g = _plain(dy)
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        dw = torch.empty(n, dtype=x.dtype, device=dev) if need_w else None
        db = torch.empty(n, dtype=x.dtype, device=dev) if need_b else None
        d.dy, d.stats, d.dx, d.dw, d.db = g.data_ptr(), stats.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db)
        with torch.cuda.device(dev):
            need = ctypes.c_size_t()
            _lib.check(lib.tam_norm_workspace(ctypes.byref(d), 1, ctypes.byref(need)), "tam_norm_workspace")
            ws = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
            _lib.check(lib.tam_norm_backward(ctypes.byref(d), _ptr(ws), need.value, _lib.stream_of(dev)),
                       "tam_norm_backward")
        del operands
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x (..., n) with n at most 32768, weight and bias (n) or None, all of one
    dtype.  The mean and the variance (the mean squared distance from the mean)
    are fp32 sums over a row held in registers, kept in fp32 for the backward
    pass, which gives the gradients of x, weight and bias; those of weight and
    bias are summed over the rows in a fixed order."""
    _check("layer_norm", x, (("weight", weight), ("bias", bias)))
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MOST_NORM:
        raise ValueError(f"turboadam_amd.layer_norm: x must have rows of 1 to {_MOST_NORM} elements, got "
                         f"{tuple(x.shape)}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != x.shape[-1:]:
            raise ValueError(f"turboadam_amd.layer_norm: {name} must have shape ({x.shape[-1]},), got "
                             f"{tuple(t.shape)}")
    if not eps >= 0:
        raise ValueError(f"turboadam_amd.layer_norm: eps must be 0 or more, got {eps}")
    if _need(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _norm_forward(x, weight, bias, float(eps), False)[0]
