"""Muon: matrices stepped by their orthogonalised momentum, next to TurboAdam for
the other parameters.

A matrix's update is made nearly orthogonal (singular values near 1) by a few
Newton-Schulz products, on the gfx950 kernels of csrc/tam_muon.hip: every
matrix of a step in the same launches.  No counterpart in the reference.
"""

import ctypes
import math

import numpy as np
import torch
from torch.optim import Optimizer

from . import _lib
from .optimizer import _host

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_MATRIX = np.dtype(_lib.TamMatrix)
_MOST_SIDE = 65536    # of a matrix (include/turboadam_amd.h)
_WORKSPACE = 4 << 30  # bytes of workspace that one call's matrices may take together; one matrix may take more


def _check_products(what: str, coefficients, steps, eps) -> None:
    if len(coefficients) != 3 or not all(abs(float(c)) < 64 for c in coefficients):
        raise ValueError(f"turboadam_amd.{what}: coefficients must be three numbers below 64, got {coefficients!r}")
    if int(steps) != steps or not 1 <= steps <= 64:
        raise ValueError(f"turboadam_amd.{what}: steps must be 1 to 64, got {steps}")
    if not ctypes.c_float(float(eps)).value > 0:  # as the kernels take it
        raise ValueError(f"turboadam_amd.{what}: eps must be above 0 in float32, got {eps}")


def _workspace_of(table) -> np.ndarray:
    """About the bytes of workspace of each matrix."""
    small = np.minimum(table["rows"], table["cols"]).astype(np.float64)
    return 8.0 * table["rows"] * (table["cols"] + 64) + 8.0 * small * (small + 64)


def _launch(table, coefficients, steps: int, device) -> None:
    """One call per run of matrices whose workspaces fit _WORKSPACE together."""
    lib = _lib.load()
    co = (ctypes.c_float * 3)(*coefficients)
    ends, used = [], 0.0
    for i, need in enumerate(_workspace_of(table).tolist()):
        if used and used + need > _WORKSPACE:
            ends.append(i)
            used = 0.0
        used += need
    ends.append(len(table))
    need = ctypes.c_size_t()
    with torch.cuda.device(device):
        begin = 0
        for end in ends:
            part = table[begin:end]
            _lib.check(lib.tam_orthogonalize_workspace(part.ctypes.data, end - begin, ctypes.byref(need)),
                       "tam_orthogonalize_workspace")
            ws = torch.empty(need.value, dtype=torch.uint8, device=device)
            _lib.check(lib.tam_orthogonalize(part.ctypes.data, end - begin, co, steps, ws.data_ptr(), need.value,
                                             _lib.stream_of(device)), "tam_orthogonalize")
            del ws  # the next call's kernels, on the same stream, may take its memory
            begin = end


def orthogonalize(g: torch.Tensor, *, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of g (..., rows, cols), each matrix for itself.

    x = g / max(|g|, eps) with the Frobenius norm, then `steps` times
    x = a x + b (x x^T) x + c (x x^T)^2 x with (a, b, c) = coefficients, on the
    shorter side.  fp32, bf16 or fp16; the result has g's dtype.  bf16: products
    of fp16 factors with fp32 sums, an error of about 1e-3 of the result's norm
    beside the result's own rounding; fp32 and fp16: factors of 22 bits.  The
    coefficients are below 64.  The factors are held in a range: the result is
    not finite where a singular value s passes 4 before the last step, or
    a + b s^2 + c s^4 passes 15 (255 where |a| + |b| + |c| is 15 or more).  It has no backward pass: a g that requires gradients is refused
    where they are on (under no_grad, or detached, it is a constant)."""
    if not isinstance(g, torch.Tensor) or not g.is_cuda:
        got = g.device if isinstance(g, torch.Tensor) else type(g).__name__
        raise RuntimeError(f"turboadam_amd.orthogonalize: tensors must be on an MI355X (HIP) device, got {got}")
    if g.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("turboadam_amd.orthogonalize: has no backward pass, and g requires gradients: pass "
                           "g.detach() where it is meant as a constant")
    _host().check_call("orthogonalize", g)
    if g.dtype not in _lib.DTYPES:
        raise ValueError(f"turboadam_amd.orthogonalize: g must be float32, bfloat16 or float16, got {g.dtype}")
    if g.dim() < 2 or max(g.shape[-2:]) > _MOST_SIDE:
        raise ValueError(f"turboadam_amd.orthogonalize: g must be (..., rows, cols) with sides of at most "
                         f"{_MOST_SIDE}, got {tuple(g.shape)}")
    _check_products("orthogonalize", coefficients, steps, eps)
    g = g.detach().resolve_neg().contiguous()
    out = torch.empty_like(g)
    rows, cols = g.shape[-2:]
    if g.numel() == 0:
        return out
    n = g.numel() // (rows * cols)
    table = np.zeros(n, dtype=_MATRIX)
    at = np.arange(n, dtype=np.uint64) * np.uint64(rows * cols * g.element_size())
    table["out"] = at + np.uint64(out.data_ptr())
    table["grad"] = at + np.uint64(g.data_ptr())
    table["rows"], table["cols"], table["dtype"], table["eps"] = rows, cols, _lib.DTYPES[g.dtype], eps
    _launch(table, coefficients, int(steps), g.device)
    return out


class Muon(Optimizer):
    """Momentum, orthogonalised, as the step of 2-D parameters.

    Per matrix (rows, cols), with m the fp32 momentum and g the gradient:
        m = momentum m + (1 - momentum) g
        u = (1 - momentum) g + momentum m   (nesterov; else u = m)
        p = (1 - lr weight_decay) p - lr adjust orthogonalize(u)
    adjust_lr: "original", adjust = sqrt(max(1, rows / cols)), or
    "match_rms_adamw", adjust = 0.2 sqrt(max(rows, cols)), with which Adam's
    learning rate and weight decay fit.  A model's vectors, embeddings and head
    belong to TurboAdam.

    Parameters are contiguous 2-D tensors on a HIP device, fp32, bf16 or fp16,
    their gradients of the same dtype.  The parameter is updated in fp32 and
    rounded once.  State: state[p]["momentum_buffer"], fp32."""

    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95,
                 nesterov: bool = True, ns_coefficients: tuple = COEFFICIENTS, eps: float = 1e-7, ns_steps: int = 5,
                 adjust_lr: str = "original"):
        defaults = dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                        ns_coefficients=tuple(ns_coefficients), eps=eps, ns_steps=ns_steps, adjust_lr=adjust_lr)
        super().__init__(params, defaults)

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
        except Exception:  # also a setting of a wrong type
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(group: dict) -> None:
        for p in group["params"]:
            if p.dim() != 2:
                raise ValueError(f"turboadam_amd.Muon: parameters must be matrices (2-D), got {tuple(p.shape)}")
            if max(p.shape) > _MOST_SIDE:
                raise ValueError(f"turboadam_amd.Muon: a side of more than {_MOST_SIDE}: {tuple(p.shape)}")
        if not group["lr"] >= 0:
            raise ValueError(f"turboadam_amd.Muon: lr must be 0 or more, got {group['lr']}")
        if not group["weight_decay"] >= 0:
            raise ValueError(f"turboadam_amd.Muon: weight_decay must be 0 or more, got {group['weight_decay']}")
        if not 0 <= group["momentum"] < 1:
            raise ValueError(f"turboadam_amd.Muon: momentum must be in [0, 1), got {group['momentum']}")
        if group["adjust_lr"] not in ("original", "match_rms_adamw"):
            raise ValueError("turboadam_amd.Muon: adjust_lr must be 'original' or 'match_rms_adamw', got "
                             f"{group['adjust_lr']!r}")
        _check_products("Muon", group["ns_coefficients"], group["ns_steps"], group["eps"])

    def _row(self, p, group):
        """One parameter's row of the table (TamMatrix without its last field)."""
        g = p.grad
        if not p.is_cuda:
            raise RuntimeError(f"turboadam_amd.Muon: parameters must be on an MI355X (HIP) device, got {p.device}")
        if p.dtype not in _lib.DTYPES:
            raise RuntimeError(f"turboadam_amd.Muon: parameters must be float32, bfloat16 or float16, got {p.dtype}")
        if not p.is_contiguous() or p.is_neg():
            raise RuntimeError("turboadam_amd.Muon: parameters must be contiguous")
        if g.layout != torch.strided or g.dtype != p.dtype or g.device != p.device or g.shape != p.shape:
            raise RuntimeError(f"turboadam_amd.Muon: the gradient of a {p.dtype} parameter {tuple(p.shape)} on "
                               f"{p.device} must be dense and like it, got {g.layout} {g.dtype} {tuple(g.shape)} on "
                               f"{g.device}")
        st = self.state[p]
        m = st.get("momentum_buffer")
        if m is None:
            m = st["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        elif (m.dtype != torch.float32 or m.device != p.device or m.shape != p.shape or not m.is_contiguous()
              or m.is_neg()):
            raise RuntimeError(f"turboadam_amd.Muon: the momentum_buffer of a parameter {tuple(p.shape)} on {p.device} "
                               f"must be contiguous float32 like it, got {m.dtype} {tuple(m.shape)} on {m.device}")
        if not g.is_contiguous() or g.is_neg():
            g = g.resolve_neg().contiguous()
        rows, cols = p.shape
        lr, keep = float(group["lr"]), float(group["momentum"])
        adjust = (math.sqrt(max(1.0, rows / cols)) if group["adjust_lr"] == "original"
                  else 0.2 * math.sqrt(max(rows, cols)))
        flags = _lib.TAM_MATRIX_UPDATE | (_lib.TAM_MATRIX_NESTEROV if group["nesterov"] else 0)
        return (p.data_ptr(), g.data_ptr(), m.data_ptr(), rows, cols, _lib.DTYPES[p.dtype], flags, keep, 1.0 - keep,
                float(group["eps"]), 1.0 - lr * float(group["weight_decay"]), lr * adjust, 0), g

    @torch.no_grad()
    def step(self, closure=None):
        """One step of every parameter with a gradient; queued on the current stream."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = {}  # matrices that share a device and the products' settings go together
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                row, g = self._row(p, group)
                key = (p.device, tuple(group["ns_coefficients"]), int(group["ns_steps"]))
                rows, held, written = calls.setdefault(key, ([], [], []))
                rows.append(row)
                held.append(g)
                written += (p, self.state[p]["momentum_buffer"])
        for (device, coefficients, steps), (rows, held, written) in calls.items():
            _launch(np.array(rows, dtype=_MATRIX), coefficients, steps, device)
            # a graph that kept one of them must not use it as if it were what it was
            torch.autograd.graph.increment_version(written)
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch.optim.Optimizer's, the momenta in fp32 whatever the parameters' dtype."""
        super().load_state_dict(state_dict)
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(saved, params):
            m = state_dict["state"].get(i, {}).get("momentum_buffer")
            if m is not None:
                self.state[p]["momentum_buffer"] = m.detach().to(p.device, torch.float32, copy=True).contiguous()
