"""What a decoder trains and serves with beside layer norm and linear: gated
feed-forward layers, the output projection with its cross entropy, and rotary
positions.

Each is one function with a backward pass on hand-written gfx950 kernels
(csrc/tam_gated.hip, csrc/tam_cross.hip, csrc/tam_rotary.hip);
csrc/tam_decoder.cpp checks the arguments and holds the autograd nodes.  The
terms of layers.py hold here too: fp32, bf16 or fp16 on a HIP device, all of a
call of one type, sums in fp32, each result rounded once, and an error for what
has no derivative.  No counterpart in the reference, which has an optimizer only.
"""

import math

import torch

from . import layers
from .layers import _ACTIVATIONS, _layers

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def gated_linear(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, *, activation: str = "silu") -> torch.Tensor:
    """act(x @ gate.T) * (x @ up.T): the first half of a gated feed-forward block.

    x (..., inputs), gate and up (outputs, inputs), all of one dtype; the result is
    (..., outputs).  Both products, the activation and their product are one kernel.
    activation: as linear's (None for a product of two projections).  Weights kept as
    (inputs, outputs) are passed as their transposed views and read in place, if both
    are.  The backward pass gives the gradients of every argument; for it the forward
    pass keeps the upper 24 bits of both products' float32 (6 bytes an output; in fp32 all
    of them, 8), and their gradients are rounded to the dtype, and have to lie in its range,
    before the products that make dx, dgate and dup."""
    if activation not in _ACTIVATIONS:
        raise ValueError("turboadam_amd.gated_linear: activation must be one of "
                         f"{sorted(k for k in _ACTIVATIONS if k)}, got {activation!r}")
    return (layers._bound or _layers()).gated_linear(x, gate, up, _ACTIVATIONS[activation])


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, reduction: str = "mean",
                         ignore_index: int = -100) -> torch.Tensor:
    """Softmax cross entropy of the logits x @ weight.T, which are never in memory as a whole (but for
    up to 64 words).

    x (..., inputs) and weight (vocabulary, inputs) of one dtype, target (...) int64.  The
    loss is fp32: of each row (reduction="none", in target's shape), their sum, or their mean
    over the rows that count.  Rows whose target is ignore_index do not: their loss is 0, their
    gradient is 0, whatever x holds there, and with more than 32 rows and 64 words they cost nothing.
    Where no row counts the sum and the mean are 0.  A target outside the vocabulary that is not
    ignore_index makes its row's loss NaN, and the gradients with it.  The backward pass makes the
    logits again, a piece of the vocabulary at a time (up to 512 MiB of their gradient), and gives
    the gradients of x and weight; softmax - onehot is rounded to the dtype before the products
    that make them."""
    if reduction not in _REDUCTIONS:
        raise ValueError("turboadam_amd.linear_cross_entropy: reduction must be one of "
                         f"{sorted(_REDUCTIONS)}, got {reduction!r}")
    return (layers._bound or _layers()).linear_cross_entropy(x, weight, target, _REDUCTIONS[reduction], int(ignore_index))


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *,
           interleaved: bool = False, magnitude: float = 1.0, q_weight: torch.Tensor = None,
           k_weight: torch.Tensor = None, eps: float = 1e-6):
    """Queries and keys turned by their positions, each head normed before, in one pass.

    q (..., tokens, heads, dim) and k of the same shape but for its heads, or None (the result is
    then the queries alone, otherwise both); dim at most 1024 (1008 where the rotated part is no
    multiple of 16).  Any strides with contiguous heads are read in place: slices of a joint
    projection, heads before tokens (passed as a transposed view; heads of 128 that lie 256 MiB or more
    apart are copied); results keep the order of dimensions.  positions (tokens,) or anything that
    broadcasts to (..., tokens), int64 or int32.  frequencies (pairs,) float64, in radians a position
    (rotary_frequencies): the first 2 * pairs elements of a head turn, the rest stays.  Pairs are elements i and i + pairs, or 2 i and 2 i + 1
    (interleaved); angles are 64-bit products.  magnitude multiplies what turns.  With q_weight
    (dim,) a query head is first divided by sqrt(mean of squares + eps) and multiplied by it; k_weight
    likewise.  eps is 0 or one of float32's normal numbers, in which the mean is taken.  The backward pass gives the gradients of q, k and the weights, those of the weights
    summed in a fixed order."""
    out = (layers._bound or _layers()).rotary(q, k, positions, frequencies, interleaved, magnitude, q_weight, k_weight, eps)
    return out[0] if k is None else (out[0], out[1])


def rotary_frequencies(dim: int, *, base: float = 10000.0, scaling: str = None, factor: float = 1.0,
                       original_length: int = None, low: float = 1.0, high: float = 4.0,
                       device=None) -> torch.Tensor:
    """Frequencies of dim / 2 pairs for rotary: base ** (-2 i / dim), float64, on `device`.

    scaling stretches them for contexts `factor` times longer than the model was trained for:
    "linear" divides all by factor; "ntk" takes base * factor ** (dim / (dim - 2)), which leaves the
    first and divides the last by factor; "bands" leaves those that turn more than `high` times in
    original_length positions, divides those that turn less than `low` times by factor, and goes over
    in between linearly in the number of turns."""
    if int(dim) != dim or dim < 2 or dim % 2:
        raise ValueError(f"turboadam_amd.rotary_frequencies: dim must be even and 2 or more, got {dim!r}")
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError(f"turboadam_amd.rotary_frequencies: base and factor must be above 0, got {base!r} and {factor!r}")
    if scaling not in (None, "linear", "ntk", "bands"):
        raise ValueError("turboadam_amd.rotary_frequencies: scaling must be None, 'linear', 'ntk' or 'bands', "
                         f"got {scaling!r}")
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("turboadam_amd.rotary_frequencies: 'ntk' needs a dim above 2")
        base = base * factor ** (dim / (dim - 2))
    f = base ** -(torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "linear":
        f = f / factor
    if scaling == "bands":
        if not original_length or original_length < 1 or not 0 <= low < high:
            raise ValueError("turboadam_amd.rotary_frequencies: 'bands' needs original_length and 0 <= low < high, got "
                             f"{original_length!r}, {low!r} and {high!r}")
        keep = ((f * (original_length / (2 * math.pi)) - low) / (high - low)).clamp(0.0, 1.0)
        f = keep * f + (1.0 - keep) * (f / factor)
    return f.to(device) if device is not None else f
