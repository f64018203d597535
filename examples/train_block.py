"""Training one transformer MLP block with the package's layers and optimizers.

    x + W2 gelu(W1 norm(x) + b1) + b2

is fitted to a fixed teacher of the same form: layer norm, two linear layers
(activation, bias and residual in their products' epilogues) and their gradients
run on the package's kernels; the two matrices are stepped by Muon, the vectors
by TurboAdam.

    python examples/train_block.py [--dim 256] [--tokens 2048] [--steps 60] [--dtype bf16]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from turboadam_amd import Muon, TurboAdam, layer_norm, linear  # noqa: E402

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


class Block(torch.nn.Module):
    def __init__(self, dim: int, dtype, generator):
        super().__init__()

        def matrix(rows, cols):
            w = torch.randn(rows, cols, generator=generator, device="cuda") * cols ** -0.5
            return torch.nn.Parameter(w.to(dtype))

        def vector(n, value):
            return torch.nn.Parameter(torch.full((n,), value, device="cuda", dtype=dtype))

        self.up, self.down = matrix(4 * dim, dim), matrix(dim, 4 * dim)
        self.scale, self.shift = vector(dim, 1.0), vector(dim, 0.0)
        self.up_bias, self.down_bias = vector(4 * dim, 0.0), vector(dim, 0.0)

    def forward(self, x):
        h = layer_norm(x, self.scale, self.shift)
        h = linear(h, self.up, self.up_bias, activation="gelu_tanh")
        return linear(h, self.down, self.down_bias, residual=x)


def train(dim: int = 256, tokens: int = 2048, steps: int = 60, dtype: str = "bf16", log=print) -> list:
    """The losses of `steps` steps."""
    g = torch.Generator(device="cuda").manual_seed(0)
    teacher, student = Block(dim, DTYPES[dtype], g), Block(dim, DTYPES[dtype], g)
    matrices = [p for p in student.parameters() if p.dim() == 2]
    vectors = [p for p in student.parameters() if p.dim() == 1]
    optimizers = [Muon(matrices, lr=0.02, weight_decay=0.0), TurboAdam(vectors, lr=1e-3)]
    losses = []
    for step in range(steps):
        x = torch.randn(tokens, dim, generator=g, device="cuda").to(DTYPES[dtype])
        with torch.no_grad():
            target = teacher(x)
        loss = (student(x).float() - target.float()).square().mean()
        for opt in optimizers:
            opt.zero_grad()
        loss.backward()
        for opt in optimizers:
            opt.step()
        losses.append(loss.detach())
        if step % 10 == 0 or step + 1 == steps:
            log(f"step {step:3d}  loss {losses[-1].item():.5f}")
    return [v.item() for v in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--dim", type=int, default=256)
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    train(**vars(ap.parse_args()))
