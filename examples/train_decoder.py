"""Training a small decoder with the package's layers and optimizers.

Layer norms, a joint projection of queries, keys and values, rotary positions with
normed heads, a gated feed-forward block and the output projection with its cross
entropy run on the package's kernels, forward and backward; attention itself is plain
torch in fp32. Matrices are stepped by Muon, embeddings and vectors by TurboAdam. The
text is made by a fixed random chain of words; the first words of a sequence, a prompt,
are not predicted (their targets are ignored).

    python examples/train_decoder.py [--dim 256] [--layers 2] [--steps 60] [--dtype bf16]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from turboadam_amd import (  # noqa: E402
    Muon, TurboAdam, gated_linear, layer_norm, linear, linear_cross_entropy, rotary, rotary_frequencies)

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HEAD = 64


class Layer(torch.nn.Module):
    def __init__(self, dim: int, dtype, generator):
        super().__init__()
        self.heads, self.kv_heads = dim // HEAD, max(1, dim // HEAD // 2)

        def matrix(rows, cols):
            w = torch.randn(rows, cols, generator=generator, device="cuda") * cols ** -0.5
            return torch.nn.Parameter(w.to(dtype))

        def vector(n):
            return torch.nn.Parameter(torch.ones(n, device="cuda", dtype=dtype))

        self.qkv = matrix((self.heads + 2 * self.kv_heads) * HEAD, dim)
        self.out = matrix(dim, self.heads * HEAD)
        self.gate, self.up, self.down = matrix(2 * dim, dim), matrix(2 * dim, dim), matrix(dim, 2 * dim)
        self.norm1, self.norm2, self.q_norm, self.k_norm = vector(dim), vector(dim), vector(HEAD), vector(HEAD)

    def forward(self, x, positions, frequencies):
        heads, kv = self.heads, self.kv_heads
        q, k, v = linear(layer_norm(x, self.norm1), self.qkv).unflatten(-1, (-1, HEAD)).split((heads, kv, kv), -2)
        q, k = rotary(q, k, positions, frequencies, q_weight=self.q_norm, k_weight=self.k_norm)
        x = linear(attention(q, k, v).to(x.dtype), self.out, residual=x)
        return linear(gated_linear(layer_norm(x, self.norm2), self.gate, self.up), self.down, residual=x)


def attention(q, k, v):
    """Causal attention of (batch, tokens, heads, HEAD), in fp32; keys and values shared by groups of heads."""
    groups = q.shape[2] // k.shape[2]
    q, k, v = [t.float().transpose(1, 2).contiguous() for t in (q, k.repeat_interleave(groups, 2), v.repeat_interleave(groups, 2))]
    scores = torch.matmul(q, k.mT.contiguous()) * HEAD ** -0.5
    mask = torch.ones(scores.shape[-2:], dtype=torch.bool, device=q.device).triu(1)
    return torch.matmul(scores.masked_fill(mask, float("-inf")).softmax(-1), v).transpose(1, 2).flatten(2)


class Decoder(torch.nn.Module):
    def __init__(self, dim: int, layers: int, words: int, dtype, generator):
        super().__init__()
        self.embedding = torch.nn.Parameter(torch.randn(words, dim, generator=generator, device="cuda").to(dtype))
        self.layers = torch.nn.ModuleList(Layer(dim, dtype, generator) for _ in range(layers))
        self.norm = torch.nn.Parameter(torch.ones(dim, device="cuda", dtype=dtype))
        self.head = torch.nn.Parameter((torch.randn(words, dim, generator=generator, device="cuda") * dim ** -0.5).to(dtype))
        self.frequencies = rotary_frequencies(HEAD, device="cuda")

    def loss(self, text, prompt: int):
        """The mean loss of each word behind the prompt, given those ahead of it."""
        x = self.embedding[text[:, :-1]]
        positions = torch.arange(x.shape[1], device=x.device)
        for layer in self.layers:
            x = layer(x, positions, self.frequencies)
        target = text[:, 1:].clone()
        target[:, :prompt] = -100
        return linear_cross_entropy(layer_norm(x, self.norm), self.head, target)


def make_text(generator, chain, sequences: int, length: int):
    """Sequences in which each word is followed by one of four."""
    words = [torch.randint(0, len(chain), (sequences,), generator=generator, device="cuda")]
    for _ in range(length - 1):
        which = torch.randint(0, chain.shape[1], (sequences,), generator=generator, device="cuda")
        words.append(chain[words[-1], which])
    return torch.stack(words, 1)


def train(dim: int = 256, layers: int = 2, words: int = 1000, sequences: int = 16, length: int = 129, steps: int = 60,
          dtype: str = "bf16", log=print) -> list:
    """The losses of `steps` steps."""
    g = torch.Generator(device="cuda").manual_seed(0)
    model = Decoder(dim, layers, words, DTYPES[dtype], g)
    chain = torch.randint(0, words, (words, 4), generator=g, device="cuda")
    matrices = [p for p in model.layers.parameters() if p.dim() == 2]
    others = [p for p in model.parameters() if all(p is not m for m in matrices)]
    optimizers = [Muon(matrices, lr=0.02, weight_decay=0.0), TurboAdam(others, lr=3e-3)]
    losses = []
    for step in range(steps):
        loss = model.loss(make_text(g, chain, sequences, length), prompt=8)
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
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    train(**vars(ap.parse_args()))
