"""Performance cases of a decoder's layers beside layer norm and linear.

Three operators that a model of this kind trains and serves with:

* ``gated_linear`` (kind "gated"): act(x gate^T) * (x up^T), the first half of a
  gated feed-forward block, with its backward pass and its form for single tokens;
* ``linear_cross_entropy`` (kind "cross"): the output projection and the softmax
  cross entropy over the vocabulary in one, with its backward pass;
* ``rotary`` (kind "rotary"): the norm of each query and key head and the rotation
  by its position, with its backward pass.

``run`` computes a pass in plain torch operations in 32 bits (angles in 64),
rounded once at the end, or (``own``) through the package's entry points.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORE = -100
EPS = 1e-6


# ------------------------------------------------------------------ cases
def _gated(name, rows, inputs, outputs, dtype, train, activation="silu", in_out=False):
    return dict(name=name, kind="gated", rows=rows, inputs=inputs, outputs=outputs, dtype=dtype, train=train,
                activation=activation, in_out=in_out)


def _cross(name, rows, inputs, vocabulary, dtype, train, reduction="mean", ignored=0.0):
    return dict(name=name, kind="cross", rows=rows, inputs=inputs, vocabulary=vocabulary, dtype=dtype, train=train,
                reduction=reduction, ignored=ignored)


def _rotary(name, batch, tokens, heads, kv_heads, dim, rotated, dtype, train, norm=False, interleaved=False, start=0,
            heads_first=False, base=10000.0, factor=1.0):
    return dict(name=name, kind="rotary", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                rotated=rotated, dtype=dtype, train=train, norm=norm, interleaved=interleaved, start=start,
                heads_first=heads_first, base=base, factor=factor)


def listed():
    return [
        # one token being generated by an 8B-shaped model: reading both weights once
        _gated("gated_token_bf16", 1, 4096, 14336, "bf16", False),
        # the same model's layer in training, 8 sequences of 1024 tokens
        _gated("gated_train_bf16", 8192, 4096, 14336, "bf16", True),
        # a small fp16 model of GPT-2's width, weights stored inputs by outputs
        _gated("gated_small_f16", 2048, 768, 2048, "f16", True, activation="gelu_tanh", in_out=True),
        # fp32, every size a multiple of nothing
        _gated("gated_odd_f32", 1531, 777, 1001, "f32", True, activation="gelu"),
        # the likelihood of one token over an 8B-shaped model's vocabulary
        _cross("cross_token_bf16", 1, 4096, 128256, "bf16", False, reduction="none"),
        # GPT-2's head in training, 8 sequences of 1024 tokens
        _cross("cross_gpt2_bf16", 8192, 768, 50257, "bf16", True),
        # an 8B-shaped model's head in training: a sixteenth of the tokens is padding
        _cross("cross_8b_bf16", 8192, 4096, 128256, "bf16", True, ignored=0.0625),
        # fp32, odd sizes, a loss and a gradient for each row, half of them prompts that do not count
        _cross("cross_odd_f32", 1237, 515, 9973, "f32", True, reduction="none", ignored=0.5),
        # one token being generated, far into its context: nothing but latency
        _rotary("rotary_token_bf16", 1, 1, 32, 8, 128, 128, "bf16", False, norm=True, start=131071, base=500000.0),
        # an 8B-shaped layer's queries and keys in training, slices of one projection's output
        _rotary("rotary_train_bf16", 8, 2048, 32, 8, 128, 128, "bf16", True, norm=True, base=500000.0),
        # GPT-2's heads in fp32, heads before tokens, pairs side by side
        _rotary("rotary_gpt2_f32", 8, 1024, 12, 12, 64, 64, "f32", True, interleaved=True, heads_first=True),
        # a part of odd-sized heads, a stretched context, fp16
        _rotary("rotary_odd_f16", 3, 413, 7, 3, 84, 20, "f16", True, norm=True, start=70001, factor=8.0),
    ]


def draw(rng):
    def size(lo, hi):
        return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))

    kind = rng.choice(["gated", "cross", "rotary"])
    dtype = rng.choice(list(DTYPES))
    slower = 12 if dtype == "f32" else 1  # fp32 products are that much slower
    train = rng.random() < 0.6
    if kind == "gated":
        # relu's slope jumps at 0: there the gradients of two right 32-bit sums differ by whole terms
        acts = ["none", "gelu", "gelu_tanh", "silu"] + ([] if train else ["relu"])
        c = _gated("", size(1, 16384), size(16, 8192), size(16, 16384), dtype, train, rng.choice(acts),
                   rng.random() < 0.3)
        while c["rows"] * c["inputs"] * c["outputs"] * slower > 8192 * 4096 * 14336:
            c["rows"] = max(1, c["rows"] // 2)
    elif kind == "cross":
        c = _cross("", size(1, 16384), size(16, 8192), size(2, 131072), dtype, train,
                   rng.choice(["mean", "sum", "none"]), rng.choice([0.0, 0.1, 0.5, 0.9]))
        while c["rows"] * c["inputs"] * c["vocabulary"] * slower > 4096 * 4096 * 65536:
            c["rows"] = max(1, c["rows"] // 2)
    else:
        heads, dim = size(1, 64), size(8, 512)
        rotated = 2 * rng.randint(1, dim // 2) if rng.random() < 0.4 else dim // 2 * 2
        c = _rotary("", size(1, 8), size(1, 8192), heads, rng.randint(1, heads), dim, rotated, dtype, train,
                    rng.random() < 0.6, rng.random() < 0.5, rng.choice([0, size(1, 1000000)]), rng.random() < 0.4,
                    rng.choice([10000.0, 500000.0]), rng.choice([1.0, 4.0, 16.0]))
        while c["batch"] * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"] > 16384 * 40 * 128 // 2:
            c["tokens"] = max(1, c["tokens"] // 2)
            c["batch"] = max(1, c["batch"] - 1)
            c["heads"] = max(c["kv_heads"], c["heads"] - 1)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _normed(g, rows, dim):
    """What a norm hands to a projection: rows of about unit variance, channels of their own scale."""
    return _randn(g, rows, dim).mul_(torch.exp(0.2 * _randn(g, dim)))


def prepare(case, seed):
    g, dtype = _gen(seed), DTYPES[case["dtype"]]
    s = dict(case)
    if case["kind"] == "gated":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        s["x"] = _normed(g, m, k).to(dtype)
        for name in ("gate", "up"):
            w = _randn(g, k, n) if case["in_out"] else _randn(g, n, k)
            w = w.mul_(1.0 / math.sqrt(k)).to(dtype)
            s[name] = w.t() if case["in_out"] else w
        if case["train"]:
            s["dy"] = (0.1 * _randn(g, m, n)).to(dtype)
        leaves = ("x", "gate", "up")
    elif case["kind"] == "cross":
        m, k, v = case["rows"], case["inputs"], case["vocabulary"]
        w = _randn(g, v, k).mul_(2.0 / math.sqrt(k))
        target = torch.randint(0, v, (m,), generator=g, device="cuda")
        # a model half way: on some rows it is sure of the target, on others not
        sure = torch.rand((m, 1), generator=g, device="cuda") * 3.0
        s["x"] = _normed(g, m, k).add_(w[target] * sure).to(dtype)
        s["weight"] = w.to(dtype)
        s["target"] = torch.where(torch.rand((m,), generator=g, device="cuda") < case["ignored"],
                                  torch.full_like(target, IGNORE), target)
        if case["train"]:
            scale = 1024.0 if case["dtype"] == "f16" else 1.0  # fp16 trains with a scaled loss
            if case["reduction"] == "none":
                s["dloss"] = torch.rand((m,), generator=g, device="cuda").add_(0.5).mul_(scale / m)
            else:
                s["dloss"] = torch.full((), scale if case["reduction"] == "mean" else scale / m, device="cuda")
        leaves = ("x", "weight")
    else:
        b, t, d = case["batch"], case["tokens"], case["dim"]
        hq, hk = case["heads"], case["kv_heads"]
        if case["heads_first"]:
            q, k = _randn(g, b, hq, t, d).to(dtype), _randn(g, b, hk, t, d).to(dtype)
            s["q"], s["k"] = q.transpose(1, 2), k.transpose(1, 2)
        else:  # slices of the projection that makes queries, keys and values
            qkv = _randn(g, b, t, (hq + 2 * hk) * d).to(dtype)
            s["q"] = qkv[..., :hq * d].unflatten(-1, (hq, d))
            s["k"] = qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
        s["positions"] = torch.arange(case["start"], case["start"] + t, device="cuda")
        # a linearly stretched context: angles as if positions were closer together
        powers = torch.arange(0, case["rotated"], 2, dtype=torch.float64, device="cuda") / case["rotated"]
        s["frequencies"] = case["base"] ** -powers / case["factor"]
        for name in ("q_weight", "k_weight"):
            s[name] = (1.0 + 0.1 * _randn(g, d)).to(dtype) if case["norm"] else None
        if case["train"]:
            s["dq"] = (0.1 * _randn(g, b, t, hq, d)).to(dtype)
            s["dk"] = (0.1 * _randn(g, b, t, hk, d)).to(dtype)
        leaves = ("q", "k", "q_weight", "k_weight")
    s["leaves"] = [name for name in leaves if s.get(name) is not None]
    if own and case["train"]:
        for name in s["leaves"]:
            s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------ the pass
def run(s):
    return {"gated": _run_gated, "cross": _run_cross, "rotary": _run_rotary}[s["kind"]](s)


def _gradients(s, outputs, grads):
    names = s["leaves"]
    return {"d_" + n: d for n, d in zip(names, torch.autograd.grad(outputs, [s[n] for n in names], grads))}


def _activation(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).float()
    if name == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return sig * (1.0 + z * (1.0 - sig))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _run_gated(s):
    if own:
        from turboadam_amd import gated_linear

        h = gated_linear(s["x"], s["gate"], s["up"], activation=s["activation"])
        return {"h": h, **_gradients(s, h, s["dy"])} if s["train"] else h
    dtype = s["x"].dtype
    x, wg, wu = s["x"].float(), s["gate"].float(), s["up"].float()
    z, u = x @ wg.t(), x @ wu.t()
    a = _activation(z, s["activation"])
    if not s["train"]:
        return (a * u).to(dtype)
    dy = s["dy"].float()
    dz, du = dy * u * _slope(z, s["activation"]), dy * a
    return {"h": (a * u).to(dtype), "d_x": (dz @ wg + du @ wu).to(dtype), "d_gate": (dz.t() @ x).to(dtype),
            "d_up": (du.t() @ x).to(dtype)}


def _run_cross(s):
    if own:
        from turboadam_amd import linear_cross_entropy

        loss = linear_cross_entropy(s["x"], s["weight"], s["target"], reduction=s["reduction"], ignore_index=IGNORE)
        return {"loss": loss, **_gradients(s, loss, s["dloss"])} if s["train"] else loss
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    counts = s["target"] != IGNORE
    at = torch.where(counts, s["target"], torch.zeros_like(s["target"]))[:, None]
    z = x @ w.t()
    top = z.amax(1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(1, keepdim=True)
    loss = torch.where(counts, (torch.log(total) + top - z.gather(1, at))[:, 0], torch.zeros_like(top[:, 0]))
    number = counts.sum().clamp(min=1)
    reduced = loss if s["reduction"] == "none" else loss.sum()
    if s["reduction"] == "mean":
        reduced = reduced / number
    if not s["train"]:
        return reduced
    del z
    weight = s["dloss"] / number if s["reduction"] == "mean" else s["dloss"]
    p.div_(total)
    p.scatter_add_(1, at, torch.full_like(top, -1.0))
    p.mul_((weight * counts)[:, None])
    return {"loss": reduced, "d_x": (p @ w).to(dtype), "d_weight": (p.t() @ x).to(dtype)}


def _pairs(x, rotated, interleaved):
    if interleaved:
        return x[..., 0:rotated:2], x[..., 1:rotated:2]
    return x[..., :rotated // 2], x[..., rotated // 2:rotated]


def _join(a, b, x, rotated, interleaved):
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., rotated:]), -1)


def _run_rotary(s):
    if own:
        from turboadam_amd import rotary

        q, k = rotary(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=s["interleaved"],
                      q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        return {"q": q, "k": k, **_gradients(s, (q, k), (s["dq"], s["dk"]))} if s["train"] else {"q": q, "k": k}
    dtype, rotated = s["q"].dtype, s["rotated"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    out, grads = {}, {}
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "_weight"]
        n = x
        if w is not None:
            rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            n = x * rstd * w.float()
        a, b = _pairs(n, rotated, s["interleaved"])
        out[name] = _join(a * cos - b * sin, a * sin + b * cos, n, rotated, s["interleaved"]).to(dtype)
        if not s["train"]:
            continue
        dy = s["d" + name].float()
        a, b = _pairs(dy, rotated, s["interleaved"])
        t = _join(a * cos + b * sin, b * cos - a * sin, dy, rotated, s["interleaved"])
        if w is not None:
            unit = x * rstd
            grads["d_" + name + "_weight"] = (t * unit).sum((0, 1, 2)).to(dtype)
            t = t * w.float()
            t = rstd * (t - unit * (t * unit).mean(-1, keepdim=True))
        grads["d_" + name] = t.to(dtype)
    return {**out, **{"d_" + n: grads["d_" + n] for n in s["leaves"]}} if s["train"] else out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "gated":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        if not case["train"]:
            return {"bytes": e * (m * k + 2 * n * k + m * n), "flops": 4 * m * n * k}
        return {"bytes": e * (2 * m * k + 4 * n * k + 2 * m * n), "flops": 12 * m * n * k}
    if case["kind"] == "cross":
        m, k, v = case["rows"], case["inputs"], case["vocabulary"]
        counted = m * (1.0 - case["ignored"])
        small = 8 * m + 4 * (m if case["reduction"] == "none" else 1)
        if not case["train"]:
            return {"bytes": e * (counted * k + v * k) + small, "flops": 2 * counted * v * k}
        return {"bytes": e * (counted * k + m * k + 2 * v * k) + small, "flops": 6 * counted * v * k}
    n = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
    return {"bytes": e * (4 if case["train"] else 2) * n, "flops": (25 if case["train"] else 10) * n}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    leaf = {n: s[n].detach().double().requires_grad_(case["train"]) for n in s["leaves"]}
    F = torch.nn.functional
    if case["kind"] == "gated":
        act = {"none": lambda z: z, "relu": torch.relu, "gelu": F.gelu,
               "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}[case["activation"]]
        h = act(torch.matmul(leaf["x"], leaf["gate"].mT)) * torch.matmul(leaf["x"], leaf["up"].mT)
        if not case["train"]:
            return h
        grads = torch.autograd.grad(h, list(leaf.values()), s["dy"].double())
        return {"h": h.detach(), **{"d_" + n: d for n, d in zip(leaf, grads)}}
    if case["kind"] == "cross":
        mean = case["reduction"] == "mean"
        loss = F.cross_entropy(torch.matmul(leaf["x"], leaf["weight"].mT), s["target"], ignore_index=IGNORE,
                               reduction="sum" if mean else case["reduction"])
        if mean:
            loss = loss / max(1, int((s["target"] != IGNORE).sum()))
        if not case["train"]:
            return loss
        grads = torch.autograd.grad(loss, list(leaf.values()), s["dloss"].double())
        return {"loss": loss.detach(), **{"d_" + n: d for n, d in zip(leaf, grads)}}
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["frequencies"]))[:, None]
    out = {}
    for name in ("q", "k"):
        x, r = leaf[name], case["rotated"]
        if case["norm"]:
            x = F.rms_norm(x, (case["dim"],), leaf[name + "_weight"], EPS)
        head = x[..., :r].unflatten(-1, (r // 2, 2)) if case["interleaved"] else x[..., :r].unflatten(-1, (2, r // 2)).mT
        head = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn)
        head = head if case["interleaved"] else head.mT
        out[name] = torch.cat((head.flatten(-2), x[..., r:]), -1)
    if not case["train"]:
        return out
    grads = torch.autograd.grad(list(out.values()), list(leaf.values()), (s["dq"].double(), s["dk"].double()))
    return {**{n: v.detach() for n, v in out.items()}, **{"d_" + n: d for n, d in zip(leaf, grads)}}
