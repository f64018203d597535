"""Performance cases of the layers and of the Muon step.

Three operators that stand next to the optimizer in a training program:

* ``layer_norm`` (kind "norm"): normalisation of the last dimension, with its
  backward pass and the reduction of the weight's and bias's gradients;
* ``linear`` (kind "linear"): matrix product with bias, activation and residual
  in its epilogue, with its backward pass, and its form for a few tokens;
* ``orthogonalize`` (kind "ortho") and ``Muon.step`` (kind "muon"): the update
  of a matrix made orthogonal by Newton-Schulz products, alone and inside the
  optimizer step that uses it for the matrices of a model.

``run`` computes a pass in plain torch operations in 32 bits, rounded once at
the end, or (``own``) through the package's entry points.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NORM_EPS = 1e-5
ORTHO_EPS = 1e-7
MOMENTUM = 0.95
WEIGHT_DECAY = 0.1


# ------------------------------------------------------------------ cases
def _norm(name, rows, dim, dtype, train, bias=True):
    return dict(name=name, kind="norm", rows=rows, dim=dim, dtype=dtype, train=train, bias=bias)


def _linear(name, rows, inputs, outputs, dtype, train, activation="none", bias=True, residual=False,
            in_out=False):
    return dict(name=name, kind="linear", rows=rows, inputs=inputs, outputs=outputs, dtype=dtype, train=train,
                activation=activation, bias=bias, residual=residual, in_out=in_out)


def _ortho(name, batch, rows, cols, dtype):
    return dict(name=name, kind="ortho", batch=batch, rows=rows, cols=cols, dtype=dtype)


def _muon(name, shapes, dtype, lr, adjust, **kw):
    return dict(name=name, kind="muon", shapes=shapes, dtype=dtype, lr=lr, adjust=adjust, **kw)


def listed():
    return [
        # one token being generated by an 8B-shaped model: nothing but latency
        _norm("norm_token_bf16", 1, 4096, "bf16", False),
        # GPT-2 trained in fp32, 8 sequences of 1024 tokens
        _norm("norm_train_f32", 8192, 768, "f32", True),
        # an 8B-shaped model's layer, 16 sequences of 1024 tokens, bf16
        _norm("norm_train_bf16", 16384, 4096, "bf16", True),
        # a width and a token count that are multiples of nothing, no bias, fp16
        _norm("norm_odd_f16", 1237, 1013, "f16", True, bias=False),
        # one token through an 8B-shaped MLP matrix: reading the weight once
        _linear("linear_token_bf16", 1, 4096, 14336, "bf16", False, activation="silu", bias=False),
        # GPT-2's MLP up-projection in training (its weight is stored inputs by outputs)
        _linear("linear_up_bf16", 8192, 768, 3072, "bf16", True, activation="gelu_tanh", in_out=True),
        # an 8B-shaped MLP down-projection in training, with the residual stream added
        _linear("linear_down_bf16", 8192, 14336, 4096, "bf16", True, bias=False, residual=True),
        # an odd fp32 layer: every size a multiple of nothing, all of the epilogue
        _linear("linear_odd_f32", 1531, 1001, 777, "f32", True, activation="gelu", residual=True),
        # one small matrix (an adapter, a router): latency of the whole chain of products
        _ortho("ortho_small_f32", 1, 128, 96, "f32"),
        # a few experts' odd-sized matrices at once, taller than wide
        _ortho("ortho_batch_f16", 8, 1300, 500, "f16"),
        # every matrix of GPT-2's blocks in fp32: the step of a small model
        _muon("muon_gpt2_f32", "gpt2", "f32", 0.02, "original"),
        # the seven matrices of one 8B-shaped layer in bf16
        _muon("muon_layer_bf16", "layer", "bf16", 3e-4, "match_rms_adamw"),
    ]


def draw(rng):
    def size(lo, hi):
        return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))

    kind = rng.choices(["norm", "linear", "ortho", "muon"], [0.3, 0.4, 0.2, 0.1])[0]
    dtype = rng.choice(list(DTYPES))
    if kind == "norm":
        c = _norm("", size(1, 32768), size(8, 16384), dtype, rng.random() < 0.7, rng.random() < 0.7)
        while c["rows"] * c["dim"] > 16384 * 4096:
            c["rows"] = max(1, c["rows"] // 2)
    elif kind == "linear":
        train = rng.random() < 0.6
        # relu's slope jumps at 0: there the gradients of two right 32-bit sums differ by whole terms
        acts = ["none", "gelu", "gelu_tanh", "silu"] + (["relu"] if dtype != "f32" or not train else [])
        c = _linear("", size(1, 16384), size(16, 16384), size(16, 16384), dtype, train, rng.choice(acts),
                    rng.random() < 0.6, rng.random() < 0.4, rng.random() < 0.4)
        while c["rows"] * c["inputs"] * c["outputs"] > 8192 * 4096 * 4096:
            c["rows"] = max(1, c["rows"] // 2)
    elif kind == "ortho":
        c = _ortho("", size(1, 16), size(8, 8192), size(8, 8192), dtype)
        while c["batch"] * c["rows"] * c["cols"] * min(c["rows"], c["cols"]) > 4096 ** 3:
            c["batch"], c["rows"] = max(1, c["batch"] // 2), c["rows"] // 2 + 1
    else:
        c = _muon("", "drawn", dtype, 10.0 ** rng.uniform(-4, -1.5), rng.choice(["original", "match_rms_adamw"]),
                  count=size(1, 24), largest=size(64, 2048), sizes_seed=rng.randrange(1 << 20))
    del c["name"]
    return c


def _shapes(case):
    """The matrices of a "muon" case, outputs by inputs."""
    if case["shapes"] == "gpt2":
        return [(2304, 768), (768, 768), (3072, 768), (768, 3072)] * 12
    if case["shapes"] == "layer":
        return [(4096, 4096), (1024, 4096), (1024, 4096), (4096, 4096), (14336, 4096), (14336, 4096), (4096, 14336)]
    import random

    r = random.Random(case["sizes_seed"])
    lo, hi = math.log(8), math.log(case["largest"])
    return [(round(math.exp(r.uniform(lo, hi))), round(math.exp(r.uniform(lo, hi)))) for _ in range(case["count"])]


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g, rows, dim):
    """A residual stream: each token at its own scale, each channel about its own mean."""
    x = _randn(g, rows, dim).mul_(torch.exp(0.3 * _randn(g, rows, 1)))
    return x.add_(0.5 * _randn(g, dim))


def _update(g, rows, cols):
    """A gradient: noise over a few strong directions."""
    x = _randn(g, rows, cols)
    return torch.addmm(x, _randn(g, rows, 8), _randn(g, 8, cols)).mul_(1e-3)


def prepare(case, seed):
    g, dtype = _gen(seed), DTYPES[case["dtype"]]
    s = dict(case)
    if case["kind"] == "norm":
        s["x"] = _activations(g, case["rows"], case["dim"]).to(dtype)
        s["weight"] = (1.0 + 0.1 * _randn(g, case["dim"])).to(dtype)
        s["bias"] = (0.1 * _randn(g, case["dim"])).to(dtype) if case["bias"] else None
        if case["train"]:
            s["dy"] = (0.1 * _randn(g, case["rows"], case["dim"])).to(dtype)
    elif case["kind"] == "linear":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        s["x"] = _activations(g, m, k).to(dtype)
        w = _randn(g, k, n) if case["in_out"] else _randn(g, n, k)
        w = w.mul_(1.0 / math.sqrt(k)).to(dtype)
        s["weight"] = w.t() if case["in_out"] else w
        s["bias"] = (0.1 * _randn(g, n)).to(dtype) if case["bias"] else None
        s["residual"] = _activations(g, m, n).to(dtype) if case["residual"] else None
        if case["train"]:
            s["dy"] = (0.1 * _randn(g, m, n)).to(dtype)
    elif case["kind"] == "ortho":
        s["g"] = torch.stack([_update(g, case["rows"], case["cols"]) for _ in range(case["batch"])]).to(dtype)
    else:
        shapes = _shapes(case)
        sizes = [a * b for a, b in shapes]
        starts = [0]
        for n in sizes:
            starts.append(starts[-1] + (n + 63) // 64 * 64)  # matrices begin on 64 elements, as buckets lay them
        s["flat"] = torch.zeros(starts[-1], device="cuda", dtype=dtype)
        s["params"], s["grads"], s["momenta"] = [], [], []
        for (a, b), n, o in zip(shapes, sizes, starts):
            s["flat"][o:o + n] = _randn(g, n).mul_(0.02)
            s["params"].append(s["flat"][o:o + n].view(a, b))
            s["grads"].append(_update(g, a, b).to(dtype))
            s["momenta"].append(_update(g, a, b).mul_(0.3))
        if own:
            from turboadam_amd import Muon

            s["params"] = [torch.nn.Parameter(p) for p in s["params"]]
            s["opt"] = Muon(s["params"], lr=case["lr"], weight_decay=WEIGHT_DECAY, momentum=MOMENTUM, nesterov=True,
                            ns_coefficients=COEFFICIENTS, ns_steps=STEPS, eps=ORTHO_EPS, adjust_lr=case["adjust"])
            s["opt"].load_state_dict({"state": {i: {"momentum_buffer": m} for i, m in enumerate(s["momenta"])},
                                      "param_groups": s["opt"].state_dict()["param_groups"]})
    if own and case.get("train"):
        for k in ("x", "weight", "bias", "residual"):
            if s.get(k) is not None:
                s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------ the pass
def run(s):
    return {"norm": _run_norm, "linear": _run_linear, "ortho": _run_ortho, "muon": _run_muon}[s["kind"]](s)


def _gradients(s, y):
    """The gradients of every input that a backward pass through y reaches."""
    names = [k for k in ("x", "weight", "bias", "residual") if s.get(k) is not None]
    return {"d" + k: d for k, d in zip(names, torch.autograd.grad(y, [s[k] for k in names], s["dy"]))}


def _run_norm(s):
    if own:
        from turboadam_amd import layer_norm

        y = layer_norm(s["x"], s["weight"], s["bias"], eps=NORM_EPS)
        return {"y": y, **_gradients(s, y)} if s["train"] else y
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    c = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + NORM_EPS)
    n = c * rstd
    y = n * w
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if not s["train"]:
        return y.to(dtype)
    dy = s["dy"].float()
    t = dy * w
    dx = rstd * (t - t.mean(1, keepdim=True) - n * (t * n).mean(1, keepdim=True))
    out = {"y": y.to(dtype), "dx": dx.to(dtype), "dweight": (dy * n).sum(0).to(dtype)}
    if s["bias"] is not None:
        out["dbias"] = dy.sum(0).to(dtype)
    return out


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


def _run_linear(s):
    if own:
        from turboadam_amd import linear

        y = linear(s["x"], s["weight"], s["bias"], activation=s["activation"], residual=s["residual"])
        return {"y": y, **_gradients(s, y)} if s["train"] else y
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _activation(z, s["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not s["train"]:
        return y.to(dtype)
    dy = s["dy"].float()
    dz = dy if s["activation"] == "none" else dy * _slope(z, s["activation"])
    out = {"y": y.to(dtype), "dx": (dz @ w).to(dtype), "dweight": (dz.t() @ x).to(dtype)}
    if s["bias"] is not None:
        out["dbias"] = dz.sum(0).to(dtype)
    if s["residual"] is not None:
        out["dresidual"] = s["dy"]
    return out


def _newton_schulz(u):
    """Newton-Schulz products in 32 bits on the shorter side."""
    a, b, c = COEFFICIENTS
    tall = u.shape[0] > u.shape[1]
    x = u.t() if tall else u
    x = x / torch.sqrt((x * x).sum()).clamp(min=ORTHO_EPS)
    for _ in range(STEPS):
        p = x @ x.t()
        x = a * x + (b * p + c * (p @ p)) @ x
    return x.t() if tall else x


def _run_ortho(s):
    if own:
        from turboadam_amd import orthogonalize

        return orthogonalize(s["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=ORTHO_EPS)
    return torch.stack([_newton_schulz(g.float()) for g in s["g"]]).to(s["g"].dtype)


def _adjusted(lr, adjust, rows, cols):
    return lr * (math.sqrt(max(1.0, rows / cols)) if adjust == "original" else 0.2 * math.sqrt(max(rows, cols)))


def _run_muon(s):
    if own:
        for p, g in zip(s["params"], s["grads"]):
            p.grad = g
        s["opt"].step()
        return {"params": s["flat"], "momenta": [s["opt"].state[p]["momentum_buffer"] for p in s["params"]]}
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        gf = g.float()
        m.mul_(MOMENTUM).add_(gf, alpha=1.0 - MOMENTUM)
        o = _newton_schulz(gf * (1.0 - MOMENTUM) + m * MOMENTUM)
        p.copy_(p.float() * (1.0 - s["lr"] * WEIGHT_DECAY) - _adjusted(s["lr"], s["adjust"], *p.shape) * o)
    return {"params": s["flat"], "momenta": s["momenta"]}


# ------------------------------------------------------------------ what a pass cannot do without
def _ns_flops(rows, cols):
    """Two of the three products of a step are symmetric: half of each is enough."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (3 * m * m * n + m * m * m)


def work(case):
    e = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "norm":
        n = case["rows"] * case["dim"]
        vectors = (2 if case["bias"] else 1) * case["dim"]
        if not case["train"]:
            return {"bytes": e * (2 * n + vectors), "flops": 8 * n}
        return {"bytes": e * (4 * n + 2 * vectors), "flops": 20 * n}
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        bias, res = n if case["bias"] else 0, m * n if case["residual"] else 0
        if not case["train"]:
            return {"bytes": e * (m * k + n * k + m * n + bias + res), "flops": 2 * m * n * k}
        # x, w, dy, the bias and the residual in; y and the gradients out (the residual's is dy itself)
        return {"bytes": e * (2 * m * k + 2 * n * k + 2 * m * n + 2 * bias + res), "flops": 6 * m * n * k}
    if case["kind"] == "ortho":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * e * n, "flops": case["batch"] * _ns_flops(case["rows"], case["cols"])}
    shapes = _shapes(case)
    return {"bytes": (3 * e + 8) * sum(a * b for a, b in shapes), "flops": sum(_ns_flops(a, b) for a, b in shapes)}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("norm", "linear"):
        names = [k for k in ("x", "weight", "bias", "residual") if s.get(k) is not None]
        leaf = {k: s[k].detach().double().requires_grad_(case["train"]) for k in names}
        if case["kind"] == "norm":
            x = leaf["x"]
            var, mean = torch.var_mean(x, dim=-1, keepdim=True, correction=0)
            y = (x - mean) * (var + NORM_EPS).pow(-0.5) * leaf["weight"]
        else:
            y = torch.matmul(leaf["x"], leaf["weight"].transpose(0, 1))
        if "bias" in leaf:
            y = y + leaf["bias"]
        if case["kind"] == "linear":
            y = {"none": lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
                 "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
                 "silu": torch.nn.functional.silu}[case["activation"]](y)
        if "residual" in leaf:
            y = y + leaf["residual"]
        if not case["train"]:
            return y
        grads = torch.autograd.grad(y, list(leaf.values()), s["dy"].double())
        return {"y": y.detach(), **{"d" + k: d for k, d in zip(leaf, grads)}}

    def orthogonal(g):
        # the odd polynomial a s + b s^3 + c s^5 applied STEPS times to g over its norm
        a, b, c = COEFFICIENTS
        x = g / max(float(torch.linalg.vector_norm(g)), ORTHO_EPS)
        eye = torch.eye(min(x.shape), dtype=torch.float64, device=x.device)
        for _ in range(STEPS):
            if x.shape[0] <= x.shape[1]:
                q = torch.matmul(x, x.mT)
                x = torch.matmul(a * eye + torch.matmul(q, b * eye + c * q), x)
            else:
                q = torch.matmul(x.mT, x)
                x = torch.matmul(x, a * eye + torch.matmul(q, b * eye + c * q))
        return x

    if case["kind"] == "ortho":
        return torch.stack([orthogonal(g.double()) for g in s["g"]])
    flat = torch.zeros(s["flat"].numel(), dtype=torch.float64, device="cuda")
    momenta = []
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        g64, m64 = g.double(), m.double()
        m64 = MOMENTUM * m64 + (1.0 - MOMENTUM) * g64
        o = orthogonal((1.0 - MOMENTUM) * g64 + MOMENTUM * m64)
        new = (1.0 - case["lr"] * WEIGHT_DECAY) * p.detach().double() - _adjusted(case["lr"], case["adjust"], *p.shape) * o
        at = p.storage_offset() - s["flat"].storage_offset()
        flat[at:at + p.numel()] = new.reshape(-1)
        momenta.append(m64)
    return {"params": flat, "momenta": momenta}
