"""GPU: linear and layer_norm with their gradients against the formulas in 64
bits, element by element.

Bounds (fixed before the first run).  u: the dtype's rounding (2^-24, 2^-8,
2^-11); a sum of n products in fp32 is off by at most (n + 16) 2^-23 times the
sum of their absolute values, whatever its order; elementary functions by 2^-20
of their result.  The backward pass of an activation sees z rounded once and
rounds dz once; the activations' second derivatives are below 1.2."""

import math
import zlib

import pytest
import torch

from tests.helpers import log

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -24}  # fp16's smallest numbers
F = torch.nn.functional
ACT = {None: lambda z: z, "relu": torch.relu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"),
       "silu": F.silu}


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _sum_error(n):
    return (n + 16) * 2.0 ** -23


def _within(got, want, bound, what):
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, what
    over = (got - want).abs() > bound
    assert not bool(over.any()) and bool(torch.isfinite(got).all()), (
        f"{what}: {int(over.sum())} of {over.numel()} over the bound, worst {float(((got - want).abs() - bound).max())}")


# ------------------------------------------------------------------ linear
def _linear_case(m, k, n, dt, act, bias, residual, in_out, integers=False):
    g, d = _gen(m, k, n, dt, act), DTYPES[dt]

    def rand(*shape):
        if integers:
            return torch.randint(-3, 4, shape, generator=g, device="cuda").to(d)
        return torch.randn(shape, generator=g, device="cuda").to(d)

    x = rand(m, k)
    w = rand(k, n) if in_out else rand(n, k)
    if not integers:
        w = w * max(k, 1) ** -0.5
    w = w.t() if in_out else w
    return x, w, rand(n) if bias else None, rand(m, n) if residual else None, rand(m, n)


def _check_linear(x, w, b, r, dy, dt, act):
    from turboadam_amd import linear

    m, n, k, u, t = x.shape[0], w.shape[0], x.shape[1], UNIT[dt], TINY[dt]
    args = [v for v in (x, w, b, r) if v is not None]
    leaves = [v.detach().requires_grad_() for v in args]
    it = iter(leaves)
    xl, wl, bl, rl = next(it), next(it), next(it) if b is not None else None, next(it) if r is not None else None
    y = linear(xl, wl, bl, activation=act, residual=rl)
    assert y.dtype == x.dtype and y.shape == (m, n)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(linear(x, w, b, activation=act, residual=r), y)  # the call without gradients
    X, W, DY = x.double(), w.double(), dy.double()
    z = X @ W.t() + (0 if b is None else b.double())
    z_err = _sum_error(k) * (X.abs() @ W.abs().t() + (0 if b is None else b.double().abs()))
    z.requires_grad_()
    a = ACT[act](z)
    slope = torch.autograd.grad(a.sum(), z)[0]
    z, a = z.detach(), a.detach()
    ref = a + (0 if r is None else r.double())
    smooth = 0.0 if act is None else 2.0 ** -20
    _within(y, ref, u * ref.abs() + (1 + u) * (1.2 * z_err + smooth * (a.abs() + z.abs())
                                               + 2.0 ** -23 * ref.abs()) + t, "y")
    if act is None:
        dz, dz_err = DY, torch.zeros_like(DY)
    else:
        dz = DY * slope
        seen = 0.0 if act == "relu" else 1.2 * (z_err + u * z.abs() + t)
        dz_err = DY.abs() * (seen + smooth) * (1 + u) + u * dz.abs() + t
    # the bias's gradient is summed before dz is rounded; the bound with its rounding holds too
    want = {"dx": (dz @ W, dz_err @ W.abs() + _sum_error(n) * (dz.abs() @ W.abs())),
            "dw": (dz.t() @ X, dz_err.t() @ X.abs() + _sum_error(m) * (dz.abs().t() @ X.abs()))}
    if b is not None:
        want["db"] = (dz.sum(0), dz_err.sum(0) + _sum_error(m) * dz.abs().sum(0))
    for (name, (v, err)), got in zip(want.items(), grads):
        _within(got, v, u * v.abs() + (1 + u) * err + t, name)
    if r is not None:
        assert torch.equal(grads[-1], dy)
    assert grads[1].stride() == w.stride() or 1 in w.shape


SHAPES = [(1, 1, 1), (1, 64, 16), (2, 4096, 130), (7, 33, 5), (16, 1000, 17), (32, 129, 64), (33, 64, 64),
          (64, 64, 64), (100, 200, 300), (129, 257, 65), (255, 40, 1), (260, 512, 264), (1, 3, 1000), (700, 8, 12),
          (40, 8192, 72), (1100, 520, 776)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_and_gradients(m, k, n, dt):
    for act, bias, residual, in_out in [(None, False, False, False), ("gelu", True, True, True),
                                        ("silu", True, False, False), ("gelu_tanh", False, True, True),
                                        (None, True, True, True)]:
        log(f"linear {m}x{k}x{n} {dt} {act} bias={bias} residual={residual} in_out={in_out}")
        _check_linear(*_linear_case(m, k, n, dt, act, bias, residual, in_out), dt, act)


@pytest.mark.parametrize("dt", list(DTYPES))
def test_linear_relu_of_whole_numbers(dt):
    # small whole numbers: z is exact, and its slope at 0 is 0 on both sides
    log(f"linear relu {dt}")
    _check_linear(*_linear_case(200, 24, 130, dt, "relu", True, True, False, integers=True), dt, "relu")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_linear_large_tiles_and_split_sums(dt):
    # many tiles of the largest size, and few tiles of a long sum
    for m, k, n in [(2048, 512, 2304), (96, 16384, 160), (2050, 1030, 1030)]:
        log(f"linear {m}x{k}x{n} {dt}")
        _check_linear(*_linear_case(m, k, n, dt, "gelu", True, True, False), dt, "gelu")


def test_linear_views_strides_and_leading_dimensions():
    from turboadam_amd import linear

    g = _gen("views")
    base = torch.randn(6, 50, 96, generator=g, device="cuda").bfloat16()
    w = torch.randn(70, 96, generator=g, device="cuda").bfloat16()
    b = torch.randn(140, generator=g, device="cuda").bfloat16()
    whole = linear(base.reshape(300, 96), w, b[:70]).reshape(6, 50, 70)
    log("linear on leading dimensions")
    assert torch.equal(linear(base, w, b[:70]), whole)
    log("linear on strided rows, an odd offset and every other bias element")
    wide = torch.zeros(300, 131, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:99] = base.reshape(300, 96)
    assert torch.equal(linear(wide[:, 3:99], w, b[:70]), whole.reshape(300, 70))
    far = torch.zeros(70, 200, device="cuda", dtype=torch.bfloat16)
    far[:, 8:104] = w
    assert torch.equal(linear(base, far[:, 8:104], b[:70]), whole)
    every = torch.zeros(96, 2, device="cuda", dtype=torch.bfloat16)
    every[:, 0] = base[0, 0]
    assert torch.equal(linear(every[:, 0], w), linear(base[0, 0], w))
    log("linear on a transposed input, an expanded one and a broadcast residual")
    t = base.reshape(300, 96).t().contiguous().t()
    assert torch.equal(linear(t, w), linear(base.reshape(300, 96), w))
    row = base[0, :1].expand(300, 96)
    assert torch.equal(linear(row, w, residual=b[:70].expand(300, 70)),
                       linear(row.contiguous(), w, residual=b[:70].expand(300, 70).contiguous()))


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("m,k,n", [(66, 130, 70), (300, 1026, 34), (35, 2, 6), (2050, 1030, 1030)])
def test_linear_rows_on_words_amid_nan(m, k, n, dt):
    # rows that begin and end on 4 bytes but not on 16, with NaN on every side of them
    for act, in_out in [(None, False), ("gelu", True)]:
        x, w, b, r, dy = _linear_case(m, k, n, dt, act, True, False, False)

        def amid(v):
            wide = torch.full((v.shape[0] + 1, v.shape[1] + 6), float("nan"), device="cuda", dtype=v.dtype)
            inner = wide[:-1, 2:2 + v.shape[1]]
            inner.copy_(v)
            return inner

        log(f"linear amid nan {m}x{k}x{n} {dt} {act} in_out={in_out}")
        flat = torch.full((w.numel() + 10,), float("nan"), device="cuda", dtype=w.dtype)
        flat[2:-8] = (w.t() if in_out else w).reshape(-1)
        w = flat[2:-8].view(k, n).t() if in_out else flat[2:-8].view(n, k)
        _check_linear(amid(x), w, b, r, dy, dt, act)


def test_linear_gradient_of_a_broadcast_input():
    from turboadam_amd import linear

    g = _gen("broadcast")
    x = torch.randn(1, 64, generator=g, device="cuda").requires_grad_()
    w = torch.randn(48, 64, generator=g, device="cuda").requires_grad_()
    r = torch.randn(48, generator=g, device="cuda").requires_grad_()
    dy = torch.randn(40, 48, generator=g, device="cuda")
    dx, dw, dr = torch.autograd.grad(linear(x.expand(40, 64), w, residual=r.expand(40, 48)), (x, w, r), dy)
    D = dy.double()
    assert torch.allclose(dx.double(), (D @ w.double()).sum(0, keepdim=True), rtol=1e-5, atol=1e-4)
    assert torch.allclose(dw.double(), D.t() @ x.double().expand(40, 64), rtol=1e-5, atol=1e-4)
    assert torch.allclose(dr.double(), D.sum(0), rtol=1e-5, atol=1e-4)


@pytest.mark.parametrize("m,k,n", [(0, 8, 8), (5, 0, 9), (40, 0, 9), (5, 8, 0), (40, 8, 0), (0, 0, 4)])
def test_linear_empty_sizes(m, k, n):
    from turboadam_amd import linear

    log(f"linear {m}x{k}x{n}")
    x = torch.ones(m, k, device="cuda", requires_grad=True)
    w = torch.ones(n, k, device="cuda", requires_grad=True)
    b = torch.full((n,), 2.0, device="cuda", requires_grad=True)
    y = linear(x, w, b, activation="relu")
    assert y.shape == (m, n) and bool((y == k + 2).all())
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert bool((dx == n).all()) and bool((dw == m).all()) and bool((db == m).all())
    assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape


@pytest.mark.parametrize("rows", [3, 80])
def test_linear_infinities_and_nan_stay_in_their_rows(rows):
    from turboadam_amd import linear

    x = torch.ones(rows, 72, device="cuda")
    x[1, 5], x[2, 71] = math.inf, math.nan
    w = torch.ones(40, 72, device="cuda")
    for act in (None, "relu", "gelu", "silu", "gelu_tanh"):
        y = linear(x, w, activation=act)
        assert bool((y[1] == math.inf).all()) and bool(y[2].isnan().all()), act
        assert bool(y[0].isfinite().all()) and bool(y[3:].isfinite().all()), act
    assert bool((linear(-x, w, activation="relu")[1] == 0).all())


@pytest.mark.parametrize("dt,size", [("f16", 1e4), ("f16", 6e4), ("bf16", 1e4), ("bf16", 2e20), ("f32", 2e20)])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_linear_gradient_where_z_passes_every_range(act, dt, size):
    """z = -8 size (for fp16 past its numbers, in y a 0; for 2e20 one whose cube is past fp32's) and, where y can hold it,
    8 size: slopes of 0 and 1, and no row or column beside them is touched."""
    from turboadam_amd import linear

    log(f"linear {act} {dt} z = 8 x {size}")
    d = DTYPES[dt]
    x = torch.full((40, 8), 0.25, device="cuda", dtype=d)
    x[3], x[5] = size, -size
    w = torch.full((18, 8), -1.0, device="cuda", dtype=d)
    w[9:] = 0.125
    if dt == "f16":  # there y's own infinities are right: only z far below 0
        x[5], w[9:] = 0.25, -0.5
    x, w = x.requires_grad_(), w.requires_grad_()
    b = torch.zeros(18, device="cuda", dtype=d, requires_grad=True)
    y = linear(x, w, b, activation=act)
    assert bool(y.isfinite().all())
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    z = (x.detach().double() @ w.detach().double().t()).requires_grad_()
    slope = torch.autograd.grad(ACT[act](z).sum(), z)[0]
    assert bool(slope.isfinite().all())
    for got, want in ((dx, slope @ w.detach().double()), (dw, slope.t() @ x.detach().double()), (db, slope.sum(0))):
        assert bool(got.isfinite().all())
        assert float((got.double() - want).norm()) <= (4 * UNIT[dt] + 2.0 ** -17) * float(want.norm())


def test_linear_gradient_against_differences():
    """fp32 directional derivatives by central differences in 64 bits of the same function of the outputs."""
    from turboadam_amd import linear

    g = _gen("differences")
    for act in ("gelu", "gelu_tanh", "silu"):
        leaves = [torch.randn(s, generator=g, device="cuda") for s in ((50, 40), (30, 40), (30,), (50, 30))]
        leaves[1] *= 40 ** -0.5
        dy = torch.randn(50, 30, generator=g, device="cuda")
        x, w, b, r = [v.clone().requires_grad_() for v in leaves]
        grads = torch.autograd.grad(linear(x, w, b, activation=act, residual=r), (x, w, b, r), dy)

        def value(x, w, b, r):
            return ((ACT[act](x @ w.t() + b) + r) * dy.double()).sum()

        for i, grad in enumerate(grads):
            step = torch.randn(leaves[i].shape, generator=g, device="cuda", dtype=torch.float64)
            at = [v.double() for v in leaves]
            up, down = list(at), list(at)
            up[i], down[i] = at[i] + 1e-5 * step, at[i] - 1e-5 * step
            want = (value(*up) - value(*down)) / 2e-5
            scale = float(grad.double().norm() * step.norm())
            assert abs(float((grad.double() * step).sum() - want)) < 1e-5 * scale, (act, i)


def test_linear_same_bits_every_time_and_on_another_stream():
    from turboadam_amd import linear

    x, w, b, r, dy = _linear_case(900, 1000, 264, "bf16", "gelu", True, True, False)
    x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()

    def call():
        y = linear(x, w, b, activation="gelu", residual=r)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = call()
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(first, second):
        assert torch.equal(a, c)


def test_layers_in_a_captured_graph():
    from turboadam_amd import layer_norm, linear

    x, w, b, r, dy = _linear_case(300, 264, 130, "bf16", "silu", True, True, False)
    s = torch.ones(264, device="cuda", dtype=torch.bfloat16)
    leaves = [v.detach().requires_grad_() for v in (x, w, b, s)]

    def call():
        y = linear(layer_norm(leaves[0], leaves[3]), leaves[1], leaves[2], activation="silu", residual=r)
        return [y, *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(300, 264, generator=_gen(i), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, call()):
            assert torch.equal(a, c), f"replay {i}"


# -------------------------------------------------------------- layer norm
def _check_norm(x, w, b, dy, dt, eps=1e-5):
    from turboadam_amd import layer_norm

    u, t, n = UNIT[dt], TINY[dt], x.shape[-1]
    leaves = [v.detach().requires_grad_() for v in (x, w, b) if v is not None]
    it = iter(leaves)
    y = layer_norm(next(it), next(it) if w is not None else None, next(it) if b is not None else None, eps=eps)
    grads = torch.autograd.grad(y, leaves, dy)
    X, DY = x.double(), dy.double()
    W = torch.ones(n, device="cuda", dtype=torch.float64) if w is None else w.double()
    c = X - X.mean(1, keepdim=True)
    rstd = (c.square().mean(1, keepdim=True) + eps).rsqrt()
    h = c * rstd
    # the mean is off by mean_err, each distance by that and a rounding; rstd by the sum's
    # error and what the distances' errors make of the variance
    mean_err = _sum_error(n) * X.abs().mean(1, keepdim=True) + 2.0 ** -23 * X.mean(1, keepdim=True).abs()
    c_err = mean_err + 2.0 ** -23 * c.abs()
    rstd_rel = _sum_error(n) + 2.0 ** -20 + rstd.square() * (c.abs() * c_err + c_err.square()).mean(1, keepdim=True)
    h_err = c_err * rstd + h.abs() * (rstd_rel + 2.0 ** -22)
    y_ref = h * W + (0 if b is None else b.double())
    _within(y, y_ref, u * y_ref.abs() + (1 + u) * (h_err * W.abs() + 2.0 ** -22 * ((h * W).abs() + y_ref.abs())) + t, "y")
    T = DY * W
    m0, m1 = T.mean(1, keepdim=True), (T * h).mean(1, keepdim=True)
    dx = rstd * (T - m0 - h * m1)
    m0_err = (_sum_error(n) + 2.0 ** -22) * T.abs().mean(1, keepdim=True)
    m1_err = (_sum_error(n) + 2.0 ** -22) * (T * h).abs().mean(1, keepdim=True) + (T.abs() * h_err).mean(1, keepdim=True)
    part = T.abs() + m0.abs() + (h * m1).abs()
    dx_err = rstd * (m0_err + h.abs() * m1_err + h_err * (m1.abs() + m1_err) + (rstd_rel + 2.0 ** -20) * part)
    _within(grads[0], dx, u * dx.abs() + (1 + u) * dx_err + t, "dx")
    rows = x.shape[0]
    if w is not None:
        dw = (DY * h).sum(0)
        err = (DY.abs() * h_err).sum(0) + _sum_error(rows) * (DY * h).abs().sum(0)
        _within(grads[1], dw, u * dw.abs() + (1 + u) * err + t, "dweight")
    if b is not None:
        db = DY.sum(0)
        _within(grads[-1], db, u * db.abs() + (1 + u) * _sum_error(rows) * DY.abs().sum(0) + t, "dbias")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (1, 4096), (5, 512), (130, 513), (1000, 768), (17, 1013),
                                    (300, 1500), (40, 4095), (33, 4097), (9, 8192), (7, 12001), (3, 16384),
                                    (5, 20000), (2, 32768)])
def test_layer_norm_and_gradients(rows, n, dt):
    g, d = _gen(rows, n, dt), DTYPES[dt]
    x = (torch.randn(rows, n, generator=g, device="cuda") * 2 + 1).to(d)
    w = torch.randn(n, generator=g, device="cuda").to(d)
    b = torch.randn(n, generator=g, device="cuda").to(d)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(d)
    for use_w, use_b in ((True, True), (True, False), (False, True), (False, False)):
        log(f"layer_norm {rows}x{n} {dt} weight={use_w} bias={use_b}")
        _check_norm(x, w if use_w else None, b if use_b else None, dy, dt)


def test_layer_norm_of_rows_far_from_zero_and_of_equal_elements():
    g = _gen("far")
    x = 1000 + torch.randn(20, 600, generator=g, device="cuda")
    dy = torch.randn(20, 600, generator=g, device="cuda")
    log("layer_norm of a large mean")
    _check_norm(x, None, None, dy, "f32")
    from turboadam_amd import layer_norm

    log("layer_norm of equal elements")
    flat = torch.full((4, 600), 3.0, device="cuda", requires_grad=True)
    y = layer_norm(flat, eps=1e-5)
    assert bool((y == 0).all())
    assert bool(torch.autograd.grad(y.sum(), flat)[0].isfinite().all())


def test_layer_norm_views_empty_rows_and_bad_rows():
    from turboadam_amd import layer_norm

    g = _gen("norm views")
    x = torch.randn(3, 10, 131, generator=g, device="cuda").half()
    whole = layer_norm(x[..., 2:99].contiguous())
    log("layer_norm on strided rows and leading dimensions")
    assert torch.equal(layer_norm(x[..., 2:99]), whole)
    assert torch.equal(layer_norm(x[1, :, 2:99]), whole[1])
    assert torch.equal(layer_norm(x[1, 4, 2:99]), whole[1, 4])
    log("layer_norm of no rows")
    none = torch.zeros(0, 40, device="cuda", requires_grad=True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    dx, dw = torch.autograd.grad(layer_norm(none, w), (none, w), torch.zeros(0, 40, device="cuda"))
    assert dx.shape == (0, 40) and bool((dw == 0).all())
    log("layer_norm: a NaN or infinity stays in its row")
    y = torch.randn(5, 97, generator=g, device="cuda")
    good = layer_norm(y)
    y[1, 3], y[3, 0] = math.nan, math.inf
    bad = layer_norm(y)
    assert bool(bad[1].isnan().all()) and bool(bad[3].isnan().all())
    assert torch.equal(bad[[0, 2, 4]], good[[0, 2, 4]])


def test_layers_refuse_what_they_cannot_take():
    from turboadam_amd import layer_norm, linear

    x = torch.ones(4, 8, device="cuda")
    w = torch.ones(6, 8, device="cuda")
    for args, kw, error, text in [
        ((x.cpu(), w), {}, RuntimeError, "MI355X"), ((x, w.cpu()), {}, RuntimeError, "weight"),
        ((x.double(), w.double()), {}, ValueError, "float32"), ((x, w.half()), {}, ValueError, "weight must be"),
        ((x, w.t()), {}, ValueError, "inputs"), ((x, w[0]), {}, ValueError, "inputs"),
        ((x, w, x[0]), {}, ValueError, "bias"), ((x, w), {"residual": x}, ValueError, "residual"),
        ((x, w), {"activation": "tanh"}, ValueError, "activation"),
    ]:
        with pytest.raises(error, match=text):
            linear(*args, **kw)
    for args, kw, error, text in [
        ((x.cpu(),), {}, RuntimeError, "MI355X"), ((x, w[0].half()), {}, ValueError, "weight must be"),
        ((x, x[:, 0]), {}, ValueError, "shape"), ((x, None, x[:, 0]), {}, ValueError, "shape"),
        ((x,), {"eps": -1.0}, ValueError, "eps"), ((x.long(),), {}, ValueError, "float32"),
        ((torch.ones(2, 32769, device="cuda"),), {}, ValueError, "32768"),
        ((torch.ones(2, 0, device="cuda"),), {}, ValueError, "1 to"),
    ]:
        with pytest.raises(error, match=text):
            layer_norm(*args, **kw)


def test_layers_and_orthogonalize_refuse_tangents():
    """Forward-mode derivatives are not computed: a dual argument raises, and with it a dual gradient."""
    import torch.autograd.forward_ad as forward

    from turboadam_amd import layer_norm, linear, orthogonalize

    g = _gen("tangents")
    x, w = torch.randn(40, 24, generator=g, device="cuda"), torch.randn(16, 24, generator=g, device="cuda")
    b, r, s = w[:, 0].contiguous(), torch.ones(40, 16, device="cuda"), torch.ones(24, device="cuda")
    plain = [linear(x, w, b, residual=r), layer_norm(x, s, s), orthogonalize(x)]
    leaf, weight = x.clone().requires_grad_(), w.clone().requires_grad_()
    graphs = [(linear(leaf, w), leaf), (linear(x, weight), weight), (layer_norm(leaf), leaf)]
    with forward.dual_level():
        def dual(v):
            return forward.make_dual(v, torch.ones_like(v))

        def calls():
            return (lambda: linear(dual(x), w), lambda: linear(x, dual(w)), lambda: linear(x, w, dual(b)),
                    lambda: linear(x, w, residual=dual(r)), lambda: linear(dual(x), weight),
                    lambda: layer_norm(dual(x)), lambda: layer_norm(x, dual(s)), lambda: layer_norm(x, s, dual(s)),
                    lambda: layer_norm(dual(x), s.clone().requires_grad_()), lambda: orthogonalize(dual(x)))

        for i, call in enumerate(calls()):
            for enabled in (True, False):
                log(f"a dual argument, call {i}, gradients {enabled}")
                with torch.set_grad_enabled(enabled), pytest.raises(RuntimeError, match="dual"):
                    call()
        for i, (y, at) in enumerate(graphs):
            log(f"a dual gradient, call {i}")
            with pytest.raises(RuntimeError, match="dual"):
                torch.autograd.grad(y, at, dual(torch.ones_like(y)))
        # a level without a tangent on any argument changes nothing
        now = [linear(x, w, b, residual=r), layer_norm(x, s, s), orthogonalize(x)]
    for a, c in zip(plain, now):
        assert torch.equal(a, c)


def test_layers_and_orthogonalize_refuse_to_be_recorded():
    """A recorder of torch operations sees only the allocation of what the kernels write: its graph would return
    uninitialised memory."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from turboadam_amd import layer_norm, linear, orthogonalize

    g = _gen("recorded")
    x, w = torch.randn(40, 24, generator=g, device="cuda"), torch.randn(16, 24, generator=g, device="cuda")
    leaf = x.clone().requires_grad_()
    y, h = linear(leaf, w), layer_norm(leaf)

    def ortho(t):
        return orthogonalize(t)

    for name, call in (("linear", lambda t: linear(t, w)), ("layer_norm", lambda t: layer_norm(t)),
                       ("orthogonalize", ortho),
                       ("linear's gradient", lambda t: torch.autograd.grad(y, leaf, t[:, :16], retain_graph=True)[0]),
                       ("layer_norm's gradient", lambda t: torch.autograd.grad(h, leaf, t, retain_graph=True)[0])):
        log(f"make_fx of {name}")
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(call)(x)
        if "gradient" not in name:
            log(f"make_fx before dispatch of {name}")
            with pytest.raises(RuntimeError, match="recorded"):
                make_fx(call, pre_dispatch=True)(x)
            log(f"trace of {name}")
            with pytest.raises(RuntimeError, match="recorded"):
                torch.jit.trace(call, (x,), check_trace=False)
            assert torch.equal(call(x), call(x))


# -------------------------------------------------- every tile and every term
def _tiles(m, k, n, dt, in_out):
    """The tiles of y, dx and dw, as the library would choose them for this call."""
    import ctypes

    from turboadam_amd import _lib

    lib, tiles = _lib.load(), []
    for backward in (0, 1):
        d = _lib.TamLinear(rows=m, inputs=k, outputs=n, ldx=k, ldw=n if in_out else k, w_in_out=in_out,
                           dtype=_lib.DTYPES[DTYPES[dt]])
        for name in ("x", "w", "y", "z", "dy", "dx", "dw"):
            setattr(d, name, 0x10000)
        out = (ctypes.c_uint32 * 4)()
        assert lib.tam_linear_tiles(ctypes.byref(d), backward, out) == 0
        tiles += [out[0]] if not backward else [out[0], out[2]]
    return tuple(tiles)


# sizes that reach each tile with remainders: rows in whole 16 bytes, rows on words (which the largest tile copies), neither
LARGE = [("bf16", 8200, 520, 8200, 256, 128, 128), ("f16", 8200, 520, 8200, 256, 128, 128),
         ("bf16", 8202, 518, 8198, 256, 128, 128), ("f16", 8201, 519, 8199, 256, 128, 128),
         ("bf16", 3000, 4104, 3000, 128, 256, 256), ("f16", 3002, 4102, 3010, 128, 256, 256),
         ("bf16", 3001, 4101, 3003, 128, 256, 256), ("bf16", 4099, 2050, 4102, 128, 128, 128),
         ("f16", 4099, 2050, 4102, 128, 128, 128), ("f32", 6000, 1032, 6000, 128, 128, 128),
         ("f32", 6003, 1031, 6005, 128, 128, 128)]


@pytest.mark.parametrize("in_out", [False, True])
@pytest.mark.parametrize("dt,m,k,n,y_tile,dx_tile,dw_tile", LARGE)
def test_linear_in_every_large_tile(dt, m, k, n, y_tile, dx_tile, dw_tile, in_out):
    log(f"linear {m}x{k}x{n} {dt} in_out={in_out}, tiles of {y_tile}, {dx_tile}, {dw_tile}")
    assert _tiles(m, k, n, dt, in_out) == (y_tile, dx_tile, dw_tile)
    _check_linear(*_linear_case(m, k, n, dt, "gelu", True, True, in_out), dt, "gelu")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("m,k,n", [(96, 16384, 160), (40, 8192, 72), (2, 4096, 130), (32, 16383, 48), (17, 5003, 33),
                                   (1, 16384, 300), (300, 9001, 65), (160, 96, 16384), (130, 70, 9001),
                                   (16384, 96, 160), (9001, 70, 130), (2050, 1030, 1030), (8202, 518, 8198),
                                   (3002, 4102, 3010), (6003, 1031, 6005)])
def test_linear_of_whole_numbers_loses_no_term(m, k, n, dt):
    """Small whole numbers, whose sums are exact in fp32 in any order and in any parts: the results are the exact ones,
    rounded.  One term lost or taken twice in a sum of thousands shows."""
    from turboadam_amd import linear

    for in_out in (False, True):
        log(f"linear of whole numbers {m}x{k}x{n} {dt} in_out={in_out}")
        x, w, b, r, dy = _linear_case(m, k, n, dt, None, True, True, in_out, integers=True)
        x, w, b = x.requires_grad_(), w.detach().requires_grad_(), b.requires_grad_()
        y = linear(x, w, b, residual=r)
        got = [y, *torch.autograd.grad(y, (x, w, b), dy)]
        X, W, D = x.detach().double(), w.detach().double(), dy.double()
        want = [X @ W.t() + b.detach().double() + r.double(), D @ W, D.t() @ X, D.sum(0)]
        for name, a, c in zip(("y", "dx", "dw", "db"), got, want):
            assert torch.equal(a.detach(), c.to(a.dtype)), name


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("n", [768, 1013, 4096, 4097, 8192, 12001, 16384, 20000, 32768])
def test_layer_norm_sees_every_element(n, dt):
    """Rows of one element that is not 0, and dy of another one: a lost or repeated chunk of a row changes the mean, the
    variance or the gradient's sums at once, where long random sums would hide it."""
    from turboadam_amd import layer_norm

    log(f"layer_norm of single elements {n} {dt}")
    at = sorted({i for i in (0, 1, 7, 8, 63, 511, 512, 1023, 2047, 2048, 4095, 4096, 8191, 8192, 16383, 16384, n // 2,
                             n - 9, n - 8, n - 1) if i < n})
    rows = torch.arange(len(at), device="cuda")
    cols = torch.tensor(at, device="cuda")
    x = torch.zeros(len(at), n, device="cuda", dtype=DTYPES[dt])
    dy = torch.zeros_like(x)
    x[rows, cols] = 3.0
    dy[rows, cols.flip(0)] = 2.0
    w = torch.ones(n, device="cuda", dtype=DTYPES[dt])
    leaves = [x.requires_grad_(), w.requires_grad_(), torch.zeros_like(w).requires_grad_()]
    y = layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    X, T = x.detach().double(), dy.double()
    c = X - X.mean(1, keepdim=True)
    rstd = (c.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    h = c * rstd
    m0, m1 = T.mean(1, keepdim=True), (T * h).mean(1, keepdim=True)
    u, t, e = UNIT[dt], TINY[dt], 2.0 ** -18  # of the terms: a few roundings of fp32
    _within(y, h, (u + e) * h.abs() + t, "y")
    ref = rstd * (T - m0 - h * m1)
    _within(dx, ref, u * ref.abs() + (1 + u) * e * rstd * (T.abs() + m0.abs() + (h * m1).abs()) + t, "dx")
    _within(dw, (T * h).sum(0), (u + e) * (T * h).abs().sum(0) + t, "dw")
    _within(db, T.sum(0), u * T.abs().sum(0) + t, "db")


def test_layers_take_zero_tensors_as_zeros():
    """autograd's zero tensors have no memory; they are arguments like any other."""
    from turboadam_amd import layer_norm, linear

    g = _gen("zero tensors")
    x, w = torch.randn(5, 24, generator=g, device="cuda"), torch.randn(7, 24, generator=g, device="cuda")

    def none(*shape):
        return torch._efficientzerotensor(shape, device="cuda", dtype=torch.float32)

    def real(*shape):
        return torch.zeros(shape, device="cuda")

    for name, call in (("layer_norm's weight", lambda z: layer_norm(x, z(24), w[0])),
                       ("layer_norm's bias", lambda z: layer_norm(x, w[0], z(24))),
                       ("layer_norm's x", lambda z: layer_norm(z(5, 24), w[0], w[1])),
                       ("linear's x", lambda z: linear(z(5, 24), w, w[:, 0])),
                       ("linear's weight", lambda z: linear(x, z(7, 24), w[:, 0])),
                       ("linear's bias", lambda z: linear(x, w, z(7))),
                       ("linear's residual", lambda z: linear(x, w, residual=z(5, 7)))):
        log(name)
        assert torch.equal(call(none), call(real)), name
    leaf = x.clone().requires_grad_()
    for y in (linear(leaf, w), layer_norm(leaf)):
        dx, = torch.autograd.grad(y, leaf, none(*y.shape))
        assert bool((dx == 0).all()) and dx.shape == x.shape


@pytest.mark.parametrize("dt", list(DTYPES))
def test_linear_gradient_of_infinite_and_missing_z(dt):
    """A NaN in a row of x makes that row's gradient NaN, whatever the activation, and an infinity gives the slopes' limits."""
    from turboadam_amd import linear

    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        log(f"linear {act} {dt}: NaN and infinities in rows")
        x = torch.ones(70, 24, device="cuda", dtype=DTYPES[dt])
        x[1, 5], x[2, 23], x[3, 0] = math.nan, math.inf, -math.inf
        x = x.requires_grad_()
        w = torch.ones(40, 24, device="cuda", dtype=DTYPES[dt])
        dx, = torch.autograd.grad(linear(x, w, activation=act), x, torch.ones(70, 40, device="cuda", dtype=DTYPES[dt]))
        assert bool(dx[1].isnan().all()), act
        assert bool((dx[2] == 40).all()) and bool((dx[3] == 0).all()), act
        assert bool(dx[[0, *range(4, 70)]].isfinite().all()), act


# ------------------------------------------------- offsets past 32 bits
def _whole(g, *shape):
    return torch.randint(-3, 4, shape, generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)


def test_linear_offsets_past_32_bits():
    """Outputs and gradients of 2.3e9 elements, in whole numbers: rows at both ends and the sums over all of them."""
    from turboadam_amd import linear

    g = _gen("long")
    m, k, n = 70001, 24, 32768
    x, w, dy = _whole(g, m, k).requires_grad_(), _whole(g, n, k).requires_grad_(), _whole(g, m, n)
    b, r = _whole(g, n).requires_grad_(), dy.roll(1, 0)
    log(f"linear {m}x{k}x{n}")
    y = linear(x, w, b, activation="relu", residual=r)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    X, W = x.detach().double(), w.detach().double()
    sum_w, sum_b = torch.zeros_like(W), torch.zeros(n, device="cuda", dtype=torch.float64)
    for i in range(0, m, 5000):
        rows = slice(i, min(i + 5000, m))
        z = X[rows] @ W.t() + b.detach().double()
        dz = dy[rows].double() * (z > 0)
        assert torch.equal(y[rows], (z.relu() + r[rows].double()).to(y.dtype)), i
        assert torch.equal(dx[rows], (dz @ W).to(dx.dtype)), i
        sum_w += dz.t() @ X[rows]
        sum_b += dz.sum(0)
    assert torch.equal(dw, sum_w.to(dw.dtype)) and torch.equal(db, sum_b.to(db.dtype))


@pytest.mark.parametrize("rows,in_out", [(1, False), (20, False), (40, False), (1, True), (40, True)])
def test_linear_weight_past_32_bits(rows, in_out):
    from turboadam_amd import linear

    g = _gen("long weight")
    k, n = 18000, 128256
    x = _whole(g, rows, k)
    w = _whole(g, k, n).t() if in_out else _whole(g, n, k)
    log(f"linear {rows}x{k}x{n} in_out={in_out}")
    y = linear(x, w)
    X = x.double()
    for i in range(0, n, 16384):
        part = slice(i, min(i + 16384, n))
        assert torch.equal(y[:, part], (X @ w[part].double().t()).to(y.dtype)), i


def test_layer_norm_offsets_past_32_bits():
    from turboadam_amd import layer_norm

    g = _gen("long norm")
    rows, n = 540001, 4096
    x = torch.randn(rows, n, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_()
    dy = torch.randn(rows, n, generator=g, device="cuda", dtype=torch.bfloat16)
    log(f"layer_norm {rows}x{n}")
    y = layer_norm(x)
    dx, = torch.autograd.grad(y, x, dy)
    for i in (0, 261000, 524288, rows - 3000):  # the same rows by themselves, whose results other tests pin
        part = x.detach()[i:i + 3000].clone().requires_grad_()
        z = layer_norm(part)
        assert torch.equal(y[i:i + 3000], z), i
        assert torch.equal(dx[i:i + 3000], torch.autograd.grad(z, part, dy[i:i + 3000])[0]), i

