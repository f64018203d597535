"""GPU: gated_linear, linear_cross_entropy and rotary with their gradients against
the formulas in 64 bits, element by element.

Bounds (fixed before the first run).  u: the dtype's rounding (2^-24, 2^-8,
2^-11); a sum of n products in fp32 is off by at most (n + 16) 2^-23 times the
sum of their absolute values, whatever its order; elementary functions by 2^-20
of their result (a sine or cosine by 2^-21).  What a backward pass keeps or hands
to a product is rounded to the type once; the activations' slopes and second
derivatives are below 1.2.  A softmax's sum of v terms is joined from tiles: 2^-22
(100 + v / 64) of it, and a factor exp(z - lse) is off by what z, lse and
|z - lse| 2^-22 are off."""

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


def _randn(g, dt, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(DTYPES[dt])


def _sum_error(n):
    return (n + 16) * 2.0 ** -23


def _within(got, want, bound, what):
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, what
    over = (got - want).abs() > bound
    assert not bool(over.any()) and bool(torch.isfinite(got).all()), (
        f"{what}: {int(over.sum())} of {over.numel()} over the bound, worst {float(((got - want).abs() - bound).max())}")


def _amid_nan(v, dims=1):
    """v as a view with NaN on every side of its rows, at an odd element's address."""
    wide = torch.full((*v.shape[:-1], v.shape[-1] + 5), float("nan"), device="cuda", dtype=v.dtype)
    inner = wide[..., 3:3 + v.shape[-1]]
    inner.copy_(v)
    return inner


# ------------------------------------------------------------ gated linear
def _gated_case(m, k, n, dt, in_out=False):
    g = _gen("gated", m, k, n, dt)

    def weight():
        w = torch.randn((k, n) if in_out else (n, k), generator=g, device="cuda") * max(k, 1) ** -0.5
        w = w.to(DTYPES[dt])
        return w.t() if in_out else w

    return _randn(g, dt, m, k), weight(), weight(), _randn(g, dt, m, n)


def _check_gated(x, wg, wu, dh, dt, act):
    from turboadam_amd import gated_linear

    (m, k), n, u, t = x.shape, wg.shape[0], UNIT[dt], TINY[dt]
    leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
    h = gated_linear(*leaves, activation=act)
    assert h.dtype == x.dtype and h.shape == (m, n)
    grads = torch.autograd.grad(h, leaves, dh)
    with torch.no_grad():
        assert torch.equal(gated_linear(x, wg, wu, activation=act), h)
    X, G, U, D = x.double(), wg.double(), wu.double(), dh.double()
    z, up = X @ G.t(), X @ U.t()
    z_err, up_err = _sum_error(k) * (X.abs() @ G.abs().t()), _sum_error(k) * (X.abs() @ U.abs().t())
    z.requires_grad_()
    a = ACT[act](z)
    slope = torch.autograd.grad(a.sum(), z)[0]
    z, a = z.detach(), a.detach()
    smooth = 0.0 if act is None else 2.0 ** -20
    a_err = 1.2 * z_err + smooth * (a.abs() + z.abs())
    want = a * up
    _within(h, want, u * want.abs() + (1 + u) * (a_err * (up.abs() + up_err) + a.abs() * up_err + 2.0 ** -23 * want.abs()) + t,
            "h")
    z_err, up_err = z_err + u * z.abs() + t, up_err + u * up.abs() + t  # as they are kept
    s_err = 0.0 if act is None else 1.2 * z_err + smooth
    a_err = 1.2 * z_err + smooth * (a.abs() + z.abs())
    dz, du = D * up * slope, D * a
    dz_err = (1 + u) * D.abs() * (s_err * (up.abs() + up_err) + (slope.abs() + 0) * up_err + 2.0 ** -22 * (slope * up).abs()) \
        + u * dz.abs() + t
    du_err = (1 + u) * D.abs() * (a_err + 2.0 ** -23 * a.abs()) + u * du.abs() + t
    names = {"dx": (dz @ G + du @ U, dz_err @ G.abs() + du_err @ U.abs()
                    + _sum_error(2 * n) * (dz.abs() @ G.abs() + du.abs() @ U.abs())),
             "dgate": (dz.t() @ X, dz_err.t() @ X.abs() + _sum_error(m) * (dz.abs().t() @ X.abs())),
             "dup": (du.t() @ X, du_err.t() @ X.abs() + _sum_error(m) * (du.abs().t() @ X.abs()))}
    for (name, (v, err)), got in zip(names.items(), grads):
        _within(got, v, u * v.abs() + (1 + u) * err + t, name)
    if wg.stride() == wu.stride() and (wg.is_contiguous() or wg.t().is_contiguous()):
        for got in grads[1:]:
            assert got.stride() == wg.stride() or 1 in wg.shape


GATED = [(1, 1, 1), (1, 64, 16), (2, 4096, 130), (7, 33, 5), (16, 1000, 17), (32, 129, 64), (33, 64, 64),
         (64, 64, 64), (100, 200, 300), (129, 257, 65), (255, 40, 1), (260, 512, 264), (1, 3, 1000), (700, 8, 12),
         (40, 8192, 72), (1100, 520, 776)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("m,k,n", GATED)
def test_gated_and_gradients(m, k, n, dt):
    for act, in_out in [("silu", False), ("gelu", True), (None, False), ("gelu_tanh", True)]:
        log(f"gated {m}x{k}x{n} {dt} {act} in_out={in_out}")
        _check_gated(*_gated_case(m, k, n, dt, in_out), dt, act)


@pytest.mark.parametrize("dt", list(DTYPES))
def test_gated_large_tiles_and_split_sums(dt):
    for m, k, n in [(2048, 512, 1152), (96, 8192, 80), (2050, 1030, 515)]:
        for in_out in (False, True):
            log(f"gated {m}x{k}x{n} {dt} in_out={in_out}")
            _check_gated(*_gated_case(m, k, n, dt, in_out), dt, "silu")


@pytest.mark.parametrize("dt", list(DTYPES))
def test_gated_relu_of_whole_numbers(dt):
    # small whole numbers: the products are exact, and the slope at 0 is 0 on both sides
    g = _gen("whole", dt)
    x, wg, wu, dh = [torch.randint(-3, 4, s, generator=g, device="cuda").to(DTYPES[dt])
                     for s in ((200, 24), (130, 24), (130, 24), (200, 130))]
    log(f"gated relu {dt}")
    _check_gated(x, wg, wu, dh, dt, "relu")


@pytest.mark.parametrize("rows", [20, 100])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_gated_of_products_below_and_near_the_ends_of_the_range(rows, dt):
    """Rows of x from 2^-24 to 1 and some zeros: products below fp16's normal numbers and below its smallest; and
    products past the middle of a type's last place, either side of 0."""
    x, wg, wu, dh = _gated_case(rows, 40, 50, dt)
    x = (x.float() * torch.exp2(-(torch.arange(rows, device="cuda") % 25.0))[:, None]).to(DTYPES[dt])
    x[3] = 0
    for act in ("silu", "gelu", None):
        log(f"gated small {rows} {dt} {act}")
        _check_gated(x, wg, wu, dh, dt, act)
    log(f"gated large {rows} {dt}")
    _check_gated(x * (64 if dt == "f16" else 2.0 ** 30), wg, wu, dh * 2.0 ** -10, dt, "relu" if dt == "f32" else "silu")


@pytest.mark.parametrize("rows", [5, 90])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_gated_views_and_weights_of_two_layouts(rows, dt):
    from turboadam_amd import gated_linear

    x, wg, wu, _ = _gated_case(rows, 50, 70, dt)
    log(f"gated views {rows} {dt}")
    want = gated_linear(x, wg, wu)
    assert torch.equal(gated_linear(_amid_nan(x), _amid_nan(wg), _amid_nan(wu)), want)
    assert torch.equal(gated_linear(x.reshape(rows, 1, 50), wg, wu), want.reshape(rows, 1, 70))
    assert torch.equal(gated_linear(x, wg, wu.t().contiguous().t()), want)
    both = torch.cat((wg, wu))  # one matrix of both, as checkpoints hold them
    assert torch.equal(gated_linear(x, both[:70], both[70:]), want)
    assert torch.equal(gated_linear(x[:1].expand(rows, 50), wg, wu), gated_linear(x[:1].repeat(rows, 1), wg, wu))
    leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
    mixed = [leaves[0], leaves[1], wu.t().contiguous().t().requires_grad_()]
    dh = torch.ones_like(want)
    for a, b in zip(torch.autograd.grad(gated_linear(*leaves), leaves, dh),
                    torch.autograd.grad(gated_linear(*mixed), mixed, dh)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("in_out", [False, True])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_gated_one_weight_at_an_odd_address(dt, in_out):
    """Rows of whole 16 bytes, a stride of their own, and only one of the weights on 4 bytes."""
    x, wg, wu, dh = _gated_case(70, 64, 48, dt, in_out)
    for off, of_gate in ((0, 1), (1, 0)):
        views = []
        for w, at in ((wg, of_gate), (wu, off)):
            m = w.t() if in_out else w
            flat = torch.full((m.shape[0] * 80 + 2,), float("nan"), device="cuda", dtype=w.dtype)
            v = flat[at:at + m.shape[0] * 80].view(m.shape[0], 80)[:, :m.shape[1]]
            v.copy_(m)
            views.append(v.t() if in_out else v)
        log(f"gated odd address {dt} in_out={in_out}")
        _check_gated(x, *views, dh, dt, "silu")


@pytest.mark.parametrize("m,k,n", [(0, 8, 8), (5, 0, 9), (40, 0, 9), (5, 8, 0), (40, 8, 0), (0, 0, 4)])
def test_gated_empty_sizes(m, k, n):
    from turboadam_amd import gated_linear

    log(f"gated {m}x{k}x{n}")
    leaves = [torch.ones(s, device="cuda", requires_grad=True) for s in ((m, k), (n, k), (n, k))]
    h = gated_linear(*leaves, activation=None)
    assert h.shape == (m, n) and bool((h == k * k).all())
    for got, leaf in zip(torch.autograd.grad(h, leaves, torch.ones_like(h)), leaves):
        assert got.shape == leaf.shape and bool((got == (2 * k * n if leaf is leaves[0] else m * k)).all())


def test_gated_gradients_of_some_arguments():
    from turboadam_amd import gated_linear

    args = _gated_case(70, 40, 50, "f32")
    leaves = [v.detach().requires_grad_() for v in args[:3]]
    whole = torch.autograd.grad(gated_linear(*leaves), leaves, args[3])
    for i in range(3):
        some = [v.detach().requires_grad_(j == i) for j, v in enumerate(args[:3])]
        got, = torch.autograd.grad(gated_linear(*some), [some[i]], args[3])
        assert torch.equal(got, whole[i]), i


@pytest.mark.parametrize("rows", [3, 80])
def test_gated_infinities_and_nan_stay_in_their_rows(rows):
    from turboadam_amd import gated_linear

    x = torch.ones(rows, 72, device="cuda")
    x[1, 5], x[2, 71] = math.inf, math.nan
    w = torch.ones(40, 72, device="cuda")
    for act in (None, "relu", "gelu", "silu", "gelu_tanh"):
        h = gated_linear(x, w, w, activation=act)
        assert bool((h[1] == math.inf).all()) and bool(h[2].isnan().all()), act
        assert bool(h[0].isfinite().all()) and bool(h[3:].isfinite().all()), act


def _differences(value, leaves, grads, what, step_size=1e-5, tolerance=1e-5):
    """Directional derivatives of value (in 64 bits) by central differences."""
    g = _gen("differences", what)
    for i, grad in enumerate(grads):
        step = torch.randn(leaves[i].shape, generator=g, device="cuda", dtype=torch.float64)
        at = [v.detach().double() for v in leaves]
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + step_size * step, at[i] - step_size * step
        want = (value(*up) - value(*down)) / (2 * step_size)
        scale = float(grad.double().norm() * step.norm())
        assert abs(float((grad.double() * step).sum() - want)) < tolerance * scale, (what, i)


def test_gated_gradient_against_differences():
    from turboadam_amd import gated_linear

    for act in ("gelu", "gelu_tanh", "silu", None):
        x, wg, wu, dh = _gated_case(50, 40, 30, "f32")
        leaves = [v.requires_grad_() for v in (x, wg, wu)]
        grads = torch.autograd.grad(gated_linear(*leaves, activation=act), leaves, dh)
        _differences(lambda x, g, u: ((ACT[act](x @ g.t()) * (x @ u.t())) * dh.double()).sum(), leaves, grads, act)


# --------------------------------------------- projection and cross entropy
def _cross_case(m, k, v, dt, ignored=0.0, scale=2.0):
    g = _gen("cross", m, k, v, dt)
    w = (torch.randn((v, k), generator=g, device="cuda") * (scale * max(k, 1) ** -0.5)).to(DTYPES[dt])
    x = _randn(g, dt, m, k)
    t = torch.randint(0, v, (m,), generator=g, device="cuda")
    t = torch.where(torch.rand((m,), generator=g, device="cuda") < ignored, torch.full_like(t, -100), t)
    return x, w, t, torch.rand((m,), generator=g, device="cuda") + 0.25


def _check_cross(x, w, t, dl, dt, reduction):
    """dl: a gradient for each row, of which a reduced loss takes the first."""
    from turboadam_amd import linear_cross_entropy

    (m, k), v, u = x.shape, w.shape[0], UNIT[dt]
    xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(xl, wl, t, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == (t.shape if reduction == "none" else ())
    dloss = dl if reduction == "none" else dl[0]
    dx, dw = torch.autograd.grad(loss, (xl, wl), dloss)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and dw.is_contiguous()
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, t, reduction=reduction), loss)
    counts = (t != -100).double()
    at = t.clamp(min=0)[:, None]
    X = torch.where(counts[:, None] > 0, x, torch.zeros_like(x)).double()
    W = w.double()
    z = X @ W.t()
    z_err = _sum_error(k) * (X.abs() @ W.abs().t())
    lse = z.logsumexp(1)
    lse_err = z_err.amax(1) + 2.0 ** -22 * (100 + v / 64)
    row = (lse - z.gather(1, at)[:, 0]) * counts
    row_err = (lse_err + z_err.gather(1, at)[:, 0] + 2.0 ** -22 * (lse.abs() + z.gather(1, at)[:, 0].abs())) * counts
    number = max(1.0, float(counts.sum()))
    if reduction == "none":
        _within(loss, row, row_err, "loss")
        weight = dl.double() * counts
    else:
        over = number if reduction == "mean" else 1.0
        _within(loss, row.sum() / over, row_err.sum() / over + 2.0 ** -23 * row.sum() / over, "loss")
        weight = torch.full_like(row, float(dl[0].double()) / over) * counts
    p = (z - lse[:, None]).exp()
    p_err = p * 1.01 * (z_err + lse_err[:, None] + 2.0 ** -22 * ((z - lse[:, None]).abs() + 4))
    p.scatter_add_(1, at, torch.full_like(lse, -1.0)[:, None])
    most = float(weight.abs().max()) if m else 0.0
    tiny = TINY[dt] * 2.0 ** -13 * most if dt == "f16" else 1e-37
    dz = p * weight[:, None]
    dz_err = weight.abs()[:, None] * ((1 + u) * (p_err + 2.0 ** -23 * (1 + p.abs())) + u * p.abs()) + tiny * counts[:, None]
    for name, got, want, err in (
            ("dx", dx, dz @ W, dz_err @ W.abs() + _sum_error(v) * (dz.abs() @ W.abs())),
            ("dw", dw, dz.t() @ X, dz_err.t() @ X.abs() + _sum_error(m) * (dz.abs().t() @ X.abs()))):
        _within(got, want, (u + 2.0 ** -22) * want.abs() + (1 + u) * err + TINY[dt], name)
    assert bool((dx[t == -100] == 0).all())
    return loss, dx, dw


CROSS = [(1, 1, 1), (1, 64, 16), (2, 4096, 130), (7, 33, 5), (16, 1000, 17), (32, 129, 641), (33, 64, 64), (64, 64, 64),
         (100, 200, 300), (129, 257, 65), (255, 40, 2), (260, 512, 264), (1, 3, 1000), (700, 8, 12), (40, 2048, 72),
         (300, 136, 2777)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("m,k,v", CROSS)
def test_cross_and_gradients(m, k, v, dt):
    for reduction, ignored in [("mean", 0.0), ("none", 0.4), ("sum", 0.9)]:
        log(f"cross {m}x{k}x{v} {dt} {reduction} ignored={ignored}")
        _check_cross(*_cross_case(m, k, v, dt, ignored), dt, reduction)


@pytest.mark.parametrize("dt", list(DTYPES))
def test_cross_large_tiles_and_split_sums(dt):
    for m, k, v in [(2048, 512, 4608), (2050, 1030, 1030), (64, 128, 30011), (5000, 24, 40), (700, 1001, 64), (701, 1001, 65),
                    (20, 96, 40000)]:
        log(f"cross {m}x{k}x{v} {dt}")
        _check_cross(*_cross_case(m, k, v, dt, 0.3), dt, "mean")


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("m,k,v", [(1, 999, 16), (15, 333, 31), (31, 1025, 32), (33, 4100, 33), (48, 515, 1), (1000, 77, 48),
                                   (97, 2050, 64), (513, 640, 15)])
def test_cross_few_words(m, k, v, dt):
    log(f"cross few words {m}x{k}x{v} {dt}")
    for reduction in ("mean", "none"):
        _check_cross(*_cross_case(m, k, v, dt, 0.3), dt, reduction)


def test_cross_few_words_of_strided_rows_and_a_graph_kept():
    from turboadam_amd import linear_cross_entropy

    x, w, t, dl = _cross_case(70, 330, 30, "bf16", 0.3)
    log("cross few words, rows inside others")
    wide, tall = torch.full((70, 401), math.nan, device="cuda").bfloat16(), torch.full((30, 333), math.nan, device="cuda").bfloat16()
    wide[:, 3:333], tall[:, 1:331] = x, w
    for a, b in zip(_check_cross(wide[:, 3:333], tall[:, 1:331], t, dl, "bf16", "none"), _check_cross(x, w, t, dl, "bf16", "none")):
        assert torch.equal(a, b)
    xl, wl = x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(xl, wl, t)
    both = torch.autograd.grad(loss, (xl, wl), retain_graph=True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(xl, wl.detach(), t), xl)[0], both[0])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(xl.detach(), wl, t), wl)[0], both[1])
    first, _ = torch.autograd.grad(loss, (xl, wl), retain_graph=True), linear_cross_entropy(xl * 2, wl, t)
    for a, b in zip(first, torch.autograd.grad(loss, (xl, wl))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("rows", [3, 32, 70])
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_cross_rows_that_do_not_count_reach_nothing(rows, reduction, dt):
    from turboadam_amd import linear_cross_entropy

    x, w, t, dl = _cross_case(rows, 40, 100, dt)
    t[1::2] = -100
    log(f"cross nan in ignored rows {rows} {reduction} {dt}")
    want = _check_cross(x, w, t, dl, dt, reduction)
    x = x.clone()
    x[1], x[-1 if rows % 2 == 0 else -2] = math.nan, math.inf
    dl = dl.clone()
    if reduction == "none":
        dl[1] = math.nan
    for got, v in zip(_check_cross(x, w, t, dl, dt, reduction), want):
        assert torch.equal(got, v)
    log("cross of no row that counts")
    t = torch.full_like(t, -100)
    xl, wl = x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(xl, wl, t, reduction=reduction)
    assert bool((loss == 0).all())
    for grad in torch.autograd.grad(loss, (xl, wl), torch.ones_like(loss)):
        assert bool((grad == 0).all())


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("rows,vocabulary", [(5, 100), (70, 100), (70, 30), (0, 30)])
def test_cross_of_no_row_that_counts_and_an_infinite_gradient(rows, vocabulary, reduction):
    from turboadam_amd import linear_cross_entropy

    x, w, t, _ = _cross_case(rows, 40, vocabulary, "bf16")
    x, w, t = x.requires_grad_(), w.requires_grad_(), torch.full_like(t, -100)
    log(f"cross of no row of {rows}, {vocabulary} words, {reduction}, an infinite gradient")
    loss = linear_cross_entropy(x, w, t, reduction=reduction)
    for value in (math.inf, math.nan):
        for grad in torch.autograd.grad(loss, (x, w), torch.full_like(loss, value), retain_graph=True):
            assert bool((grad == 0).all())


@pytest.mark.parametrize("rows", [3, 70])
def test_cross_targets_outside_the_vocabulary_are_nan(rows):
    from turboadam_amd import linear_cross_entropy

    for bad in (100, -1, -99, 1 << 32, -(1 << 32) + 5):
        x, w, t, dl = _cross_case(rows, 40, 100, "f32")
        t[2] = bad
        log(f"cross target {bad} of {rows} rows")
        x, w = x.requires_grad_(), w.requires_grad_()
        loss = linear_cross_entropy(x, w, t, reduction="none")
        assert bool(loss[2].isnan()) and bool(loss[:2].isfinite().all()) and bool(loss[3:].isfinite().all())
        assert bool(linear_cross_entropy(x, w, t).isnan())
        dx, dw = torch.autograd.grad(loss, (x, w), dl)
        assert bool(dx[2].isnan().all()) and bool(dx[:2].isfinite().all()) and bool(dw.isnan().all())


@pytest.mark.parametrize("rows", [4, 60])
def test_cross_of_infinite_and_nan_logits(rows):
    from turboadam_amd import linear_cross_entropy

    x, w, t, _ = _cross_case(rows, 16, 90, "f32")
    want = linear_cross_entropy(x, w, t, reduction="none")
    x = x.clone()
    x[0, 3], x[1, 0], x[2] = math.nan, math.inf, 1e30
    got = linear_cross_entropy(x, w, t, reduction="none")
    assert bool(got[:2].isnan().all()) and not bool(got[2].isnan()) and torch.equal(got[3:], want[3:])
    log("cross of words that cannot be: logits of -inf")
    x, w = torch.ones(rows, 8, device="cuda"), torch.zeros(90, 8, device="cuda")
    w[5:] = -math.inf
    x = x.requires_grad_()
    loss = linear_cross_entropy(x, w, torch.zeros(rows, dtype=torch.long, device="cuda"), reduction="none")
    assert bool(((loss - math.log(5.0)).abs() < 1e-6).all())


def test_cross_shapes_reductions_and_strides():
    from turboadam_amd import linear_cross_entropy

    x, w, t, dl = _cross_case(60, 50, 77, "bf16", 0.2)
    want = linear_cross_entropy(x, w, t, reduction="none")
    log("cross of leading dimensions, strided rows and a transposed weight")
    assert torch.equal(linear_cross_entropy(x.reshape(3, 4, 5, 50), w, t.reshape(3, 4, 5), reduction="none"),
                       want.reshape(3, 4, 5))
    assert torch.equal(linear_cross_entropy(_amid_nan(x), _amid_nan(w), t, reduction="none"), want)
    assert torch.equal(linear_cross_entropy(x, w.t().contiguous().t(), t, reduction="none"), want)
    every = torch.zeros(60, 2, dtype=torch.long, device="cuda")
    every[:, 0] = t
    assert torch.equal(linear_cross_entropy(x, w, every[:, 0], reduction="none"), want)
    assert torch.equal(linear_cross_entropy(x[7], w, t[7], reduction="none"),
                       linear_cross_entropy(x[7:8], w, t[7:8], reduction="none")[0])
    assert torch.equal(linear_cross_entropy(x, w, torch.where(t == -100, 3, t), reduction="none", ignore_index=3)[t == 3],
                       torch.zeros_like(want[t == 3]))
    log("cross gradients of a sum of rows, of strided gradients and of gradients of any size")
    xl, wl = x.requires_grad_(), w.requires_grad_()

    def grads(d):
        return torch.autograd.grad(linear_cross_entropy(xl, wl, t, reduction="none"), (xl, wl), d)

    for a, b in zip(grads(torch.ones(1, device="cuda").expand(60)), grads(torch.ones(60, device="cuda"))):
        assert torch.equal(a, b)
    for a, b in zip(grads(torch.stack((dl, dl), 1)[:, 0]), grads(dl)):
        assert torch.equal(a, b)
    for power in (-60, -20, 20, 60):  # a power of two changes no bit of a bf16 gradient's digits
        for a, b in zip(grads(dl * 2.0 ** power), grads(dl)):
            assert torch.equal(a.double() * 2.0 ** -power, b.double()), power
    for a in grads(torch.zeros(60, device="cuda")):
        assert bool((a == 0).all())


def test_cross_empty_sizes():
    from turboadam_amd import linear_cross_entropy

    w = torch.ones(9, 8, device="cuda", requires_grad=True)
    x = torch.ones(0, 8, device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.long, device="cuda")
    for reduction in ("none", "sum", "mean"):
        loss = linear_cross_entropy(x, w, t, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and bool((loss == 0).all())
        dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
        assert dx.shape == (0, 8) and bool((dw == 0).all())
    for rows in (5, 50):
        x, w = torch.ones(rows, 0, device="cuda", requires_grad=True), torch.ones(9, 0, device="cuda", requires_grad=True)
        loss = linear_cross_entropy(x, w, torch.zeros(rows, dtype=torch.long, device="cuda"))
        assert abs(float(loss.detach()) - math.log(9.0)) < 1e-6
        dx, dw = torch.autograd.grad(loss, (x, w))
        assert dx.shape == (rows, 0) and dw.shape == (9, 0)


def test_cross_gradient_against_differences():
    from turboadam_amd import linear_cross_entropy

    x, w, t, dl = _cross_case(50, 40, 33, "f32", 0.2)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    for reduction in ("none", "mean", "sum"):
        loss = linear_cross_entropy(*leaves, t, reduction=reduction)
        d = dl if reduction == "none" else dl[0]
        grads = torch.autograd.grad(loss, leaves, d)

        def value(x, w):
            return (F.cross_entropy(x @ w.t(), t, reduction=reduction) * d.double()).sum()

        _differences(value, leaves, grads, reduction)


@pytest.mark.parametrize("dt", list(DTYPES))
def test_cross_in_pieces_of_the_vocabulary(dt):
    """The C entry with pieces of 256 words: dw has the same bits, dx the same sum in another order."""
    import ctypes

    from turboadam_amd import _lib, linear_cross_entropy

    lib = _lib.load()
    m, k, v = 200, 72, 1111
    x, w, t, _ = _cross_case(m, k, v, dt, 0.25)
    xl, wl = x.requires_grad_(), w.requires_grad_()
    log(f"cross in pieces {dt}")
    loss = linear_cross_entropy(xl, wl, t, reduction="sum")
    whole = torch.autograd.grad(loss, (xl, wl), torch.ones_like(loss))
    d = _lib.TamCross()
    d.x, d.w, d.target = x.data_ptr(), w.data_ptr(), t.data_ptr()
    d.rows, d.inputs, d.vocabulary, d.ldx, d.ldw, d.ignored = m, k, v, k, k, -100
    d.dtype, d.reduction, d.piece = _lib.DTYPES[x.dtype], _lib.TAM_CROSS_SUM, 256
    kept = torch.empty(lib.tam_cross_kept(ctypes.byref(d)), dtype=torch.uint8, device="cuda")
    out, one = torch.empty((), device="cuda"), torch.ones((), device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    d.loss, d.kept, d.dloss, d.dx, d.dw = out.data_ptr(), kept.data_ptr(), one.data_ptr(), dx.data_ptr(), dw.data_ptr()
    stream = _lib.stream_of(x.device)
    for backward, call in ((0, lib.tam_cross), (1, lib.tam_cross_backward)):
        need = ctypes.c_size_t()
        _lib.check(lib.tam_cross_workspace(ctypes.byref(d), backward, ctypes.byref(need)), "workspace")
        ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
        _lib.check(call(ctypes.byref(d), ws.data_ptr(), need.value, stream), "cross")
        torch.cuda.synchronize()
    tiles = (ctypes.c_uint32 * 4)()
    assert lib.tam_cross_tiles(ctypes.byref(d), 1, tiles) == 0 and tiles[1] == 256
    assert torch.equal(out, loss) and torch.equal(dw, whole[1])
    scale = float(whole[0].double().abs().max())
    assert float((dx.double() - whole[0].double()).abs().max()) <= (UNIT[dt] * 4 + 2.0 ** -18) * scale


# ------------------------------------------------------------------ rotary
def _turned(x, angle, rotated, interleaved, magnitude, back=False):
    cos, sin = angle.cos() * magnitude, angle.sin() * magnitude * (-1 if back else 1)
    a, b = (x[..., 0:rotated:2], x[..., 1:rotated:2]) if interleaved else (x[..., :rotated // 2], x[..., rotated // 2:rotated])
    ya, yb = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((ya, yb), -1).flatten(-2) if interleaved else torch.cat((ya, yb), -1)
    both = (a.abs() + b.abs()) * magnitude
    err = torch.stack((both, both), -1).flatten(-2) if interleaved else torch.cat((both, both), -1)
    return torch.cat((y, x[..., rotated:]), -1), torch.cat((err, x[..., rotated:].abs()), -1)


def _check_rotary(q, k, positions, frequencies, dt, interleaved=False, magnitude=1.0, wq=None, wk=None, eps=1e-6, dq=None,
                  dk=None):
    from turboadam_amd import rotary

    u, tiny, d, r = UNIT[dt], TINY[dt], q.shape[-1], 2 * frequencies.numel()
    leaves = {n: v.detach().requires_grad_() for n, v in (("q", q), ("k", k), ("wq", wq), ("wk", wk)) if v is not None}
    out = rotary(leaves["q"], leaves.get("k"), positions, frequencies, interleaved=interleaved, magnitude=magnitude,
                 q_weight=leaves.get("wq"), k_weight=leaves.get("wk"), eps=eps)
    out = [out] if k is None else list(out)
    dys = [dq, dk][:len(out)]
    grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dys)))
    with torch.no_grad():
        again = rotary(q, k, positions, frequencies, interleaved=interleaved, magnitude=magnitude, q_weight=wq, k_weight=wk,
                       eps=eps)
        for a, b in zip([again] if k is None else again, out):
            assert torch.equal(a, b)
    angle = (positions.double().expand(q.shape[:-2])[..., None] * frequencies)[..., None, :]
    rel = (d + 64) * 2.0 ** -24  # of a normed element, before it is rounded
    for name, x, w, y, dy in (("q", q, wq, out[0], dq), ("k", k, wk, out[-1], dk)):
        if x is None:
            continue
        X, D = x.double(), dy.double()
        n0, rstd = X, 1.0
        if w is not None:
            rstd = (X.square().mean(-1, keepdim=True) + eps).rsqrt()
            n0 = X * rstd
        n = n0 if w is None else n0 * w.double()
        want, parts = _turned(n, angle, r, interleaved, magnitude)
        slack = 2.0 ** -21 + (0 if w is None else rel)
        assert y.shape == x.shape and y.dtype == x.dtype
        _within(y, want, u * want.abs() + (1 + u) * slack * parts + tiny, name)
        t, parts = _turned(D, angle, r, interleaved, magnitude, back=True)
        t_err = 2.0 ** -21 * parts
        if w is None:
            _within(grads[name], t, u * t.abs() + (1 + u) * t_err + tiny, "d" + name)
            continue
        W = w.double()
        rows = max(1, X[..., 0].numel())
        dims = tuple(range(X.dim() - 1))
        dw = (t * n0).sum(dims)
        dw_err = ((t_err + t.abs() * (rel + 2.0 ** -22)) * n0.abs()).sum(dims) + _sum_error(rows) * (t * n0).abs().sum(dims)
        _within(grads["w" + name], dw, u * dw.abs() + (1 + u) * dw_err + tiny, "dw" + name)
        g = t * W
        g_err = t_err * W.abs() + 2.0 ** -23 * g.abs()
        mean = (g * n0).mean(-1, keepdim=True)
        mean_err = ((g_err + g.abs() * (2 * rel + _sum_error(d))) * n0.abs()).mean(-1, keepdim=True)
        dx = rstd * (g - n0 * mean)
        err = rstd * (g_err + n0.abs() * mean_err + (3 * rel + 2.0 ** -21) * (g.abs() + (n0 * mean).abs()))
        _within(grads[name], dx, u * dx.abs() + (1 + u) * err + tiny, "d" + name)
    return out, grads


def _rotary_case(b, t, hq, hk, d, pairs, dt, norm, start=0):
    from turboadam_amd import rotary_frequencies

    g = _gen("rotary", b, t, hq, hk, d, pairs, dt, norm)
    q, k = _randn(g, dt, b, t, hq, d), _randn(g, dt, b, t, hk, d)
    f = rotary_frequencies(2 * pairs, device="cuda") if pairs else torch.zeros(0, dtype=torch.float64, device="cuda")
    w = [(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(DTYPES[dt]) if norm else None for _ in range(2)]
    positions = torch.arange(start, start + t, device="cuda")
    return q, k, positions, f, w, _randn(g, dt, b, t, hq, d), _randn(g, dt, b, t, hk, d)


ROTARY = [(1, 1, 1, 1, 1, 0), (1, 1, 32, 8, 128, 64), (2, 3, 5, 2, 2, 1), (1, 7, 3, 1, 64, 32), (2, 33, 12, 12, 64, 32),
          (3, 50, 7, 3, 84, 10), (1, 9, 40, 40, 80, 40), (2, 5, 6, 2, 33, 7), (1, 130, 2, 1, 8, 4), (1, 6, 9, 3, 256, 128),
          (2, 4, 3, 2, 1024, 512), (1, 5, 2, 1, 1008, 500), (1, 300, 1, 1, 17, 0), (1, 3, 70, 1, 48, 24), (2, 700, 4, 4, 32, 16),
          (1, 4, 2, 2, 576, 32)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("b,t,hq,hk,d,pairs", ROTARY)
def test_rotary_and_gradients(b, t, hq, hk, d, pairs, dt):
    for interleaved, norm, magnitude, start in [(False, True, 1.0, 0), (True, True, 1.25, 999), (False, False, 0.75, 131000),
                                                (True, False, 1.0, 5)]:
        q, k, p, f, w, dq, dk = _rotary_case(b, t, hq, hk, d, pairs, dt, norm, start)
        log(f"rotary {b}x{t} {hq}/{hk} heads of {d}, {pairs} pairs {dt} interleaved={interleaved} norm={norm}")
        _check_rotary(q, k, p, f, dt, interleaved, magnitude, w[0], w[1], dq=dq, dk=dk)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_rotary_many_tokens_and_one_norm_of_two(dt):
    q, k, p, f, w, dq, dk = _rotary_case(2, 5000, 4, 2, 64, 32, dt, True)
    log(f"rotary many tokens {dt}")
    _check_rotary(q, k, p, f, dt, wq=w[0], wk=w[1], dq=dq, dk=dk)
    log("rotary of queries normed alone, of keys normed alone, of queries alone")
    q, k, p, f, w, dq, dk = _rotary_case(2, 40, 4, 2, 64, 32, dt, True)
    _check_rotary(q, k, p, f, dt, wq=w[0], dq=dq, dk=dk)
    _check_rotary(q, k, p, f, dt, wk=w[1], dq=dq, dk=dk)
    _check_rotary(q, None, p, f, dt, wq=w[0], dq=dq)
    _check_rotary(q, None, p, f, dt, dq=dq)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_rotary_strides(dt, norm):
    from turboadam_amd import rotary

    b, t, hq, hk, d = 2, 19, 6, 2, 40
    q, k, p, f, w, dq, dk = _rotary_case(b, t, hq, hk, d, 20, dt, norm, 7)
    kw = dict(q_weight=w[0], k_weight=w[1])
    want = rotary(q, k, p, f, **kw)
    log(f"rotary of slices of a joint projection {dt} {norm}")
    joint = torch.full((b, t, (hq + 2 * hk) * d + 3), float("nan"), device="cuda", dtype=q.dtype)
    jq, jk = joint[..., 1:1 + hq * d].unflatten(-1, (hq, d)), joint[..., 1 + hq * d:1 + (hq + hk) * d].unflatten(-1, (hk, d))
    jq.copy_(q)
    jk.copy_(k)
    for a, c in zip(rotary(jq, jk, p, f, **kw), want):
        assert torch.equal(a, c) and a.is_contiguous()
    log("rotary of heads before tokens, results in the same order, gradients in any")
    turned = [v.transpose(1, 2).contiguous().transpose(1, 2) for v in (q, k)]
    for a, c, v in zip(rotary(*turned, p, f, **kw), want, turned):
        assert torch.equal(a, c) and a.stride() == v.stride()
    _check_rotary(*turned, p, f, dt, wq=w[0], wk=w[1], dq=dq.transpose(1, 2).contiguous().transpose(1, 2),
                  dk=_amid_nan(dk))
    log("rotary of three and five dimensions, expanded heads and positions of their own")
    for a, c in zip(rotary(q[1], k[1], p, f, **kw), want):
        assert torch.equal(a, c[1])
    for a, c in zip(rotary(q[None], k[None], p.expand(1, b, t), f, **kw), want):
        assert torch.equal(a, c[None])
    own = torch.stack((p, p.flip(0) * 3))
    _check_rotary(q, k, own, f, dt, wq=w[0], wk=w[1], dq=dq, dk=dk)
    _check_rotary(q, k, own.t().contiguous().t().int(), f, dt, wq=w[0], wk=w[1], dq=dq, dk=dk)
    _check_rotary(q, k, p[3], f, dt, wq=w[0], wk=w[1], dq=dq, dk=dk)
    _check_rotary(q, k[:, :, :1].expand(b, t, hk, d), p, f, dt, wq=w[0], wk=w[1], dq=dq, dk=dk)
    _check_rotary(q, k, p, f, dt, wq=w[0], wk=w[1], dq=dq[:, :1, :1].expand(b, t, hq, d), dk=dk)


def test_rotary_far_positions_and_turning_back():
    from turboadam_amd import rotary, rotary_frequencies

    g = _gen("far")
    f = rotary_frequencies(64, base=500000.0, device="cuda")
    p = torch.tensor([0, 1, -1, 1 << 20, (1 << 31) + 5, -(1 << 40), (1 << 40) + 1], device="cuda")
    q, dq = torch.randn(7, 2, 64, generator=g, device="cuda"), torch.randn(7, 2, 64, generator=g, device="cuda")
    near = p.abs() <= 1 << 20  # farther on, the angle itself is a rounded product
    _check_rotary(q[near], None, p[near], f, "f32", dq=dq[near])
    y = rotary(q, None, p, f)
    assert torch.equal(y[0], q[0])
    assert float((rotary(y, None, -p, f) - q).abs().max()) < 2.0 ** -19
    # the length of a pair stays, and angles depend on differences of positions alone
    assert torch.allclose(y.square().sum(-1), q.square().sum(-1), rtol=1e-5)
    shifted = rotary(rotary(q, None, p, f), None, torch.full((7,), 77, device="cuda"), f)
    # an angle is a product of a position and a frequency in turns that are each rounded to 2^-53 of it, so of
    # p f radians, f <= 1, either side is off by up to 3 2^-53 |p|, times the pair's |a| + |b| (at 2^40: 7e-4)
    pair = q[..., :32].abs() + q[..., 32:].abs()
    slack = 2e-5 + 6 * 2.0 ** -53 * (p.abs() + 77).double()[:, None, None] * torch.cat((pair, pair), -1).double()
    assert bool(((shifted.double() - rotary(q, None, p + 77, f).double()).abs() <= slack).all())


def test_rotary_nan_stays_in_its_head():
    from turboadam_amd import rotary

    q, k, p, f, w, _, _ = _rotary_case(1, 9, 5, 2, 64, 32, "f32", True)
    want = rotary(q, k, p, f, q_weight=w[0], k_weight=w[1])
    q = q.clone()
    q[0, 3, 2, 7], q[0, 4, 1, 63] = math.nan, math.inf
    got = rotary(q, k, p, f, q_weight=w[0], k_weight=w[1])
    same = torch.ones(1, 9, 5, dtype=torch.bool, device="cuda")
    same[0, 3, 2] = same[0, 4, 1] = False
    assert bool(got[0][0, 3, 2].isnan().all()) and torch.equal(got[0][same], want[0][same]) and torch.equal(got[1], want[1])
    zero = rotary(torch.zeros_like(k), None, p, f, q_weight=w[0])
    assert bool((zero == 0).all())


@pytest.mark.parametrize("shape", [(0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8), (0, 2, 8)])
def test_rotary_empty_sizes(shape):
    from turboadam_amd import rotary

    log(f"rotary of {shape}")
    f = torch.ones(4, dtype=torch.float64, device="cuda")
    q, k, w = [torch.ones(s, device="cuda", requires_grad=True) for s in (shape, shape, (8,))]
    p = torch.arange(shape[-3], device="cuda")
    out = rotary(q, k, p, f, q_weight=w)
    assert out[0].shape == shape and out[1].shape == shape
    for got, leaf in zip(torch.autograd.grad(out, (q, k, w), out), (q, k, w)):
        assert got.shape == leaf.shape and bool((got == 0).all())


def test_rotary_gradients_of_some_arguments_and_of_one_output():
    from turboadam_amd import rotary

    q, k, p, f, w, dq, dk = _rotary_case(2, 30, 4, 2, 48, 16, "f32", True)
    args = dict(q=q, k=k, q_weight=w[0], k_weight=w[1])

    def call(names):
        a = {n: v.detach().requires_grad_(n in names) for n, v in args.items()}
        return a, rotary(a["q"], a["k"], p, f, q_weight=a["q_weight"], k_weight=a["k_weight"])

    # which rows a lane adds up, and so a weight's sum of n terms, whose order may be any, depends on the heads of
    # the call: two right sums are within twice _sum_error(n) of the sum of absolute values of each other
    angle = (p.double()[:, None] * f)[None, :, None, :]
    slack = {}
    for n, x, dy in (("q_weight", q, dq), ("k_weight", k, dk)):
        t, _ = _turned(dy.double(), angle, 32, False, 1.0, back=True)
        n0 = x.double() * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        slack[n] = 2 * _sum_error(60 * x.shape[2]) * (t * n0).abs().sum((0, 1, 2))

    def same(n, got):
        return torch.equal(got, whole[n]) if n in "qk" else bool(((got - whole[n]).abs().double() <= slack[n]).all())

    a, out = call(list(args))
    whole = dict(zip(a, torch.autograd.grad(out, list(a.values()), (dq, dk))))
    for n in args:
        b, out = call([n])
        got, = torch.autograd.grad(out, [b[n]], (dq, dk), allow_unused=True)
        assert same(n, got), n
    for i, (dy, with_) in enumerate(((dq, ("q", "q_weight")), (dk, ("k", "k_weight")))):
        a, out = call(list(args))
        for n, got in zip(a, torch.autograd.grad(out[i], list(a.values()), dy, allow_unused=True)):
            assert same(n, got) if n in with_ else got is None, n


def test_rotary_gradient_against_differences():
    from turboadam_amd import rotary

    for interleaved in (False, True):
        q, k, p, f, w, dq, dk = _rotary_case(1, 11, 3, 2, 20, 7, "f32", True, 50)
        leaves = [v.requires_grad_() for v in (q, k, w[0], w[1])]
        out = rotary(q, k, p, f, interleaved=interleaved, magnitude=1.1, q_weight=w[0], k_weight=w[1])
        grads = torch.autograd.grad(out, leaves, (dq, dk))
        angle = (p.double()[:, None] * f)[None, :, None, :]

        def value(q, k, wq, wk):
            total = 0.0
            for x, w, dy in ((q, wq, dq), (k, wk, dk)):
                n = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
                total = total + (_turned(n, angle, 14, interleaved, 1.1)[0] * dy.double()).sum()
            return total

        _differences(value, leaves, grads, ("rotary", interleaved))


# ------------------------------------------------------------ all of them
def _streams_case():
    g = _gen("streams")
    x, wg, wu, _ = _gated_case(900, 264, 300, "bf16")
    head = _randn(g, "bf16", 1000, 300)
    t = torch.randint(0, 1000, (900,), generator=g, device="cuda")
    t[::7] = -100
    q, k, p, f, w, dq, dk = _rotary_case(1, 900, 4, 2, 64, 32, "bf16", True)
    leaves = [v.detach().requires_grad_() for v in (x, wg, wu, head, q, k, w[0], w[1])]

    def call():
        from turboadam_amd import gated_linear, linear_cross_entropy, rotary

        h = gated_linear(*leaves[:3])
        loss = linear_cross_entropy(h, leaves[3], t)
        r = rotary(leaves[4], leaves[5], p, f, q_weight=leaves[6], k_weight=leaves[7])
        return [h.detach(), loss.detach(), r[0].detach(), r[1].detach(),
                *torch.autograd.grad((loss, *r), leaves, (torch.ones_like(loss), dq, dk))]

    return leaves, call


def test_same_bits_every_time_and_on_another_stream():
    _, call = _streams_case()
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = call()
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(first, second):
        assert torch.equal(a, c)


def test_in_a_captured_graph():
    leaves, call = _streams_case()
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
            for leaf in (leaves[0], leaves[4]):
                leaf.copy_(torch.randn(leaf.shape, generator=_gen(i), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, call()):
            assert torch.equal(a, c), f"replay {i}"


def test_two_streams_at_once_and_two_graphs_of_one_pool():
    """Calls of one process that overlap, and captured ones whose workspaces share their memory: no call's
    workspace is another's while it is needed."""
    cases = [_streams_case(), _streams_case()]
    with torch.no_grad():
        for leaf in cases[1][0]:
            leaf.mul_(0.5)
    want = [[v.clone() for v in call()] for _, call in cases]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (_, call) in enumerate(cases):
            with torch.cuda.stream(sides[i]):
                got[i].append(call())
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            for a, c in zip(out, want[i]):
                assert torch.equal(a, c), i
    graphs, outs = [], []
    for _, call in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(call())
        graphs.append(graph)
    for turn in range(3):
        for i in range(2):
            graphs[i].replay()
            torch.cuda.synchronize()
            for a, c in zip(outs[i], want[i]):
                assert torch.equal(a, c), (turn, i)
            for a, c in zip(cases[i][1](), want[i]):
                assert torch.equal(a, c), (turn, i)


def test_refusals():
    from turboadam_amd import gated_linear, linear_cross_entropy, rotary

    x, w = torch.ones(4, 8, device="cuda"), torch.ones(6, 8, device="cuda")
    t = torch.zeros(4, dtype=torch.long, device="cuda")
    q, f, p = torch.ones(4, 2, 8, device="cuda"), torch.ones(4, dtype=torch.float64, device="cuda"), torch.arange(4, device="cuda")
    for error, text, call in [
            (ValueError, "gate", lambda: gated_linear(x, w[:, :7], w)),
            (ValueError, "up must", lambda: gated_linear(x, w, w[:5])),
            (ValueError, "up must be", lambda: gated_linear(x, w, w.half())),
            (RuntimeError, "up must be dense", lambda: gated_linear(x, w, w.cpu())),
            (ValueError, "activation", lambda: gated_linear(x, w, w, activation="tanh")),
            (ValueError, "float32", lambda: gated_linear(x.double(), w, w)),
            (ValueError, "weight", lambda: linear_cross_entropy(x, w[:, :7], t)),
            (ValueError, "int64", lambda: linear_cross_entropy(x, w, t.int())),
            (ValueError, "target must have", lambda: linear_cross_entropy(x, w, t[:3])),
            (RuntimeError, "target must be dense", lambda: linear_cross_entropy(x, w, t.cpu())),
            (ValueError, "reduction", lambda: linear_cross_entropy(x, w, t, reduction="max")),
            (ValueError, "vocabulary", lambda: linear_cross_entropy(x, w[:0], t)),
            (ValueError, "tokens, heads", lambda: rotary(x, None, p, f)),
            (ValueError, "k must", lambda: rotary(q, q[:3], p, f)),
            (ValueError, "k must", lambda: rotary(q, q[..., :6], p, f)),
            (ValueError, "broadcast", lambda: rotary(q, None, p[:3], f)),
            (ValueError, "int64 or int32", lambda: rotary(q, None, p.float(), f)),
            (ValueError, "float64", lambda: rotary(q, None, p, f.float())),
            (ValueError, "at most 4 pairs", lambda: rotary(q, None, p, torch.ones(5, dtype=torch.float64, device="cuda"))),
            (RuntimeError, "no gradient", lambda: rotary(q, None, p, f.clone().requires_grad_())),
            (ValueError, "eps", lambda: rotary(q, None, p, f, eps=-1.0)),
            (ValueError, "q_weight", lambda: rotary(q, None, p, f, q_weight=w[0, :7])),
            (ValueError, "without k", lambda: rotary(q, None, p, f, k_weight=w[0])),
            (RuntimeError, "1024", lambda: rotary(torch.ones(1, 1, 1030, device="cuda"), None, p[:1], f))]:
        with pytest.raises(error, match=text):
            call()


def test_what_has_no_derivative_raises():
    import torch.autograd.forward_ad as fwd

    from turboadam_amd import gated_linear, linear_cross_entropy, rotary

    x, w = torch.ones(4, 8, device="cuda", requires_grad=True), torch.ones(6, 8, device="cuda", requires_grad=True)
    t = torch.zeros(4, dtype=torch.long, device="cuda")
    q = torch.ones(4, 2, 8, device="cuda", requires_grad=True)
    f, p = torch.ones(4, dtype=torch.float64, device="cuda"), torch.arange(4, device="cuda")
    calls = {"gated_linear": (lambda x, q: gated_linear(x, w, w)), "linear_cross_entropy": (lambda x, q: linear_cross_entropy(x, w, t)),
             "rotary": (lambda x, q: rotary(q, None, p, f))}
    for name, call in calls.items():
        y = call(x, q)
        with pytest.raises(RuntimeError, match=f"{name}.*create_graph"):
            torch.autograd.grad(y.sum(), q if name == "rotary" else x, create_graph=True)
        with fwd.dual_level(), pytest.raises(RuntimeError, match=f"{name}.*dual"):
            call(fwd.make_dual(x.detach(), torch.ones_like(x)), fwd.make_dual(q.detach(), torch.ones_like(q)))
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(lambda x, q: call(x, q), (x.detach(), q.detach()), check_trace=False)


# ------------------------------------------------- every tile, and offsets past 32 bits
def _gated_tiles(m, k, n, dt, backward, in_out=False):
    import ctypes

    from turboadam_amd import _lib

    d = _lib.TamGated()
    d.x = d.gate = d.up = d.h = d.kept = d.dh = d.dx = d.dgate = d.dup = 0x10000
    d.rows, d.inputs, d.outputs, d.ldx, d.ldw = m, k, n, k, n if in_out else k
    d.w_in_out, d.dtype = in_out, _lib.DTYPES[DTYPES[dt]]
    out = (ctypes.c_uint32 * 4)()
    assert _lib.load().tam_gated_tiles(ctypes.byref(d), backward, out) == 0
    return list(out)


@pytest.mark.parametrize("m,k,n,dt,tiles", [
    (4096, 512, 4000, "bf16", [256, 1]), (5000, 264, 1200, "f16", [256, 1]), (300, 200, 1000, "bf16", [64, 1]),
    (96, 8192, 80, "bf16", [64, 32]), (1100, 8192, 520, "f16", [128, 3]), (2048, 512, 2048, "f32", [128, 1]),
    (200, 2048, 130, "f32", [64, 12])])
def test_gated_tiles_forward(m, k, n, dt, tiles):
    # several tiles to a workgroup where they are the largest, ragged ones among them, sums in one part and in more
    log(f"gated {m}x{k}x{n} {dt} tiles {_gated_tiles(m, k, n, dt, 0)}")
    assert _gated_tiles(m, k, n, dt, 0)[:2] == tiles
    _check_gated(*_gated_case(m, k, n, dt), dt, "silu")


@pytest.mark.parametrize("m,k,n,dt,in_out,tile,x_parts,w_parts", [
    (6000, 2048, 3000, "bf16", False, 128, 1, 1), (6000, 2048, 3000, "f16", True, 128, 1, 1),
    (2048, 2048, 4096, "bf16", False, 256, 2, 1), (2048, 2048, 4096, "f16", True, 256, 2, 1),
    (300, 200, 200, "bf16", True, 64, 1, 1), (1024, 1024, 2048, "f32", False, 128, 4, 1),
    (5000, 40, 60, "bf16", False, 64, 1, 32)])
def test_gated_tiles_backward(m, k, n, dt, in_out, tile, x_parts, w_parts):
    got = _gated_tiles(m, k, n, dt, 1, in_out)
    log(f"gated {m}x{k}x{n} {dt} in_out={in_out} tiles {got}")
    assert got == [tile, x_parts, tile, w_parts]
    _check_gated(*_gated_case(m, k, n, dt, in_out), dt, "gelu")


def _cross_tiles(m, k, v, dt, backward):
    import ctypes

    from turboadam_amd import _lib

    d = _lib.TamCross()
    d.x = d.w = d.target = d.loss = d.kept = d.dloss = d.dx = d.dw = 0x10000
    d.rows, d.inputs, d.vocabulary, d.ldx, d.ldw, d.dtype = m, k, v, k, k, _lib.DTYPES[DTYPES[dt]]
    out = (ctypes.c_uint32 * 4)()
    assert _lib.load().tam_cross_tiles(ctypes.byref(d), backward, out) == 0
    return list(out)


@pytest.mark.parametrize("m,k,v,dt,z,both,x_parts,w_parts", [
    (4096, 264, 9973, "bf16", 256, 128, 2, 1), (4096, 1032, 9973, "f16", 256, 256, 3, 1), (1000, 300, 2100, "bf16", 64, 64, 2, 1),
    (8192, 40, 2100, "f16", 128, 64, 2, 8), (4000, 1024, 4000, "f32", 128, 128, 1, 1), (200, 100, 700, "f32", 64, 64, 2, 1),
    (8192, 768, 20011, "bf16", 256, 256, 2, 1), (5000, 24, 40, "f32", 0, 64, 1, 32)])
def test_cross_tiles(m, k, v, dt, z, both, x_parts, w_parts):
    got = _cross_tiles(m, k, v, dt, 1)
    log(f"cross {m}x{k}x{v} {dt} tiles {_cross_tiles(m, k, v, dt, 0)} and {got}")
    assert _cross_tiles(m, k, v, dt, 0)[0] == z and [got[0], *got[2:]] == [z, both, x_parts << 16 | w_parts]
    for ignored in (0.0, 0.6, 0.95):  # where few rows count, dx's sums are cut into more parts
        _check_cross(*_cross_case(m, k, v, dt, ignored), dt, "none" if ignored == 0.6 else "mean")


def _whole(g, *shape):
    return torch.randint(-3, 4, shape, generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)


def test_gated_offsets_past_32_bits():
    """Outputs of 2.3e9 elements, in whole numbers: every row, and the sums over all of them."""
    from turboadam_amd import gated_linear

    g = _gen("long")
    m, k, n = 70001, 24, 32768
    x, wg, wu, dh = _whole(g, m, k).requires_grad_(), _whole(g, n, k).requires_grad_(), _whole(g, n, k).requires_grad_(), \
        _whole(g, m, n)
    log(f"gated {m}x{k}x{n}")
    h = gated_linear(x, wg, wu, activation="relu")
    dx, dgate, dup = torch.autograd.grad(h, (x, wg, wu), dh)
    X, G, U = x.detach().double(), wg.detach().double(), wu.detach().double()
    sums = torch.zeros_like(G), torch.zeros_like(U)
    for i in range(0, m, 5000):
        rows = slice(i, min(i + 5000, m))
        z, u, d = X[rows] @ G.t(), X[rows] @ U.t(), dh[rows].double()
        assert torch.equal(h[rows], (z.relu() * u).to(h.dtype)), i
        dz, du = (d * u * (z > 0)).bfloat16().double(), (d * z.relu()).bfloat16().double()
        want = dz @ G + du @ U  # sums of whole numbers past fp32's: in any order within 2^-23 (n + 16) of their parts
        slack = (dz.abs() @ G.abs() + du.abs() @ U.abs()) * _sum_error(2 * n) + want.abs() * UNIT["bf16"]
        assert bool(((dx[rows].double() - want).abs() <= slack).all()), i
        sums[0].add_(dz.t() @ X[rows])
        sums[1].add_(du.t() @ X[rows])
    for got, want in zip((dgate, dup), sums):  # of 70001 whole numbers up to 2^11
        assert float((got.double() - want).norm()) <= (UNIT["bf16"] + 2.0 ** -18) * float(want.norm())


def test_cross_offsets_past_32_bits():
    from turboadam_amd import linear_cross_entropy

    log("cross of 2.2e9 elements of x")
    g = _gen("long cross")
    m, k, v = 540001, 4096, 70
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_()
    w = (torch.randn(v, k, generator=g, device="cuda") / 64).bfloat16().requires_grad_()
    t = torch.randint(0, v, (m,), generator=g, device="cuda")
    t[5::7] = -100
    loss = linear_cross_entropy(x, w, t, reduction="none")
    dx, = torch.autograd.grad(loss, x, torch.ones_like(loss), retain_graph=True)
    for i in (0, 262000, 524288, m - 3000):
        part = x.detach()[i:i + 3000].clone().requires_grad_()
        want = linear_cross_entropy(part, w.detach(), t[i:i + 3000], reduction="none")
        assert float((loss.detach()[i:i + 3000] - want.detach()).abs().max()) < 2e-5, i
        d, = torch.autograd.grad(want, part, torch.ones_like(want))
        assert float((dx[i:i + 3000].double() - d.double()).norm()) <= 2 * UNIT["bf16"] * float(d.double().norm()), i
    del dx, x
    log("cross of 2.3e9 elements of w")
    k, v = 18000, 128256
    x, w = _whole(g, 40, k), _whole(g, v, k)
    x = (x / 64).requires_grad_()
    w.requires_grad_()
    t = torch.randint(0, v, (40,), generator=g, device="cuda")
    loss = linear_cross_entropy(x, w, t, reduction="sum")
    dw, = torch.autograd.grad(loss, w)
    z = torch.cat([x.detach().double() @ p.double().t() for p in w.detach().split(16384)], 1)
    assert abs(float(loss.detach()) - float(F.cross_entropy(z, t, reduction="sum"))) < 1e-4 * float(loss.detach())
    p = z.softmax(1)
    p[torch.arange(40, device="cuda"), t] -= 1
    for i in range(0, v, 16384):
        want = p[:, i:i + 16384].t() @ x.detach().double()
        assert float((dw[i:i + 16384].double() - want).norm()) <= 2 * UNIT["bf16"] * float(want.norm()) + 1e-6, i


def test_rotary_offsets_past_32_bits():
    from turboadam_amd import rotary, rotary_frequencies

    g = _gen("long rotary")
    t, h, d = 540001, 16, 256
    log(f"rotary of {t}x{h}x{d}")
    q = torch.randn(t, h, d, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_()
    w = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).bfloat16()
    f, p = rotary_frequencies(d, device="cuda"), torch.arange(t, device="cuda")
    y = rotary(q, None, p, f, q_weight=w)
    dq, = torch.autograd.grad(y, q, y)
    for i in (0, 262000, 524288, t - 3000):  # the same rows by themselves, whose results other tests pin
        part = q.detach()[i:i + 3000].clone().requires_grad_()
        z = rotary(part, None, p[i:i + 3000], f, q_weight=w)
        assert torch.equal(y[i:i + 3000], z), i
        assert torch.equal(dq[i:i + 3000], torch.autograd.grad(z, part, z)[0]), i


@pytest.mark.parametrize("tokens", [(1 << 20) - 8, (1 << 20) + 8])
def test_rotary_heads_far_apart(tokens):
    """2 heads of 128, one whole behind the other: of 8 heads a wave's offsets would end before and past 2^31 bytes."""
    from turboadam_amd import rotary, rotary_frequencies

    g = _gen("far heads", tokens)
    log(f"rotary of 2 heads {tokens} x 128 elements apart")
    q = torch.randn(2, tokens, 128, generator=g, device="cuda", dtype=torch.bfloat16).transpose(0, 1).requires_grad_()
    w = (1 + 0.1 * torch.randn(128, generator=g, device="cuda")).bfloat16()
    f, p = rotary_frequencies(128, device="cuda"), torch.arange(tokens, device="cuda")
    for weight in (None, w):
        y = rotary(q, None, p, f, q_weight=weight)
        dq, = torch.autograd.grad(y, q, y.detach())
        for i in (0, 500000, tokens - 2000):  # the same rows by themselves, whose results other tests pin
            part = q.detach()[i:i + 2000].contiguous().requires_grad_()
            z = rotary(part, None, p[i:i + 2000], f, q_weight=weight)
            assert torch.equal(y[i:i + 2000], z), i
            assert torch.equal(dq[i:i + 2000], torch.autograd.grad(z, part, z)[0]), i


# ------------------------------------------------------------ the example
def _example():
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_decoder.py")
    spec = importlib.util.spec_from_file_location("train_decoder", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_example_runs():
    mod = _example()
    for dtype in ("bf16", "f32"):
        losses = mod.train(dim=128, layers=1, words=300, sequences=4, length=33, steps=3, dtype=dtype, log=log)
        assert len(losses) == 3 and all(math.isfinite(v) for v in losses)


def test_example_gradients():
    """The example's decoder in fp32: its loss and every gradient against the same network in 64 bits and plain torch.
    Its sums have up to 512 terms of fp32 (2^-14 of their parts at most), its depth is a dozen of them: 1e-3 of a
    gradient's norm is far above what they add up to, and far below a wrong term."""
    mod = _example()
    g = torch.Generator(device="cuda").manual_seed(1)
    model = mod.Decoder(128, 2, 200, torch.float32, g)
    text = mod.make_text(g, torch.randint(0, 200, (200, 4), generator=g, device="cuda"), 3, 41)
    names, params = zip(*model.named_parameters())
    loss = model.loss(text, prompt=8)
    grads = torch.autograd.grad(loss, params)
    P = {n: p.detach().double().requires_grad_() for n, p in zip(names, params)}
    head, f = mod.HEAD, model.frequencies

    def turn(x, w):
        x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        return _turned(x, (torch.arange(40, device="cuda").double()[:, None] * f)[:, None, :], head, False, 1.0)[0]

    x = P["embedding"][text[:, :-1]]
    for i, layer in enumerate(model.layers):
        at = {n: P[f"layers.{i}.{n}"] for n, _ in layer.named_parameters()}
        n = F.layer_norm(x, (128,), at["norm1"])
        q, k, v = (n @ at["qkv"].t()).unflatten(-1, (-1, head)).split((layer.heads, layer.kv_heads, layer.kv_heads), -2)
        q, k = turn(q, at["q_norm"]), turn(k, at["k_norm"])
        groups = layer.heads // layer.kv_heads
        q, k, v = q.transpose(1, 2), k.repeat_interleave(groups, 2).transpose(1, 2), v.repeat_interleave(groups, 2).transpose(1, 2)
        s = (q @ k.mT * head ** -0.5).masked_fill(torch.ones(40, 40, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        x = x + (s.softmax(-1) @ v).transpose(1, 2).flatten(2) @ at["out"].t()
        n = F.layer_norm(x, (128,), at["norm2"])
        x = x + (F.silu(n @ at["gate"].t()) * (n @ at["up"].t())) @ at["down"].t()
    target = text[:, 1:].clone()
    target[:, :8] = -100
    want = F.cross_entropy((F.layer_norm(x, (128,), P["norm"]) @ P["head"].t()).flatten(0, 1), target.flatten())
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5 * float(want.detach())
    for n, got, ref in zip(names, grads, torch.autograd.grad(want, list(P.values()))):
        assert float((got.double() - ref).norm()) <= 1e-3 * float(ref.norm()), n
