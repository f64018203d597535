"""GPU: orthogonalize and Muon against Newton-Schulz products in 64 bits.

Bounds (fixed before the first run), in the 2-norm relative to the result.  bf16:
the result's rounding, 2^-8, and for each of 5 steps the roundings of x, q and p to
11 bits, each about 2^-12 in the norm and amplified no more than the step's own growth:
15 * 2^-12 in all, 2^-8 + 15 * 2^-12 = 7.6e-3.  fp32 and fp16: factors of 22 bits and
fp32 sums of up to a few thousand terms (random roundings: about sqrt(n) 2^-24),
15 * (2^-22 + 2^-19) = 3.3e-5 beside the result's rounding (2^-24, 2^-11)."""

import copy
import math
import zlib

import pytest
import torch

from tests.helpers import log

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BOUND = {"f32": 2.0 ** -24 + 15 * (2.0 ** -22 + 2.0 ** -19), "bf16": 2.0 ** -8 + 15 * 2.0 ** -12,
         "f16": 2.0 ** -11 + 15 * (2.0 ** -22 + 2.0 ** -19)}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _reference(u, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = u.double() / max(float(u.double().norm()), eps)
    for _ in range(steps):
        if x.shape[0] <= x.shape[1]:
            q = x @ x.t()
            x = a * x + (b * q + c * q @ q) @ x
        else:
            q = x.t() @ x
            x = a * x + x @ (b * q + c * q @ q)
    return x


def _off(got, want):
    norm = float(want.norm())
    return float((got.double() - want).norm()) / norm if norm else float(got.double().norm())


def _matrix(g, rows, cols, kind):
    x = torch.randn(rows, cols, generator=g, device="cuda")
    if kind == "strong":  # a few directions over noise
        x = x + torch.randn(rows, 4, generator=g, device="cuda") @ torch.randn(4, cols, generator=g, device="cuda")
    return x * 1e-3


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("batch,rows,cols", [(1, 1, 1), (2, 1, 300), (2, 300, 1), (3, 5, 70), (2, 70, 5), (4, 64, 64),
                                             (1, 96, 128), (2, 129, 257), (2, 300, 100), (70, 17, 23), (1, 500, 520),
                                             (1, 1300, 260)])
def test_orthogonalize(batch, rows, cols, dt):
    from turboadam_amd import orthogonalize

    g = _gen(batch, rows, cols)
    for kind in ("noise", "strong"):
        log(f"orthogonalize {batch}x{rows}x{cols} {dt} {kind}")
        x = torch.stack([_matrix(g, rows, cols, kind) for _ in range(batch)]).to(DTYPES[dt])
        out = orthogonalize(x)
        assert out.dtype == x.dtype and out.shape == x.shape
        for i in range(0, batch, 7):
            off = _off(out[i], _reference(x[i]))
            assert off <= BOUND[dt], (i, off)


@pytest.mark.parametrize("dt,rows,cols", [("bf16", 2100, 2300), ("bf16", 4600, 1100), ("f32", 1500, 1400)])
def test_orthogonalize_large(dt, rows, cols):
    from turboadam_amd import orthogonalize

    log(f"orthogonalize {rows}x{cols} {dt}")
    x = _matrix(_gen(rows, cols), rows, cols, "strong").to(DTYPES[dt])
    off = _off(orthogonalize(x), _reference(x))
    assert off <= BOUND[dt], off


@pytest.mark.parametrize("dt", list(DTYPES))
def test_orthogonalize_small_directions(dt):
    """Singular values over four decades: the products raise small directions hundreds of times, and their
    errors with them unless the iterate keeps more bits than its products' factors."""
    from turboadam_amd import orthogonalize

    log(f"orthogonalize small directions {dt}")
    n = 200
    u, _ = torch.linalg.qr(torch.randn(n, n, generator=_gen("u"), device="cuda").double())
    v, _ = torch.linalg.qr(torch.randn(320, n, generator=_gen("v"), device="cuda").double())
    x = ((u * torch.logspace(0, -4, n, device="cuda", dtype=torch.float64)) @ v.t()).to(DTYPES[dt])
    for y in (x, x.t().contiguous()):
        off = _off(orthogonalize(y), _reference(y))
        assert off <= BOUND[dt], off


def test_orthogonalize_result_is_near_orthogonal():
    from turboadam_amd import orthogonalize

    x = _matrix(_gen("singular"), 300, 500, "noise")
    s = torch.linalg.svdvals(orthogonalize(x).double())
    assert float(s.max()) < 1.3 and float(s.min()) > 0.5


def test_orthogonalize_zero_tiny_huge_and_bad_matrices():
    from turboadam_amd import orthogonalize

    log("orthogonalize zeros")
    for dt in DTYPES.values():
        assert bool((orthogonalize(torch.zeros(3, 40, 30, device="cuda", dtype=dt)) == 0).all())
    x = torch.randn(50, 70, generator=_gen("scale"), device="cuda")
    for scale in (1e-30, 1e-9, 1e15):
        log(f"orthogonalize scale {scale}")
        y = x * scale
        # squares below fp32's smallest numbers: such a norm is 0, and eps takes its place
        want = _reference(y) if scale > 1e-20 else torch.zeros_like(y, dtype=torch.float64)
        assert float((orthogonalize(y).double() - want).norm()) <= 1e-4 * max(1.0, float(want.norm()))
    log("orthogonalize: one matrix's NaN stays its own")
    b = torch.stack([x, x, x])
    b[1, 3, 4] = math.nan
    out = orthogonalize(b)
    assert bool(out[1].isnan().all()) and torch.equal(out[0], out[2]) and bool(out[0].isfinite().all())
    assert torch.equal(out[0], orthogonalize(x))


def test_orthogonalize_other_coefficients_and_views():
    from turboadam_amd import orthogonalize

    x = _matrix(_gen("views"), 90, 120, "noise")
    log("orthogonalize with other coefficients")
    for steps, co in ((1, (1.0, 0.0, 0.0)), (1, (0.0, 1.0, 0.0)), (1, (0.0, 0.0, 1.0)), (12, (1.5, -0.5, 0.0)),
                      (8, (2.0, -1.5, 0.5))):
        off = _off(orthogonalize(x, steps=steps, coefficients=co), _reference(x, steps, co))
        assert off <= BOUND["f32"], (steps, co, off)
    log("orthogonalize of views")
    want = orthogonalize(x)
    wide = torch.zeros(90, 131, device="cuda")
    wide[:, 5:125] = x
    assert torch.equal(orthogonalize(wide[:, 5:125]), want)
    odd = torch.zeros(90 * 120 + 1, device="cuda")
    odd[1:] = x.reshape(-1)
    assert torch.equal(orthogonalize(odd[1:].view(90, 120)), want)
    assert orthogonalize(torch.zeros(0, 4, 5, device="cuda")).shape == (0, 4, 5)


# -------------------------------------------------------------------- Muon
def _muon_reference(p, g, m, kw):
    lr, wd, mu = kw["lr"], kw["weight_decay"], kw["momentum"]
    m = mu * m.double() + (1 - mu) * g.double()
    u = (1 - mu) * g.double() + mu * m if kw["nesterov"] else m
    rows, cols = p.shape
    adjust = (math.sqrt(max(1.0, rows / cols)) if kw["adjust_lr"] == "original" else 0.2 * math.sqrt(max(rows, cols)))
    return (1 - lr * wd) * p.double() - lr * adjust * _reference(u), m, lr * adjust


SHAPES = [(128, 96), (33, 257), (300, 40), (64, 64), (1, 9), (520, 260)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("nesterov,adjust", [(True, "original"), (False, "match_rms_adamw")])
def test_muon_steps(dt, nesterov, adjust):
    from turboadam_amd import Muon

    kw = dict(lr=0.02, weight_decay=0.1, momentum=0.9, nesterov=nesterov, adjust_lr=adjust)
    g = _gen(dt, nesterov)
    params = [torch.nn.Parameter((0.1 * torch.randn(s, generator=g, device="cuda")).to(DTYPES[dt])) for s in SHAPES]
    opt = Muon(params, **kw)
    unit = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dt]
    for step in range(3):
        before = [(p.detach().clone(), opt.state[p]["momentum_buffer"].clone() if step else torch.zeros_like(p.float()))
                  for p in params]
        for p in params:
            p.grad = _matrix(g, *p.shape, "strong").to(DTYPES[dt])
        if step == 1:  # a gradient that is missing: nothing of its parameter moves
            params[2].grad = None
        opt.step()
        log(f"muon {dt} step {step + 1}")
        for i, (p, (p0, m0)) in enumerate(zip(params, before)):
            if p.grad is None:
                assert torch.equal(p, p0) and torch.equal(opt.state[p]["momentum_buffer"], m0)
                continue
            want, m, rate = _muon_reference(p0, p.grad, m0, kw)
            got = opt.state[p]["momentum_buffer"]
            assert got.dtype == torch.float32
            assert bool(((got.double() - m).abs() <= 2.0 ** -22 * (m.abs() + m0.double().abs())).all())
            # the direction's bound times the rate, and the parameter's own rounding
            size = math.sqrt(min(p.shape))
            bound = BOUND[dt] * rate * 1.2 * size + (unit + 2.0 ** -22) * float(want.norm())
            assert float((p.double() - want).norm()) <= bound, (i, step)


def test_muon_groups_types_and_odd_addresses_in_one_step():
    from turboadam_amd import Muon

    g = _gen("groups")
    flat = torch.randn(20000, generator=g, device="cuda").bfloat16()
    odd = [torch.nn.Parameter(flat[1:1 + 60 * 50].view(60, 50)), torch.nn.Parameter(flat[3001:3001 + 77 * 31].view(77, 31))]
    f32 = [torch.nn.Parameter(torch.randn(40, 90, generator=g, device="cuda"))]
    opt = Muon([{"params": odd}, {"params": f32, "lr": 0.1, "ns_steps": 3}], lr=0.01, weight_decay=0.0, momentum=0.5)
    single = []
    for p, lr, steps in ((odd[0], 0.01, 5), (odd[1], 0.01, 5), (f32[0], 0.1, 3)):
        p.grad = _matrix(g, *p.shape, "noise").to(p.dtype)
        q = torch.nn.Parameter(p.detach().clone())
        q.grad = p.grad.clone()
        Muon([q], lr=lr, weight_decay=0.0, momentum=0.5, ns_steps=steps).step()
        single.append(q)
    rest = flat.clone()
    opt.step()
    for p, q in zip([*odd, *f32], single):
        assert torch.equal(p, q)
    kept = torch.ones_like(flat, dtype=torch.bool)
    for p in odd:
        kept[p.storage_offset():p.storage_offset() + p.numel()] = False
    assert torch.equal(flat[kept], rest[kept])


def test_muon_step_is_seen_by_graphs_that_kept_the_parameter():
    from turboadam_amd import Muon, linear

    g = _gen("versions")
    w, other = (torch.nn.Parameter(torch.randn(30, 20, generator=g, device="cuda")) for _ in range(2))
    x = torch.randn(8, 20, generator=g, device="cuda", requires_grad=True)
    opt = Muon([w, other])
    w.grad = torch.randn(30, 20, generator=g, device="cuda")
    y = linear(x, w)
    before = [t._version for t in (w, other)]
    opt.step()
    assert w._version > before[0] and other._version == before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    m = opt.state[w]["momentum_buffer"]
    at = m._version
    opt.step()
    assert m._version > at
    linear(x, w).sum().backward()


def test_muon_state_dict_keeps_fp32_momentum():
    from turboadam_amd import Muon

    g = _gen("state")
    start = torch.randn(50, 30, generator=g, device="cuda").bfloat16()
    grads = [torch.randn(50, 30, generator=g, device="cuda").bfloat16() for _ in range(4)]
    a = torch.nn.Parameter(start.clone())
    oa = Muon([a], lr=0.02)
    for gr in grads[:2]:
        a.grad = gr
        oa.step()
    b = torch.nn.Parameter(a.detach().clone())
    ob = Muon([b], lr=0.5)
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    assert ob.param_groups[0]["lr"] == 0.02
    m = ob.state[b]["momentum_buffer"]
    assert m.dtype == torch.float32 and torch.equal(m, oa.state[a]["momentum_buffer"])
    assert m.data_ptr() != oa.state[a]["momentum_buffer"].data_ptr()
    for gr in grads[2:]:
        a.grad, b.grad = gr, gr
        oa.step()
        ob.step()
    assert torch.equal(a, b)


def test_muon_step_in_a_captured_graph():
    from turboadam_amd import Muon

    g = _gen("graph")
    grads = [torch.randn(s, generator=g, device="cuda") for s in ((200, 120), (64, 300))]
    kept = [torch.randn(s, generator=g, device="cuda") for s in ((200, 120), (64, 300))]
    pa = [torch.nn.Parameter(k.clone()) for k in kept]
    pb = [torch.nn.Parameter(k.clone()) for k in kept]
    oa, ob = Muon(pa, lr=0.02), Muon(pb, lr=0.02)
    for p, q, gr in zip(pa, pb, grads):
        p.grad, q.grad = gr, gr.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        oa.step()
    torch.cuda.current_stream().wait_stream(side)
    ob.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    for i in range(4):
        for p, q in zip(pa, pb):
            p.grad.normal_(generator=g)
            q.grad.copy_(p.grad)
        graph.replay()
        ob.step()
        torch.cuda.synchronize()
        for p, q in zip(pa, pb):
            assert torch.equal(p, q), f"replay {i}"


def test_muon_and_orthogonalize_refuse_what_they_cannot_take():
    from turboadam_amd import Muon, orthogonalize

    x = torch.ones(4, 6, device="cuda")
    for args, kw, error, text in [
        ((x.cpu(),), {}, RuntimeError, "MI355X"), ((x.double(),), {}, ValueError, "float32"),
        ((x[0],), {}, ValueError, "rows, cols"), ((x,), {"steps": 0}, ValueError, "steps"),
        ((x,), {"steps": 65}, ValueError, "steps"), ((x,), {"eps": 0.0}, ValueError, "eps"),
        ((x,), {"coefficients": (1.0, 2.0)}, ValueError, "three"),
        ((x,), {"coefficients": (1.0, 2.0, math.nan)}, ValueError, "three"),
        ((torch.ones(1, 65537, device="cuda"),), {}, ValueError, "65536"),
    ]:
        with pytest.raises(error, match=text):
            orthogonalize(*args, **kw)
    p = torch.nn.Parameter(x.clone())
    for kw, text in [({"lr": -1.0}, "lr"), ({"momentum": 1.0}, "momentum"), ({"weight_decay": -0.1}, "weight_decay"),
                     ({"adjust_lr": "none"}, "adjust_lr"), ({"ns_steps": 0}, "steps")]:
        with pytest.raises(ValueError, match=text):
            Muon([p], **kw)
    with pytest.raises(ValueError, match="2-D"):
        Muon([torch.nn.Parameter(x[0].clone())])
    opt = Muon([p])
    p.grad = torch.ones_like(p)
    opt.step()
    before = p.detach().clone()
    opt.state[p]["momentum_buffer"] = torch.zeros(4, 6, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="momentum_buffer"):
        opt.step()
    assert torch.equal(p, before)
    q = torch.nn.Parameter(torch.ones(6, 4, device="cuda").t())
    q.grad = torch.ones(4, 6, device="cuda")
    with pytest.raises(RuntimeError, match="contiguous"):
        Muon([q]).step()


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows,cols", [(30, 40), (40, 30), (150, 200), (200, 150)])
def test_orthogonalize_large_coefficients(rows, cols, dt):
    """Coefficients whose polynomial passes 16 (fp16's numbers at 2^-12): its sums fit, and a zero matrix stays one."""
    from turboadam_amd import orthogonalize

    x = _matrix(_gen("large coefficients", rows, cols), rows, cols, "noise").to(DTYPES[dt])
    assert bool(orthogonalize(torch.ones(1, 1, device="cuda"), steps=1, coefficients=(63.9, 63.9, 63.9)).isfinite())
    for co in ((16.0, 0.0, 0.0), (20.0, -3.0, 1.0), (63.9, -60.0, 1.0), (0.0, 63.9, 0.0), (0.0, 0.0, 63.9),
               (-63.9, 63.9, 63.9), (15.0, 0.0, 0.0)):
        log(f"orthogonalize {rows}x{cols} {dt} {co}")
        for steps in (1, 5):
            assert bool((orthogonalize(torch.zeros_like(x), steps=steps, coefficients=co) == 0).all())
        off = _off(orthogonalize(x, steps=1, coefficients=co), _reference(x, 1, co))
        assert off <= BOUND[dt], (co, off)


@pytest.mark.parametrize("rows,cols", [(20, 30), (150, 200), (200, 150)])
def test_orthogonalize_any_norm_and_eps(rows, cols):
    """|u| and eps anywhere in fp32's range: squares are summed in 64 bits, and no factor of the quotient leaves it."""
    from turboadam_amd import orthogonalize

    x = torch.randn(rows, cols, generator=_gen("norms", rows, cols), device="cuda")
    zero = torch.zeros_like(x)
    for scale, eps in ((1e-22, 1e-30), (1e-30, 1e-38), (1e-36, 1e-44), (1e-20, 1e-7), (1e-30, 1e-28), (1e18, 1e-7),
                       (1e25, 1e-7), (1e37, 1e-7), (1e36, 1e30), (1e-3, 1e38)):
        log(f"orthogonalize {rows}x{cols} scale {scale} eps {eps}")
        y = x * scale
        want = _reference(y, eps=eps)
        # denormal numbers of u are right to their last bit, 2^-149
        bound = BOUND["f32"] * float(want.norm()) + 2.0 ** -149 / max(scale, eps) * 500 * want.norm()
        # below 2^-24 / 2^12 of 1 the factors' low parts have no bits: such a result is near 0 and no more
        assert float((orthogonalize(y, eps=eps).double() - want).norm()) <= float(bound) + 1e-6, (scale, eps)
        assert bool((orthogonalize(zero, eps=eps) == 0).all())
    for dt in DTYPES.values():
        assert bool((orthogonalize(zero.to(dt), eps=1e-38) == 0).all())


@pytest.mark.parametrize("rows,cols", [(20, 30), (150, 200)])
def test_muon_of_a_huge_gradient(rows, cols):
    from turboadam_amd import Muon

    kw = dict(lr=0.02, weight_decay=0.1, momentum=0.9, nesterov=True, adjust_lr="original")
    g = _gen("huge", rows)
    p = torch.nn.Parameter(torch.randn(rows, cols, generator=g, device="cuda"))
    p0, m0 = p.detach().clone(), torch.zeros(rows, cols, device="cuda")
    p.grad = 1e30 * torch.randn(rows, cols, generator=g, device="cuda")
    Muon([p], **kw).step()
    want, _, rate = _muon_reference(p0, p.grad, m0, kw)
    bound = BOUND["f32"] * rate * 1.2 * math.sqrt(rows) + 2.0 ** -21 * float(want.norm())
    assert float((p.detach().double() - want).norm()) <= bound


# lists that reach each tile (of q, p and x) with remainders, wide and tall
TILES = [([(1507, 1601), (1603, 1500), (1500, 1600)], (128, 128, 128)), ([(5001, 4201)], (128, 128, 256)),
         ([(4201, 5003)], (128, 128, 256)), ([(1281, 1922)] * 5 + [(1923, 1282)] * 5, (256, 256, 256)),
         ([(1030, 1033)] * 8 + [(1035, 1031)] * 7, (256, 256, 128))]


def _tiles(shapes, dt):
    import ctypes

    from turboadam_amd import _lib

    m, out = (_lib.TamMatrix * len(shapes))(), (ctypes.c_uint32 * 4)()
    for d, (rows, cols) in zip(m, shapes):
        d.out = d.grad = 0x10000
        d.rows, d.cols, d.eps, d.dtype = rows, cols, 1e-7, _lib.DTYPES[DTYPES[dt]]
    assert _lib.load().tam_orthogonalize_tiles(ctypes.addressof(m), len(shapes), out) == 0
    return out[0], out[2], out[3]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("shapes,tiles", TILES)
def test_muon_in_every_large_tile(shapes, tiles, dt):
    from turboadam_amd import Muon

    log(f"muon {len(shapes)} matrices like {shapes[0]} {dt}, tiles of {tiles}")
    assert _tiles(shapes, dt) == tiles
    kw = dict(lr=0.5, weight_decay=0.1, momentum=0.9, nesterov=True, adjust_lr="original")
    g = _gen("tiles", len(shapes), dt)
    params = [torch.nn.Parameter((0.01 * torch.randn(s, generator=g, device="cuda")).to(DTYPES[dt])) for s in shapes]
    before = [p.detach().clone() for p in params]
    for p in params:
        p.grad = _matrix(g, *p.shape, "strong").to(DTYPES[dt])
    Muon(params, **kw).step()
    unit = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dt]
    for i, (p, p0) in enumerate(zip(params, before)):
        want, _, rate = _muon_reference(p0, p.grad, torch.zeros_like(p0, dtype=torch.float32), kw)
        bound = BOUND[dt] * rate * 1.2 * math.sqrt(min(p.shape)) + (unit + 2.0 ** -22) * float(want.norm())
        assert float((p.detach().double() - want).norm()) <= bound, i


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("batch,rows,cols,tiles", [(3, 1507, 1601, (128, 128, 128)), (1, 5001, 4201, (128, 128, 256)),
                                                   (10, 1281, 1922, (256, 256, 256)), (10, 1922, 1281, (256, 256, 256)),
                                                   (15, 1030, 1033, (256, 256, 128))])
def test_orthogonalize_in_every_large_tile(batch, rows, cols, tiles, dt):
    from turboadam_amd import orthogonalize

    log(f"orthogonalize {batch}x{rows}x{cols} {dt}, tiles of {tiles}")
    assert _tiles([(rows, cols)] * batch, dt) == tiles
    g = _gen("tiles", batch, rows, cols)
    x = torch.stack([_matrix(g, rows, cols, "strong") for _ in range(batch)]).to(DTYPES[dt])
    out = orthogonalize(x)
    for i in {0, batch // 2, batch - 1}:
        want = _reference(x[i])
        off = _off(out[i], want)
        assert off <= BOUND[dt], (i, off)
        # no row or column is left far behind the others (the bound above is over the whole matrix)
        for dim in (0, 1):
            far = (out[i].double() - want).norm(dim=dim) / want.norm(dim=dim)
            assert float(far.max()) <= 8 * BOUND[dt], (i, dim, int(far.argmax()))


@pytest.mark.parametrize("rows,cols", [(65536, 33001), (33001, 65535)])
def test_orthogonalize_offsets_past_32_bits(rows, cols):
    """2.2e9 elements: one step of a polynomial that leaves the normalised matrix, and one that scales each of its rows
    (columns, where it is tall) by q's diagonal, q being diagonal here."""
    from turboadam_amd import orthogonalize

    log(f"orthogonalize {rows}x{cols}")
    x = torch.randn(rows, cols, generator=_gen("long", rows), device="cuda", dtype=torch.bfloat16)
    out = orthogonalize(x, steps=1, coefficients=(1.0, 0.0, 0.0))
    squares = sum(float(p.double().square().sum()) for p in x.split(4096))
    for p, o in zip(x.split(4096), out.split(4096)):
        want = p.double() / math.sqrt(squares)
        assert float((o.double() - want).norm()) <= BOUND["bf16"] * float(want.norm())
    # one element to each of the last 40 lines of the shorter side: q = diag(e^2) / |e|^2, x' = (1 + 40 q) x
    x.zero_()
    at = torch.arange(min(rows, cols) - 40, min(rows, cols), device="cuda")
    other = (at * 1601) % max(rows, cols)
    e = 1.0 + (at % 13).float()
    i, j = (at, other) if rows <= cols else (other, at)
    x[i, j] = e.to(x.dtype)
    out = orthogonalize(x, steps=1, coefficients=(1.0, 40.0, 0.0))
    n = e.double() / e.double().norm()
    want = (1 + 40 * n * n) * n
    assert float((out[i, j].double() - want).norm()) <= BOUND["bf16"] * float(want.norm())
    assert int(out.count_nonzero()) == len(at)


def test_orthogonalize_refuses_to_drop_a_gradient():
    from turboadam_amd import orthogonalize

    x = _matrix(_gen("gradient"), 20, 30, "noise")
    want = orthogonalize(x)
    leaf = x.clone().requires_grad_()
    for g in (leaf, leaf * 1.0):
        with pytest.raises(RuntimeError, match="no backward pass"):
            orthogonalize(g)
        assert torch.equal(orthogonalize(g.detach()), want)
        with torch.no_grad():
            assert torch.equal(orthogonalize(g), want)


def test_example_trains_a_block():
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_block.py")
    spec = importlib.util.spec_from_file_location("train_block", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    for dtype in ("bf16", "f32"):
        losses = mod.train(dim=128, tokens=512, steps=30, dtype=dtype, log=log)
        assert all(math.isfinite(v) for v in losses) and losses[-1] < 0.5 * losses[0], losses
