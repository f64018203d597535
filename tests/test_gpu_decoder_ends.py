"""GPU: gated_linear, linear_cross_entropy and rotary at the ends of their ranges: infinities and NaN beside what
does not touch them, an eps of 0, values that a type cannot hold, losses of large logits, gradients of 2^127 and more.

Bounds (fixed before the first run) are derived beside each test."""

import math

import pytest
import torch

from tests.helpers import log
from tests.test_gpu_decoder import DTYPES, UNIT, _check_rotary, _gen, _rotary_case, _within

pytestmark = pytest.mark.gpu

BITS = {torch.float32: torch.int32, torch.bfloat16: torch.int16, torch.float16: torch.int16}


def _same_bits(a, b):
    """Bit for bit, -0 from 0 too, but any NaN as any other."""
    bits = BITS[a.dtype]
    return a.shape == b.shape and bool(((a.contiguous().view(bits) == b.contiguous().view(bits)) | (a.isnan() & b.isnan())).all())


# ------------------------------------------------------------------ rotary
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,pairs", [(40, 8), (33, 7), (64, 16), (24, 0), (300, 100)])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_rotary_what_does_not_turn_stays_as_it_is(d, pairs, interleaved, dt):
    """Infinities, NaN and -0 behind the rotated part of heads without a norm: forward and backward they come out as they
    went in, and no other element changes a bit."""
    from turboadam_amd import rotary

    q, k, p, f, _, dq, dk = _rotary_case(2, 9, 3, 2, d, pairs, dt, False, 3)
    log(f"rotary rest of {d}, {pairs} pairs, {dt} interleaved={interleaved}")

    def both(q, k, dq, dk):
        leaves = [v.detach().requires_grad_() for v in (q, k)]
        out = rotary(*leaves, p, f, interleaved=interleaved)
        return [v.detach() for v in out] + list(torch.autograd.grad(out, leaves, (dq, dk)))

    want = both(q, k, dq, dk)
    special = (math.inf, -math.inf, math.nan, -0.0)
    marked = []
    for v in (q, k, dq, dk):
        v = v.clone()
        g = _gen("where", d, pairs, len(marked))
        where = torch.rand(v.shape, generator=g, device="cuda") < 0.2
        where[..., :2 * pairs] = False
        v[where] = torch.tensor(special, device="cuda").to(v.dtype)[torch.arange(int(where.sum()), device="cuda") % 4]
        marked.append(v)
    for got, ref, v in zip(both(*marked), want, marked):
        assert _same_bits(got[..., 2 * pairs:], v[..., 2 * pairs:])
        assert _same_bits(got[..., :2 * pairs], ref[..., :2 * pairs])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_rotary_an_infinity_in_the_rest_of_a_normed_head(interleaved, dt):
    """The norm divides by an infinite root: by the formula it is NaN itself and every other element of its head 0."""
    from turboadam_amd import rotary

    q, k, p, f, w, _, _ = _rotary_case(1, 9, 3, 2, 40, 8, dt, True, 3)
    want = rotary(q, k, p, f, interleaved=interleaved, q_weight=w[0], k_weight=w[1])
    q = q.clone()
    q[0, 4, 1, 21] = math.inf
    log(f"rotary of an infinity beside a norm {dt} interleaved={interleaved}")
    got = rotary(q, k, p, f, interleaved=interleaved, q_weight=w[0], k_weight=w[1])
    head = got[0][0, 4, 1]
    assert bool(head[21].isnan()) and bool((head[torch.arange(40, device="cuda") != 21] == 0).all())
    got[0][0, 4, 1] = want[0][0, 4, 1]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("b,t,hq,hk,d,pairs", [(1, 5, 32, 4, 128, 64), (2, 7, 7, 3, 84, 42), (1, 33, 2, 1, 64, 16), (3, 3, 1, 5, 40, 0)])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_rotary_norm_of_an_eps_of_zero(b, t, hq, hk, d, pairs, dt):
    """Heads that are no multiple of a wave's rows, and tokens that leave a wave's last ones empty: what has no row adds
    nothing to the weights' gradients, though its own norm would divide by 0."""
    q, k, p, f, w, dq, dk = _rotary_case(b, t, hq, hk, d, pairs, dt, True, 5)
    for interleaved in (False, True):
        log(f"rotary eps 0, {b}x{t} {hq}/{hk} heads of {d} {dt} interleaved={interleaved}")
        _check_rotary(q, k, p, f, dt, interleaved, 1.0, w[0], w[1], eps=0.0, dq=dq, dk=dk)
        _check_rotary(q, k, p, f, dt, interleaved, 1.0, w[0], None, eps=0.0, dq=dq, dk=dk)


def test_rotary_eps_is_zero_or_a_normal_number():
    """A head of zeros is divided by sqrt(eps): an eps that float32 has not, or that the hardware's root takes for 0, would
    make it NaN."""
    from turboadam_amd import rotary

    log("rotary eps at its ends")
    f, p = torch.ones(4, dtype=torch.float64, device="cuda"), torch.arange(4, device="cuda")
    for dt in DTYPES.values():
        q, w = torch.zeros(4, 2, 8, device="cuda", dtype=dt), torch.ones(8, device="cuda", dtype=dt)
        for eps in (1e-50, 2.0 ** -127, 1e39, math.inf, math.nan):
            with pytest.raises(ValueError, match="eps"):
                rotary(q, None, p, f, q_weight=w, eps=eps)
        assert bool((rotary(q, None, p, f, q_weight=w, eps=2.0 ** -126) == 0).all())


# ------------------------------------------------------------ gated linear
@pytest.mark.parametrize("in_out", [False, True])
@pytest.mark.parametrize("rows", [20, 100])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_gated_of_products_that_the_type_cannot_hold(rows, dt, in_out):
    """g = a G and u = b U, of which fp16 holds neither in some rows (g of -2.6e5 or 2.6e5, u of 1e5 either sign) but h and
    every gradient in all of them.  The bounds are those of the other gated tests."""
    from tests.test_gpu_decoder import _check_gated

    g = _gen("past the range", rows)
    a = torch.tensor([-512.0, -300.0, 512.0, 16.0, -0.02], device="cuda")[torch.arange(rows, device="cuda") % 5]
    b = torch.tensor([0.008, 1.0, 2.0 ** -12, 0.008, 200.0], device="cuda")[torch.arange(rows, device="cuda") % 5]
    x = torch.zeros(rows, 8, device="cuda")
    x[:, 0], x[:, 1] = a, b
    gate, up = torch.zeros(2, 40, 8, device="cuda").unbind(0)
    gate[:, 0] = torch.rand(40, generator=g, device="cuda") * 500 + 12
    up[:, 1] = (torch.rand(40, generator=g, device="cuda") - 0.5) * 1000
    x, gate, up = [v.to(DTYPES[dt]) for v in (x, gate, up)]
    if in_out:
        gate, up = [v.t().contiguous().t() for v in (gate, up)]
    dh = (torch.randn(rows, 40, generator=g, device="cuda") * 2.0 ** -15).to(DTYPES[dt])
    for act in ("silu", "gelu_tanh", "gelu", "relu"):
        log(f"gated past the range {rows} {dt} {act} in_out={in_out}")
        _check_gated(x, gate, up, dh, dt, act)


# --------------------------------------------- projection and cross entropy
def _exact_case(rows, inputs, words, dt, scale):
    """One column of x and w that is not zero: the logits are products of two numbers of the type, exact in fp32, so that
    the loss alone is measured."""
    g = _gen("exact", rows, words, scale)
    x, w = torch.zeros(rows, inputs, device="cuda"), torch.zeros(words, inputs, device="cuda")
    x[:, inputs // 2] = (1 + torch.rand(rows, generator=g, device="cuda")) * scale
    w[:, inputs // 2] = 2 - torch.rand(words, generator=g, device="cuda") * 2.0 ** torch.randint(
        -7, 3, (words,), generator=g, device="cuda")
    few = torch.float16 if dt == "f16" else torch.bfloat16  # digits, in fp32 too
    return [v.to(few).to(DTYPES[dt]) for v in (x, w)] + [torch.randint(0, words, (rows,), generator=g, device="cuda")]


@pytest.mark.parametrize("scale", [1.0, 300.0, 9000.0])
@pytest.mark.parametrize("rows,inputs,words", [(1, 9, 1000), (20, 64, 30011), (50, 24, 60), (40, 8, 10), (300, 40, 2777),
                                               (700, 264, 5001), (4096, 264, 9973)])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_cross_loss_of_exact_logits_of_any_size(rows, inputs, words, dt, scale):
    """Off by: a term's 2^x and its argument's rounding, 2^-23 (1 + |z - top|) of it, whose mean over the softmax is taken
    here; fp32 sums, at most 16 + 4 + 8 terms in a part and parts / 16 + 26 of them one after another, 2^-24 a step, two
    steps to a part (a factor and a sum); the difference to the target and the logarithm, 2^-23 of either."""
    from turboadam_amd import linear_cross_entropy

    x, w, t = _exact_case(rows, inputs, words, dt, scale)
    log(f"cross of exact logits {rows}x{inputs}x{words} {dt} scale {scale}")
    z = x.double() @ w.double().t()
    assert torch.equal(z, (x.float() @ w.float().t()).double())  # exact
    top, hit = z.amax(1), z.gather(1, t[:, None])[:, 0]
    away = ((z - top[:, None]).exp() * (top[:, None] - z)).sum(1) / (z - top[:, None]).exp().sum(1)
    want = z.logsumexp(1) - hit
    log_sum = z.logsumexp(1) - top
    bound = 2.0 ** -23 * (1 + away) + 2.0 ** -24 * (28 + 2 * (words / 256 + 26)) + 2.0 ** -23 * ((top - hit) + log_sum) + 2.0 ** -23 * want
    _within(linear_cross_entropy(x, w, t, reduction="none"), want, bound, "loss")


@pytest.mark.parametrize("rows,words", [(5, 1000), (60, 1000), (60, 40)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_cross_of_logits_near_the_end_of_float32(rows, words, dt):
    """Logits of up to 1.5 * 2^127 either side of 0: far apart, so that a loss is the difference of two of them."""
    from turboadam_amd import linear_cross_entropy

    log(f"cross of the largest logits {rows} {words} {dt}")
    x, w = torch.zeros(rows, 16, device="cuda"), torch.zeros(words, 16, device="cuda")
    x[:, 3] = 2.0 ** 64
    x[1::2, 3] = -(2.0 ** 64)
    w[:, 3] = torch.arange(words, device="cuda") % 5 * 2.0 ** 60
    w[17, 3], w[23, 3] = 1.5 * 2.0 ** 63, -1.25 * 2.0 ** 63
    x, w = x.to(DTYPES[dt]).requires_grad_(), w.to(DTYPES[dt]).requires_grad_()
    t = torch.arange(rows, device="cuda") % words
    t[:4] = torch.tensor([17, 23, 2, 7], device="cuda")
    odd = torch.arange(rows, device="cuda") % 2
    t[(t == 17) & (odd == 1)] = t[(t == 23) & (odd == 0)] = 3  # whose losses float32 could not hold
    z = x.detach().double() @ w.detach().double().t()
    want = z.amax(1) - z.gather(1, t[:, None])[:, 0]
    loss = linear_cross_entropy(x, w, t, reduction="none")
    _within(loss, want, 2.0 ** -23 * want, "loss")
    dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    p = (z == z.amax(1, keepdim=True)).double()
    p.scatter_add_(1, t[:, None], torch.full_like(want, -1.0)[:, None])
    ref = p @ w.detach().double()  # two terms a row
    _within(dx, ref, (UNIT[dt] + 2.0 ** -22) * ref.abs() + 2.0 ** -22 * (p.abs() @ w.detach().double().abs()), "dx")


@pytest.mark.parametrize("rows,words", [(6, 100), (70, 100), (70, 30)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_cross_gradients_of_the_largest_losses_gradients(rows, words, dt):
    """Gradients of single losses past 2^127 (no power of two in fp32 lies above them) beside others, with a weight so
    small that dx is finite: the same digits as of gradients 2^127 times smaller, which other tests pin."""
    from tests.test_gpu_decoder import _cross_case
    from turboadam_amd import linear_cross_entropy

    log(f"cross of the largest gradients {rows} {words} {dt}")
    x, w, t, dl = _cross_case(rows, 40, words, dt, 0.2, scale=2.0 ** -9)
    dl[1], dl[3] = 1.75, -1.5
    leaves = [v.requires_grad_() for v in (x, w)]
    small = torch.autograd.grad(linear_cross_entropy(*leaves, t, reduction="none"), leaves, dl)
    large = torch.autograd.grad(linear_cross_entropy(*leaves, t, reduction="none"), leaves[:1], dl * 2.0 ** 127)
    for a, b in zip(large, small):  # a power of two changes no bit but of what lies below 2^-126 in the second
        a, b = a.double() * 2.0 ** -127, b.double()
        assert bool(torch.isfinite(a).all()) and bool(((a - b).abs() <= 2.0 ** -126).all())


@pytest.mark.parametrize("rows,inputs,words", [(8, 331, 5003), (30, 64, 700), (70, 331, 40), (90, 48, 333)])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_cross_gradients_of_one_argument(rows, inputs, words, dt):
    """Passes for dx or dw alone, which copy nothing that they do not read; their sums may be cut otherwise than those of
    both, so either is within its rounding and 2^-18 of its norm of the other (sums of up to 5003 terms, 2^-23 of their
    parts a step, of random signs)."""
    from tests.test_gpu_decoder import _cross_case
    from turboadam_amd import linear_cross_entropy

    log(f"cross of one gradient {rows}x{inputs}x{words} {dt}")
    x, w, t, _ = _cross_case(rows, inputs, words, dt, 0.2)
    leaves = [v.requires_grad_() for v in (x, w)]
    both = torch.autograd.grad(linear_cross_entropy(*leaves, t), leaves)
    for i in range(2):
        some = [v.detach().requires_grad_(j == i) for j, v in enumerate((x, w))]
        got, = torch.autograd.grad(linear_cross_entropy(*some, t), [some[i]])
        assert float((got.double() - both[i].double()).norm()) <= (2 * UNIT[dt] + 2.0 ** -18) * float(both[i].double().norm()), i


@pytest.mark.parametrize("dt", list(DTYPES))
def test_cross_few_rows_over_more_words_than_a_piece(dt):
    """Past 2^20 words the backward pass of few rows takes pieces by tiles; the bounds are those of the other tests."""
    from tests.test_gpu_decoder import _check_cross, _cross_case

    log(f"cross of few rows over more words than a piece {dt}")
    _check_cross(*_cross_case(5, 24, (1 << 20) + 777, dt, 0.3), dt, "mean")
    _check_cross(*_cross_case(30, 9, (1 << 20) + 2, dt, 0.3), dt, "none")


@pytest.mark.parametrize("scale", [2.0 ** 21, 2.0 ** 26, 2.0 ** 28, 2.0 ** 40])
@pytest.mark.parametrize("rows,words", [(20, 3001), (50, 60), (300, 2777)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_cross_loss_of_exact_logits_past_single_steps(rows, words, dt, scale):
    """Logits that lie a thousandth of themselves apart or are the same: a loss is the difference to the largest and the
    logarithm of how many of those there are, 2^-23 of either."""
    from turboadam_amd import linear_cross_entropy

    log(f"cross of exact logits {rows}x{words} {dt} scale {scale}")
    x, w, t = _exact_case(rows, 16, words, dt, scale)
    z = x.double() @ w.double().t()
    number = (z == z.amax(1, keepdim=True)).sum(1).double().log()
    want = z.amax(1) - z.gather(1, t[:, None])[:, 0] + number  # in 64 bits too a sum with the logarithm would be rounded
    away = torch.where(z < z.amax(1, keepdim=True), z.amax(1, keepdim=True) - z, math.inf).amin(1)
    assert bool((away > 100).all())  # nothing else counts
    _within(linear_cross_entropy(x, w, t, reduction="none"), want, 2.0 ** -22 * (want.abs() + number), "loss")
