"""CPU: limits that the C entries of gated layers, cross entropy and rotary heads check before any launch, and what they
choose and lay out for calls that want some of the gradients.  No GPU call."""

import ctypes

import pytest

from tests.test_decoder_cpu import _cross, _gated, _need, _rotary
from turboadam_amd import _lib


@pytest.mark.parametrize("eps,code", [(0.0, 0), (2.0 ** -126, 0), (1.0, 0), (2.0 ** -127, 1), (2.0 ** -149, 1), (float("inf"), 1)])
def test_rotary_eps_is_zero_or_a_normal_number(eps, code):
    for backward in (0, 1):
        rc, _, msg = _need(_lib.load().tam_rotary_workspace, _rotary(eps=eps), backward)
        assert rc == code and (rc == 0 or "eps" in msg), (rc, msg)


def _tiles(fn, d):
    out = (ctypes.c_uint32 * 4)()
    assert fn(ctypes.byref(d), 1, out) == 0
    return list(out)


def test_weights_gradients_alone_are_cut_by_their_own_sums():
    """Without dx the estimate takes the rows' sums, not those of the product that is not run: these calls' sums are cut, or
    their pieces and tiles are those of the whole pass, where the other length had 1 part, 4096 words and tiles of 128."""
    lib, bf16, f32 = _lib.load(), _lib.TAM_DTYPE_BF16, _lib.TAM_DTYPE_F32
    one = _gated(rows=8192, inputs=256, outputs=8192, dtype=bf16, dx=None)
    assert _tiles(lib.tam_gated_tiles, one) == [0, 0, 128, 2]
    for kw, piece, tile, parts in ((dict(rows=8192, inputs=4096, vocabulary=128256, dtype=bf16), 32256, 256, 1),
                                   (dict(rows=8192, inputs=768, vocabulary=50257, dtype=bf16), 21760, 256, 1),
                                   (dict(rows=1237, inputs=515, vocabulary=9973, dtype=f32), 9984, 64, 2)):
        got = _tiles(lib.tam_cross_tiles, _cross(dx=None, **kw))
        assert got[1:] == [piece, tile, 1 << 16 | parts], (kw, got)


def test_cross_takes_no_memory_for_copies_that_nothing_reads():
    """x's rows are copied for dw and for tiles of logits, w's (odd ones) for dx and those: a pass without either takes
    its gradient of the logits and a few bytes a row."""
    lib, bf16 = _lib.load(), _lib.TAM_DTYPE_BF16

    def need(**kw):
        rc, bytes_, msg = _need(lib.tam_cross_workspace, _cross(dtype=bf16, **kw), 1)
        assert rc == 0, msg
        return bytes_

    many = dict(rows=540001, inputs=4096, vocabulary=40)
    assert need(dw=None, **many) < 540001 * (128 + 16) + 4096
    assert need(**many) > 540001 * 4096 * 2
    few = dict(rows=8, inputs=7191, vocabulary=72376)
    dz, w = 8 * (72376 + 64) * 2, 72376 * 7191 * 2
    assert need(dx=None, **few) < dz + 8 * 7232 * 2 + 4096  # with x's rows
    assert w < need(dw=None, **few) < w + 72376 * 82 + dz + 33 * 8 * 7191 * 4  # with w's, and dx's sums in parts
    assert need(dw=None, rows=8, inputs=8000, vocabulary=40) < 8 * 128 + 4096
    assert need(dw=None, dx=None, **few) == 0


@pytest.mark.parametrize("backward", [0, 1])
def test_launches_of_too_many_threads_are_refused_before_any(backward):
    """A launch takes fewer than 2^32 threads: 2^24 workgroups of 256. What needs more is refused where the workspace's size
    is asked, and what is just below is not."""
    lib, f32, bf16 = _lib.load(), _lib.TAM_DTYPE_F32, _lib.TAM_DTYPE_BF16
    most = 1 << 31
    for entry, make, kw, code in [
            # 64-tiles of short rows: 2^25 of them, and 2^23
            (lib.tam_gated_workspace, _gated, dict(rows=most - 1, inputs=8, outputs=16), 4),
            (lib.tam_gated_workspace, _gated, dict(rows=most >> 3, inputs=8, outputs=16), 0),
            (lib.tam_cross_workspace, _cross, dict(rows=most - 1, inputs=8, vocabulary=1000), 4),
            (lib.tam_cross_workspace, _cross, dict(rows=1 << 20, inputs=8, vocabulary=1000), 0),
            # copies of odd rows: 2^32 units of 8, and 2^28
            (lib.tam_gated_workspace, _gated, dict(rows=1 << 27, inputs=249, outputs=8), 4),
            (lib.tam_gated_workspace, _gated, dict(rows=1 << 23, inputs=249, outputs=8), 0),
            # columns of few rows: 2^27 of them are 2^32 threads, but a backward pass takes 2^20 at a time
            (lib.tam_cross_workspace, _cross, dict(rows=2, inputs=8, vocabulary=1 << 28), 0 if backward else 4),
            (lib.tam_cross_workspace, _cross, dict(rows=2, inputs=8, vocabulary=1 << 20), 0)]:
        for dtype in (f32, bf16):
            rc, _, msg = _need(entry, make(dtype=dtype, **kw), backward)
            assert rc == code and (rc == 0 or "2^32" in msg), (kw, dtype, rc, msg)
