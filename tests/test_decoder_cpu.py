"""CPU: the C entries of gated layers, cross entropy and rotary heads check their arguments before
any launch and lay out their workspaces; the Python entries refuse host tensors; rotary's
frequencies.  No GPU call."""

import ctypes
import math

import pytest
import torch

from turboadam_amd import _lib


def _gated(**kw):
    d = _lib.TamGated()
    d.rows, d.inputs, d.outputs, d.dtype = 40, 24, 56, _lib.TAM_DTYPE_BF16
    for k in ("x", "gate", "up", "h", "kept", "dh", "dx", "dgate", "dup"):
        setattr(d, k, 0x10000)
    for k, v in kw.items():
        setattr(d, k, v)
    d.ldx = kw.get("ldx", d.inputs)
    d.ldw = kw.get("ldw", d.outputs if d.w_in_out else d.inputs)
    return d


def _cross(**kw):
    d = _lib.TamCross()
    d.rows, d.inputs, d.vocabulary, d.dtype, d.reduction = 40, 24, 56, _lib.TAM_DTYPE_BF16, _lib.TAM_CROSS_MEAN
    for k in ("x", "w", "target", "loss", "kept", "dloss", "dx", "dw"):
        setattr(d, k, 0x10000)
    for k, v in kw.items():
        setattr(d, k, v)
    d.ldx, d.ldw = kw.get("ldx", d.inputs), kw.get("ldw", d.inputs)
    return d


def _rotary(**kw):
    d = _lib.TamRotary()
    d.batch, d.tokens, d.dim, d.rotated, d.positions64 = 2, 5, 64, 32, 1
    d.positions = d.frequencies = 0x10000
    for h in (d.q, d.k):
        h.x = h.w = h.dy = h.y = h.dw = 0x10000
        h.heads = 3
    for k, v in kw.items():
        at, _, name = k.rpartition("__")
        setattr(getattr(d, at) if at else d, name, v)
    return d


def _need(fn, d, backward):
    need = ctypes.c_size_t(123)
    rc = fn(ctypes.byref(d), backward, ctypes.byref(need))
    return rc, need.value, _lib.load().tam_last_error().decode()


def test_struct_mirrors_have_the_headers_sizes():
    assert ctypes.sizeof(_lib.TamGated) == 128
    assert ctypes.sizeof(_lib.TamCross) == 136
    assert ctypes.sizeof(_lib.TamHeads) == 120
    assert ctypes.sizeof(_lib.TamRotary) == 328


@pytest.mark.parametrize("kw,code,text", [
    ({"dtype": 3}, 1, "dtype"), ({"activation": 5}, 1, "activation"), ({"x": None}, 1, "null"), ({"gate": None}, 1, "null"),
    ({"up": None}, 1, "null"), ({"ldx": 23}, 1, "stride"), ({"ldw": 23}, 1, "stride"), ({"w_in_out": 1, "ldw": 55}, 1, "stride"),
    ({"rows": 1 << 31}, 4, "2^31"), ({"ldx": 1 << 21}, 4, "2^21"), ({"outputs": (1 << 20) - 64}, 4, "2^20"),
])
def test_gated_rejects(kw, code, text):
    lib = _lib.load()
    for backward in (0, 1):
        rc, _, msg = _need(lib.tam_gated_workspace, _gated(**kw), backward)
        assert rc == code and text in msg, (rc, msg)
    assert lib.tam_gated(ctypes.byref(_gated(**kw)), None, 0, None) == code


def test_gated_missing_arrays_workspaces_and_nothing():
    lib = _lib.load()
    assert _need(lib.tam_gated_workspace, _gated(h=None), 0)[0] == 1
    assert _need(lib.tam_gated_workspace, _gated(dh=None), 1)[0] == 1
    assert _need(lib.tam_gated_workspace, _gated(kept=None), 1)[0] == 1
    assert _need(lib.tam_gated_workspace, _gated(kept=0x10008), 1)[0] == 1
    assert _need(lib.tam_gated_workspace, _gated(), 0)[:2] == (0, 0)
    rc, need, _ = _need(lib.tam_gated_workspace, _gated(), 1)
    assert rc == 0 and need >= 40 * 2 * 64 * 2  # dg and du, rows of whole lines
    d = _gated(inputs=25)  # rows that are not whole 16 bytes: copied
    rc, need, _ = _need(lib.tam_gated_workspace, d, 0)
    assert rc == 0 and need >= 2 * 64 * (40 + 56 + 56)
    assert lib.tam_gated(ctypes.byref(d), 0x1000, need - 1, None) == 2
    assert lib.tam_gated(ctypes.byref(d), 0x1010, need, None) == 1
    assert lib.tam_gated(None, None, 0, None) == 1
    assert lib.tam_gated_workspace(ctypes.byref(d), 0, None) == 1
    for kw in ({"rows": 0}, {"outputs": 0, "ldw": 24}):
        assert lib.tam_gated(ctypes.byref(_gated(x=None, gate=None, up=None, h=None, **kw)), None, 0, None) == 0
    assert lib.tam_gated_kept(3, 9, _lib.TAM_DTYPE_BF16) == 3 * 2 * 48
    assert lib.tam_gated_kept(3, 9, _lib.TAM_DTYPE_F32) == 3 * 2 * 64
    out = (ctypes.c_uint32 * 4)(9, 9, 9, 9)
    assert lib.tam_gated_tiles(ctypes.byref(_gated(rows=32)), 0, out) == 0 and list(out) == [0, 0, 0, 0]
    assert lib.tam_gated_tiles(ctypes.byref(_gated()), 0, out) == 0 and list(out) == [64, 1, 0, 0]
    assert lib.tam_gated_tiles(ctypes.byref(_gated()), 1, out) == 0 and out[0] == 64 and out[2] == 64
    assert lib.tam_gated_tiles(ctypes.byref(_gated()), 0, None) == 1


@pytest.mark.parametrize("kw,code,text", [
    ({"dtype": 3}, 1, "dtype"), ({"reduction": 3}, 1, "reduction"), ({"x": None}, 1, "null"), ({"w": None}, 1, "null"),
    ({"ldx": 23}, 1, "stride"), ({"ldw": 23}, 1, "stride"), ({"rows": 1 << 31}, 4, "2^31"),
    ({"ldw": 1 << 21}, 4, "2^21"), ({"vocabulary": 0}, 1, "vocabulary"), ({"piece": 100}, 1, "256"),
    ({"piece": 1 << 21}, 1, "2^20"), ({"kept": 0x10010}, 1, "256 bytes"),
])
def test_cross_rejects(kw, code, text):
    lib = _lib.load()
    for backward in (0, 1):
        rc, _, msg = _need(lib.tam_cross_workspace, _cross(**kw), backward)
        assert rc == code and text in msg, (rc, msg)
    assert lib.tam_cross(ctypes.byref(_cross(**kw)), None, 0, None) == code


def test_cross_missing_arrays_workspaces_and_nothing():
    lib = _lib.load()
    assert _need(lib.tam_cross_workspace, _cross(loss=None), 0)[0] == 1
    assert _need(lib.tam_cross_workspace, _cross(target=None), 0)[0] == 1
    for k in ("kept", "dloss"):
        assert _need(lib.tam_cross_workspace, _cross(**{k: None}), 1)[0] == 1
    d = _cross()
    for backward, call in ((0, lib.tam_cross), (1, lib.tam_cross_backward)):
        rc, need, _ = _need(lib.tam_cross_workspace, d, backward)
        assert rc == 0 and need > 0
        assert call(ctypes.byref(d), 0x1000, need - 1, None) == 2
        assert call(ctypes.byref(d), 0x1010, need, None) == 1
    assert lib.tam_cross(None, None, 0, None) == 1
    assert lib.tam_cross_workspace(ctypes.byref(d), 0, None) == 1
    assert lib.tam_cross_backward(ctypes.byref(_cross(dx=None, dw=None)), None, 0, None) == 0
    empty = dict(x=None, w=None, target=None, rows=0)
    assert lib.tam_cross(ctypes.byref(_cross(reduction=0, loss=None, **empty)), None, 0, None) == 0
    assert lib.tam_cross_kept(ctypes.byref(_cross(rows=100, vocabulary=65))) >= 256 + 1600 + 100 * 64 * 2
    assert lib.tam_cross_kept(ctypes.byref(_cross(rows=100, vocabulary=64))) < 256 + 1600 + 256 + 100 * 64 * 4
    for kw, reads in (({"rows": 32, "vocabulary": 1000}, 1), ({"rows": 33, "vocabulary": 64}, 1), ({"rows": 33, "vocabulary": 65}, 0)):
        assert lib.tam_cross_reads_x(ctypes.byref(_cross(**kw))) == reads
    assert _need(lib.tam_cross_workspace, _cross(x=None, vocabulary=65), 1)[0] == 0  # its rows are kept
    assert _need(lib.tam_cross_workspace, _cross(x=None, vocabulary=64), 1)[0] == 1
    # a piece's gradient of the logits stays within its bound, whatever the rows and words
    tiles = (ctypes.c_uint32 * 4)()
    for rows, words, size in ((8192, 128256, 2), (65536, 128256, 2), (65536, 128256, 4), (40, 1 << 22, 2), (8, 100, 4)):
        d = _cross(rows=rows, vocabulary=words, dtype=1 if size == 2 else 0)
        assert lib.tam_cross_tiles(ctypes.byref(d), 1, tiles) == 0
        piece = tiles[1]
        assert piece % 256 == 0 and 256 <= piece <= 1 << 20 and (piece == 256 or rows * (piece - 256) * size <= 512 << 20)


@pytest.mark.parametrize("kw,code,text", [
    ({"dtype": 3}, 1, "dtype"), ({"dim": 0, "rotated": 0}, 1, "no elements"), ({"rotated": 31}, 1, "odd"),
    ({"rotated": 66}, 1, "longer"), ({"dim": 1025}, 4, "1024"), ({"dim": 1024, "rotated": 1000}, 4, "1008"),
    ({"eps": -1.0}, 1, "eps"), ({"eps": math.nan}, 1, "eps"), ({"tokens": 1 << 31}, 4, "2^31"), ({"positions": None}, 1, "null"),
    ({"frequencies": None}, 1, "null"), ({"q__y": None}, 1, "null"), ({"k__y": None}, 1, "null"),
])
def test_rotary_rejects(kw, code, text):
    lib = _lib.load()
    for backward in (0, 1):
        rc, _, msg = _need(lib.tam_rotary_workspace, _rotary(**kw), backward)
        assert rc == code and text in msg, (rc, msg)
    assert lib.tam_rotary(ctypes.byref(_rotary(**kw)), None) == code


def test_rotary_missing_arrays_workspaces_and_nothing():
    lib = _lib.load()
    assert lib.tam_rotary(ctypes.byref(_rotary(q__x=None)), None) == 1
    assert _need(lib.tam_rotary_workspace, _rotary(q__dy=None), 1)[0] == 1
    assert _need(lib.tam_rotary_workspace, _rotary(q__x=None), 1)[0] == 1      # the norm's backward pass reads it
    assert _need(lib.tam_rotary_workspace, _rotary(k__w=None), 1)[0] == 1      # dw without a weight
    assert _need(lib.tam_rotary_workspace, _rotary(), 0)[:2] == (0, 0)
    rc, need, _ = _need(lib.tam_rotary_workspace, _rotary(), 1)
    assert rc == 0 and need > 0
    assert lib.tam_rotary_backward(ctypes.byref(_rotary()), 0x1000, need - 1, None) == 2
    assert lib.tam_rotary_backward(ctypes.byref(_rotary()), 0x1010, need, None) == 1
    assert lib.tam_rotary(ctypes.byref(_rotary(tokens=0)), None) == 0
    assert lib.tam_rotary(ctypes.byref(_rotary(q__heads=0, k__heads=0)), None) == 0


def test_python_entries_refuse_host_tensors():
    from turboadam_amd import gated_linear, linear_cross_entropy, rotary

    x, w, t = torch.ones(3, 4), torch.ones(5, 4), torch.zeros(3, dtype=torch.long)
    q, f = torch.ones(3, 2, 4), torch.ones(2, dtype=torch.float64)
    for call in (lambda: gated_linear(x, w, w), lambda: linear_cross_entropy(x, w, t), lambda: rotary(q, None, t, f)):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(ValueError, match="activation"):
        gated_linear(x, w, w, activation="tanh")


def test_rotary_frequencies():
    from turboadam_amd import rotary_frequencies

    f = rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1.0
    assert torch.allclose(f, torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(rotary_frequencies(64, scaling="linear", factor=4.0), f / 4.0)
    ntk = rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and abs(float(ntk[-1] * 4.0 / f[-1]) - 1.0) < 1e-12 and bool((ntk <= f).all())
    bands = rotary_frequencies(64, scaling="bands", factor=8.0, original_length=8192, low=1.0, high=4.0)
    turns = f * 8192 / (2 * math.pi)
    assert torch.equal(bands[turns > 4], f[turns > 4]) and torch.equal(bands[turns < 1], f[turns < 1] / 8.0)
    middle = (turns > 1) & (turns < 4)
    assert bool(middle.any()) and bool((bands[middle] < f[middle]).all()) and bool((bands[middle] > f[middle] / 8.0).all())
    for kw in ({"dim": 3}, {"dim": 0}, {"dim": 8, "base": 0.0}, {"dim": 8, "factor": -1.0}, {"dim": 8, "scaling": "other"},
               {"dim": 2, "scaling": "ntk"}, {"dim": 8, "scaling": "bands"},
               {"dim": 8, "scaling": "bands", "original_length": 8, "low": 4.0, "high": 4.0}):
        with pytest.raises(ValueError):
            rotary_frequencies(kw.pop("dim"), **kw)
