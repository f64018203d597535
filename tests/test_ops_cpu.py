"""CPU: the layers' and Muon's C entries check their arguments before any launch,
lay out their workspaces, and the Python entries refuse host tensors.  No GPU call."""

import ctypes

import pytest
import torch

from turboadam_amd import _lib


def _linear(**kw):
    d = _lib.TamLinear()
    d.rows, d.inputs, d.outputs, d.dtype = 40, 24, 56, _lib.TAM_DTYPE_BF16
    for k in ("x", "w", "y", "z", "dy", "dx", "dw", "db"):
        setattr(d, k, 0x10000)
    for k, v in kw.items():
        setattr(d, k, v)
    d.ldx = kw.get("ldx", d.inputs)
    d.ldw = kw.get("ldw", d.outputs if d.w_in_out else d.inputs)
    return d


def _need(fn, d, backward):
    need = ctypes.c_size_t(123)
    rc = fn(ctypes.byref(d), backward, ctypes.byref(need))
    return rc, need.value, _lib.load().tam_last_error().decode()


def test_struct_mirrors_have_the_headers_sizes():
    assert ctypes.sizeof(_lib.TamLinear) == 136
    assert ctypes.sizeof(_lib.TamNorm) == 104
    assert ctypes.sizeof(_lib.TamMatrix) == 72


@pytest.mark.parametrize("kw,code,text", [
    ({"dtype": 3}, 1, "dtype"), ({"activation": 5}, 1, "activation"), ({"x": None}, 1, "null"),
    ({"w": None}, 1, "null"), ({"ldx": 23}, 1, "stride"), ({"ldw": 23}, 1, "stride"),
    ({"w_in_out": 1, "ldw": 55}, 1, "stride"), ({"rows": 1 << 31}, 4, "2^31"), ({"ldx": 1 << 21}, 4, "2^21"),
])
def test_linear_rejects(kw, code, text):
    lib = _lib.load()
    for backward in (0, 1):
        rc, _, msg = _need(lib.tam_linear_workspace, _linear(**kw), backward)
        assert rc == code and text in msg, (rc, msg)
    assert lib.tam_linear(ctypes.byref(_linear(**kw)), None, 0, None) == code


def test_linear_rejects_missing_arrays_of_its_pass_and_small_workspaces():
    lib = _lib.load()
    assert _need(lib.tam_linear_workspace, _linear(y=None), 0)[0] == 1
    assert _need(lib.tam_linear_workspace, _linear(dy=None), 1)[0] == 1
    assert _need(lib.tam_linear_workspace, _linear(z=None, activation=2), 1)[0] == 1
    d = _linear(inputs=25, ldx=25, ldw=25)  # rows that are not whole 16 bytes: copied
    rc, need, _ = _need(lib.tam_linear_workspace, d, 0)
    assert rc == 0 and need >= 2 * 32 * (40 + 56)
    assert lib.tam_linear(ctypes.byref(d), 0x1000, need - 1, None) == 2
    assert "workspace" in lib.tam_last_error().decode()
    assert lib.tam_linear(ctypes.byref(d), 0x1010, need, None) == 1
    assert lib.tam_linear(None, None, 0, None) == 1
    assert lib.tam_linear_workspace(ctypes.byref(d), 0, None) == 1


def test_linear_of_nothing_launches_nothing():
    lib = _lib.load()
    for kw in ({"rows": 0}, {"outputs": 0, "ldw": 24}):
        assert lib.tam_linear(ctypes.byref(_linear(x=None, w=None, y=None, **kw)), None, 0, None) == 0


def _norm(**kw):
    d = _lib.TamNorm()
    d.rows, d.n, d.ldx, d.eps = 10, 100, 100, 1e-5
    for k in ("x", "w", "b", "y", "stats", "dy", "dx", "dw", "db"):
        setattr(d, k, 0x10000)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,code,text", [
    ({"dtype": 3}, 1, "dtype"), ({"n": 0}, 1, "no elements"), ({"n": 32769, "ldx": 32769}, 4, "32768"),
    ({"ldx": 99}, 1, "stride"), ({"eps": -1.0}, 1, "eps"), ({"eps": float("nan")}, 1, "eps"), ({"x": None}, 1, "null"),
    ({"rows": 1 << 31}, 4, "2^31"),
])
def test_norm_rejects(kw, code, text):
    lib = _lib.load()
    for backward in (0, 1):
        rc, _, msg = _need(lib.tam_norm_workspace, _norm(**kw), backward)
        assert rc == code and text in msg
    assert lib.tam_norm(ctypes.byref(_norm(**kw)), None) == code


def test_norm_workspace():
    lib = _lib.load()
    assert _need(lib.tam_norm_workspace, _norm(), 0)[:2] == (0, 0)
    rc, need, _ = _need(lib.tam_norm_workspace, _norm(), 1)
    assert rc == 0 and need > 0
    assert _need(lib.tam_norm_workspace, _norm(dw=None, db=None), 1)[:2] == (0, 0)
    assert lib.tam_norm_backward(ctypes.byref(_norm()), 0x1000, need - 1, None) == 2
    assert lib.tam_norm(ctypes.byref(_norm(y=None)), None) == 1
    assert lib.tam_norm_backward(ctypes.byref(_norm(stats=None)), 0x1000, need, None) == 1


def _matrices(*shapes, **kw):
    m = (_lib.TamMatrix * len(shapes))()
    for d, (rows, cols) in zip(m, shapes):
        d.out = d.grad = d.momentum = 0x10000
        d.rows, d.cols, d.eps = rows, cols, 1e-7
        for k, v in kw.items():
            setattr(d, k, v)
    return m


def _ns(m, n=None):
    lib, need = _lib.load(), ctypes.c_size_t()
    rc = lib.tam_orthogonalize_workspace(ctypes.addressof(m), len(m) if n is None else n, ctypes.byref(need))
    return rc, need.value, lib.tam_last_error().decode()


@pytest.mark.parametrize("kw,code,text", [
    ({"out": None}, 1, "null"), ({"grad": None}, 1, "null"), ({"rows": 0}, 1, "no elements"),
    ({"cols": 65537}, 4, "65536"), ({"dtype": 3}, 1, "dtype"), ({"eps": 0.0}, 1, "eps"),
    ({"momentum": 0x10002}, 1, "misaligned"),
])
def test_orthogonalize_rejects(kw, code, text):
    rc, _, msg = _ns(_matrices((8, 8), (40, 24), **kw))
    assert rc == code and text in msg and "matrix 0" in msg


def test_orthogonalize_workspace_and_settings():
    lib = _lib.load()
    m = _matrices((200, 60), (33, 270))
    rc, need, _ = _ns(m)
    # two turns of x in two fp16 parts; q and p in two parts (fp32)
    assert rc == 0 and need >= 8 * (200 * 64 + 33 * 272) + 8 * (60 * 64 + 33 * 40)
    half = _ns(_matrices((200, 60), (33, 270), dtype=_lib.TAM_DTYPE_BF16))[1]
    assert need > half >= 6 * (200 * 64 + 33 * 272) + 4 * (60 * 64 + 33 * 40)
    co = (ctypes.c_float * 3)(3.4445, -4.775, 2.0315)
    bad = (ctypes.c_float * 3)(3.4445, float("nan"), 2.0315)
    at = ctypes.addressof(m)
    assert lib.tam_orthogonalize(at, 2, co, 0, 0x1000, need, None) == 1
    assert lib.tam_orthogonalize(at, 2, co, 65, 0x1000, need, None) == 1
    assert lib.tam_orthogonalize(at, 2, bad, 5, 0x1000, need, None) == 1
    assert lib.tam_orthogonalize(at, 2, None, 5, 0x1000, need, None) == 1
    assert lib.tam_orthogonalize(at, 2, co, 5, 0x1000, need - 1, None) == 2
    assert lib.tam_orthogonalize(at, 2, co, 5, 0x1010, need, None) == 1
    assert lib.tam_orthogonalize(at, -1, co, 5, 0x1000, need, None) == 1
    assert lib.tam_orthogonalize(None, 0, co, 5, None, 0, None) == 0
    assert lib.tam_orthogonalize_workspace(at, 2, None) == 1


def test_python_entries_refuse_host_tensors():
    from turboadam_amd import Muon, layer_norm, linear, orthogonalize

    x, w = torch.ones(3, 4), torch.ones(5, 4)
    for call in (lambda: linear(x, w), lambda: layer_norm(x), lambda: orthogonalize(x)):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()
    p = torch.nn.Parameter(w)
    p.grad = torch.ones_like(w)
    with pytest.raises(RuntimeError, match="MI355X"):
        Muon([p]).step()
    assert torch.equal(p, torch.ones(5, 4))


def test_muon_checks_its_settings():
    from turboadam_amd import Muon

    p = torch.nn.Parameter(torch.ones(4, 6))
    opt = Muon([p])
    with pytest.raises(ValueError, match="2-D"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(3))]})
    assert len(opt.param_groups) == 1
    assert opt.defaults["ns_steps"] == 5


def test_muon_refuses_an_eps_that_is_zero_to_the_kernels():
    from turboadam_amd import Muon

    p = torch.nn.Parameter(torch.ones(4, 6))
    for eps in (1e-50, 0.0, -1e-7, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            Muon([p], eps=eps)
    Muon([p], eps=1e-44)


def test_counting_library_holds_what_the_binding_loads(monkeypatch):
    """_lib.load binds every symbol, of the counting build too: it is linked of the library's sources, all of them."""
    from turboadam_amd import build

    calls = []
    monkeypatch.setattr(build, "_hipcc", lambda sources, out, verbose, extra=(): calls.append((list(sources), out, extra)))
    build.build_stats_library()
    (sources, out, extra), = calls
    assert sources == build.SOURCES and out == build.STATS_LIB_PATH and "-DTAM_STATS=1" in extra


@pytest.mark.parametrize("kw", [{"ns_coefficients": None}, {"lr": "fast"}, {"ns_steps": "many"}, {"eps": None},
                                {"lr": -1.0}])
def test_muon_keeps_no_group_that_it_refuses(kw):
    from turboadam_amd import Muon

    opt = Muon([torch.nn.Parameter(torch.ones(4, 6))])
    p = torch.nn.Parameter(torch.ones(3, 5))
    with pytest.raises((TypeError, ValueError)):
        opt.add_param_group({"params": [p], **kw})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [p]})  # and so the parameter is free


def test_tiles_are_told():
    lib, out = _lib.load(), (ctypes.c_uint32 * 4)(9, 9, 9, 9)
    assert lib.tam_linear_tiles(ctypes.byref(_linear(rows=32)), 0, out) == 0 and list(out) == [0, 0, 0, 0]
    assert lib.tam_linear_tiles(ctypes.byref(_linear(rows=33)), 0, out) == 0 and list(out) == [64, 1, 0, 0]
    assert lib.tam_linear_tiles(ctypes.byref(_linear()), 1, out) == 0 and out[0] == 64 and out[2] == 64
    assert lib.tam_linear_tiles(ctypes.byref(_linear(dx=None)), 1, out) == 0 and out[0] == 0 and out[2] == 64
    assert lib.tam_linear_tiles(ctypes.byref(_linear(dw=None)), 1, out) == 0 and out[0] == 64 and out[2] == 0
    assert lib.tam_linear_tiles(ctypes.byref(_linear(dtype=3)), 0, out) == 1
    assert lib.tam_linear_tiles(ctypes.byref(_linear()), 0, None) == 1
    small, large = _matrices((128, 128), (9, 7)), _matrices((129, 128))
    assert lib.tam_orthogonalize_tiles(ctypes.addressof(small), 2, out) == 0 and list(out) == [0, 0, 0, 0]
    assert lib.tam_orthogonalize_tiles(ctypes.addressof(large), 1, out) == 0 and list(out) == [64, 1, 64, 64]
    assert lib.tam_orthogonalize_tiles(None, 0, out) == 0 and list(out) == [0, 0, 0, 0]
    assert lib.tam_orthogonalize_tiles(ctypes.addressof(large), -1, out) == 1
    assert lib.tam_orthogonalize_tiles(ctypes.addressof(large), 1, None) == 1
