"""CPU tests of when the compiled calls of the 8-bit linear path are built and used, and of the checks in Python in their place."""
import ctypes as C
import os
import shutil

import pytest


@pytest.fixture(scope="module")
def built():
    from hearth_b200 import build
    build.build()
    return build


@pytest.fixture()
def api(built):
    from hearth_b200 import api
    yield api
    api._F32 = None
    api._i8_torch()


def test_a_module_of_another_torch_is_built_anew(built, tmp_path, monkeypatch):
    src = os.path.join(built.CSRC, "pycall.cpp")
    copy = tmp_path / "_pycall.so"
    shutil.copy2(built.PYCALL, copy)
    monkeypatch.setattr(built, "PYCALL", str(copy))
    assert not built._pycall_stale(src)
    made_for = built.pycall_for()
    monkeypatch.setattr(built, "pycall_for", lambda: made_for.replace("torch ", "torch 1"))
    assert built._pycall_stale(src)


@pytest.mark.parametrize("compiler", ["/nonexistent/g++", "false"])
def test_a_missing_compiler_is_a_warning_and_no_half_module(built, tmp_path, monkeypatch, compiler):
    monkeypatch.setattr(built, "PYCALL", str(tmp_path / "_pycall.so"))
    monkeypatch.setenv("CXX", compiler)
    with pytest.warns(UserWarning, match="checked in Python"):
        assert built.build_pycall() is None
    assert not os.listdir(tmp_path)


def test_a_module_of_another_torch_is_not_used(api, monkeypatch):
    from hearth_b200 import _pycall
    api._F32 = None
    api._i8_torch()
    assert api._fast is _pycall
    monkeypatch.setattr(_pycall, "built_for", "cpython-312 torch 1.0")
    api._F32 = None
    with pytest.warns(UserWarning, match="is not used"):
        api._i8_torch()
    assert api._fast is api._ChecksInPython


def test_a_missing_module_is_not_needed(api, monkeypatch):
    import sys
    import hearth_b200
    monkeypatch.setitem(sys.modules, "hearth_b200._pycall", None)  # importing it raises
    monkeypatch.delattr(hearth_b200, "_pycall", raising=False)
    api._F32 = None
    with pytest.warns(UserWarning, match="is not used"):
        api._i8_torch()
    assert api._fast is api._ChecksInPython


class _Stream:
    cuda_stream = 0x77


class _Lib:
    """Records what the C entry points get."""

    def __init__(self):
        self.got = []

    def __getattr__(self, name):
        return lambda *a: self.got.append((name, *(x.value if isinstance(x, C._SimpleCData) else x for x in a))) or 0


def test_the_checks_in_python_pass_on_the_same(api, monkeypatch):
    """Both ways, on host tensors and a handle of device -1: what arrives at the C entry points is the same."""
    import torch
    api._F32 = None
    api._i8_torch()
    compiled, lib = api._fast, _Lib()
    names = ("hb200_act_i8_quantize_dev", "hb200_act_i8_add_rms_norm_dev", "hb200_act_i8_silu_mul_dev", "hb200_act_i8_dequantize_dev", "hb200_matmul_i8_dev")
    vp, sz, i, fl = C.c_void_p, C.c_size_t, C.c_int, C.c_float
    kinds = [(vp, vp, sz, sz, vp), (vp, vp, vp, sz, vp, fl, sz, vp, sz, vp), (vp, vp, vp, sz, sz, vp), (vp, vp, sz, sz, vp), (vp, vp, sz, vp, sz, i, vp)]
    keep = [C.CFUNCTYPE(i, *k)(lambda *a, n=n: lib.got.append((n, *a)) or 0) for n, k in zip(names, kinds)]
    A, W = object.__new__(api.ActI8), object.__new__(api.WeightI8)
    A._h, A._p, A.device, A.n_cols, A.max_seq_len, A._lib = vp(0x10), 0x10, -1, 96, 4, lib
    W._h, W._p, W.device, W.n_rows, W.n_cols = vp(0x20), 0x20, -1, 70, 96
    x, y, w, o = torch.zeros(4, 100)[:, :96], torch.zeros(4, 100)[:, :96], torch.zeros(96), torch.zeros(5, 72)
    st = _Stream()

    def all_calls():
        A.quantize(x, 4, stream=st)
        A.add_rms_norm(x, w, 0.5, 4, residual_dev=y, sum_dev=y, stream=st)
        A.add_rms_norm(x, w, 0.5, 1, stream=st)
        A.silu_mul(x, y, 3, stream=st)
        A.dequantize(x, 4, stream=st)
        api.matmul_i8_dev(W, A, 4, o, accumulate=True, stream=st)
        got, lib.got = lib.got, []
        return got

    compiled.bind(*(C.cast(f, vp).value for f in keep))
    first = all_calls()
    monkeypatch.setattr(api, "_fast", api._ChecksInPython)
    assert all_calls() == first and len(first) == 6
    with pytest.raises(api.Hb200Error):
        A.quantize(x[:, :95], 4, stream=st)
    with pytest.raises(api.Hb200Error):
        A.silu_mul(x, torch.zeros(4, 97)[:, :96], 4, stream=st)
    assert not lib.got
