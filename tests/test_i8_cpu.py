"""CPU tests of the 8-bit linear path: refusals that need no device, kernel names, and the restatement the GPU tests use."""
import ctypes as C

import numpy as np
import pytest

import i8_ref as R


@pytest.fixture(scope="module")
def lib():
    from hearth_b200 import build, lib as L
    build.build()
    return L.load()


def test_limits_are_clear_errors(lib):
    h = C.c_void_p()
    assert lib.hb200_act_i8_create(0, 128, C.byref(h)) == -4
    assert lib.hb200_act_i8_create(4, 0, C.byref(h)) == -4
    assert lib.hb200_act_i8_create(65536, 128, C.byref(h)) == -8 and b"65535" in lib.hb200_last_error()
    assert lib.hb200_act_i8_create(4, 65537, C.byref(h)) == -8 and b"65536" in lib.hb200_last_error()
    assert lib.hb200_act_i8_create(4, 128, None) == -5
    assert lib.hb200_weight_i8_info(None, None, None, None, None) == -5
    assert lib.hb200_act_i8_info(None, None, None, None) == -5
    assert lib.hb200_weight_i8_free(None) == 0 and lib.hb200_act_i8_free(None) == 0


def test_no_device_means_error_not_fallback(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is present; this test is about the device-less case")
    h = C.c_void_p()
    one = np.zeros(128, dtype=np.float32)
    p = C.c_void_p(one.ctypes.data)
    assert lib.hb200_act_i8_create(4, 128, C.byref(h)) == -1
    assert lib.hb200_weight_i8_upload(1, 128, p, p, C.byref(h)) == -1
    assert lib.hb200_weight_i8_upload_rows(1, 128, p, p, 0, 1, C.byref(h)) == -1
    assert lib.hb200_weight_i8_upload_dev(1, 128, p, 128, p, None, C.byref(h)) == -1
    assert lib.hb200_weight_i8_quantize_dev(1, 128, p, 128, None, C.byref(h)) == -1
    assert lib.hb200_weight_i8_store_dev(None, p, 128, p, None) == -1
    assert lib.hb200_act_i8_quantize_dev(None, p, 128, 1, None) == -1
    assert lib.hb200_act_i8_add_rms_norm_dev(None, p, p, 128, p, 1e-6, 1, p, 128, None) == -1
    assert lib.hb200_act_i8_silu_mul_dev(None, p, p, 128, 1, None) == -1
    assert lib.hb200_act_i8_load_dev(None, p, 128, p, 1, None) == -1
    assert lib.hb200_act_i8_store_dev(None, p, 128, p, 1, None) == -1
    assert lib.hb200_act_i8_dequantize_dev(None, p, 128, 1, None) == -1
    assert lib.hb200_matmul_i8_dev(None, None, 1, p, 128, 0, None) == -1
    assert lib.hb200_matmul_i8(None, p, 1, p) == -1


def test_kernel_names(lib):
    from hearth_b200 import api
    assert api.matmul_i8_kernel(0, 128, 1) == "none"
    assert api.matmul_i8_kernel(128, 65537, 1) == "none"
    assert api.matmul_i8_kernel(128, 128, 65536) == "none"
    for m in (1, 17, 100, 5000):
        assert api.matmul_i8_kernel(4096, 4096, m).startswith("i8_tcgen05_")


def test_restatement_rounds_and_refuses_like_the_header_says():
    v = np.array([[0.5, -1.0, 0.25, 2.0], [0, 0, 0, 0], [1e-31, 0, 0, 0], [1, np.inf, 0, 0], [1, 2, np.nan, 0]], dtype=np.float32)
    q, s = R.round_rows(v)
    assert q[0].tolist() == [32, -64, 16, 127] and s[0] == np.float32(2) / np.float32(127)  # 31.75, -63.5 (to even), 15.875
    assert (q[1:] == 0).all() and s[1] == 0 and s[2] == 0 and np.isnan(s[3:]).all()
    big = np.random.default_rng(0).standard_normal((50, 300)).astype(np.float32)
    q, s = R.round_rows(big)
    assert (np.abs(q).max(axis=1) == 127).all()
    assert np.abs(q * s[:, None].astype(np.float64) - big).max() <= s.max() * (0.5 + 127 * 4 * R.U)


@pytest.fixture()
def pycall(lib):
    """The compiled calls bound to functions that record what arrives, then bound back.  Device -1 stands for the CPU."""
    import torch
    from hearth_b200 import api
    api._i8_torch()
    from hearth_b200 import _pycall
    got = []
    vp, sz, i, fl = C.c_void_p, C.c_size_t, C.c_int, C.c_float
    kinds = [(vp, vp, sz, sz, vp), (vp, vp, vp, sz, vp, fl, sz, vp, sz, vp), (vp, vp, vp, sz, sz, vp), (vp, vp, sz, sz, vp), (vp, vp, sz, vp, sz, i, vp)]
    keep = [C.CFUNCTYPE(i, *k)(lambda *a: got.append(a) or len(got)) for k in kinds]
    _pycall.bind(*(C.cast(f, vp).value for f in keep))
    yield _pycall, got, torch
    api._F32 = None
    api._i8_torch()
    del keep


class _Stream:
    cuda_stream = 0x77


def test_compiled_calls_pass_what_they_are_given(pycall):
    call, got, torch = pycall
    st = _Stream()
    x, y = torch.zeros(4, 100)[:, :96], torch.zeros(5, 128)[:, :100]
    y100 = torch.zeros(500)[:500].view(5, 100)
    w, one = torch.zeros(96), torch.zeros(1, 96)
    X, Y, W = x.data_ptr(), y100.data_ptr(), w.data_ptr()
    assert call.quantize(0x10, -1, 96, x, 4, st) == 1 and got[-1] == (0x10, X, 100, 4, 0x77)
    assert call.dequantize(0x10, -1, 96, one.as_strided((1, 96), (1, 1)), 1, st) == 2 and got[-1] == (0x10, one.data_ptr(), 96, 1, 0x77)
    assert call.silu_mul(0x10, -1, 96, x, y100, 4, st) == 3 and got[-1] == (0x10, X, Y, 100, 4, 0x77)
    assert call.add_rms_norm(0x10, -1, 96, x, y100, w, 0.5, 4, None, st) == 4 and got[-1] == (0x10, X, Y, 100, W, 0.5, 4, None, 0, 0x77)
    assert call.add_rms_norm(0x10, -1, 96, x, None, w, 0.5, 4, y, st) == 5 and got[-1] == (0x10, X, None, 100, W, 0.5, 4, y.data_ptr(), 128, 0x77)
    assert call.matmul(0x20, 0x10, -1, 96, 4, x, True, st) == 6 and got[-1] == (0x20, 0x10, 4, X, 100, 1, 0x77)
    empty = torch.zeros(0, 96)
    assert call.quantize(0x10, -1, 96, empty, 0, st) == 7 and got[-1][2:4] == (96, 0)


def test_compiled_calls_leave_everything_else_to_the_checks_in_python(pycall):
    call, got, torch = pycall
    st = _Stream()
    x, w = torch.zeros(4, 96), torch.zeros(96)
    other = [None, 3, x.half(), x.numpy(), torch.zeros(3, 96), torch.zeros(4, 95), torch.zeros(96, 4).t(), torch.zeros(96), torch.zeros(1, 4, 96), x.to_sparse(),
             torch.zeros(4, 96, device="meta")]
    for t in other:
        assert call.quantize(0x10, -1, 96, t, 4, st) is None
        assert call.dequantize(0x10, -1, 96, t, 4, st) is None
        assert call.silu_mul(0x10, -1, 96, t, x, 4, st) is None and call.silu_mul(0x10, -1, 96, x, t, 4, st) is None
        assert call.add_rms_norm(0x10, -1, 96, t, None, w, 0.5, 4, None, st) is None
        assert call.matmul(0x20, 0x10, -1, 96, 4, t, False, st) is None
        if t is not None:
            assert call.add_rms_norm(0x10, -1, 96, x, t, w, 0.5, 4, None, st) is None
            assert call.add_rms_norm(0x10, -1, 96, x, None, w, 0.5, 4, t, st) is None
    wide = torch.zeros(4, 97)
    assert call.silu_mul(0x10, -1, 96, x, wide, 4, st) is None and call.add_rms_norm(0x10, -1, 96, x, wide, w, 0.5, 4, None, st) is None
    assert call.add_rms_norm(0x10, -1, 96, x, None, x, 0.5, 4, None, st) is None and call.add_rms_norm(0x10, -1, 96, x, None, w, 1, 4, None, st) is None
    assert call.quantize(0x10, 0, 96, x, 4, st) is None  # a CPU tensor where the handle lives on a GPU
    assert call.quantize(0x10, -1, 96, x, -1, st) is None and call.quantize(0x10, -1, 96, x, 4, "stream") is None and call.quantize(0x10, -1, 96, x) is None
    assert call.quantize(0x10, -1, 96, x, 4, None) is None
    assert not got
    with pytest.raises(TypeError):
        call.bind(0, 0, 0, 0, 0)
