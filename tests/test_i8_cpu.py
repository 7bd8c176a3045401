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
