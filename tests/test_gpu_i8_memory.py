"""GPU tests: weights are made from memory of the current slot's device only; anything else is refused on the host, before a kernel
could read it."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_host_memory_is_refused(hb):
    import torch
    from hearth_b200 import lib
    L = lib.load()
    f, q = np.ones((4, 128), dtype=np.float32), np.ones((4, 128), dtype=np.int8)
    fd, qd = torch.from_numpy(f).cuda(), torch.from_numpy(q).cuda()
    h = C.c_void_p()
    assert L.hb200_weight_i8_quantize_dev(4, 128, f.ctypes.data, 128, None, C.byref(h)) == -4 and b"device" in L.hb200_last_error()
    assert L.hb200_weight_i8_upload_dev(4, 128, q.ctypes.data, 128, fd.data_ptr(), None, C.byref(h)) == -4
    assert L.hb200_weight_i8_upload_dev(4, 128, qd.data_ptr(), 128, f.ctypes.data, None, C.byref(h)) == -4
    assert not h
    torch.ones(3, device="cuda").add_(1)  # and the refusals leave no CUDA error behind
    # page-locked host memory is readable from the device, and memory inside an allocation is memory of the device
    pinned = torch.from_numpy(f).pin_memory()
    for p in (pinned.data_ptr(), fd[1:].data_ptr()):
        assert L.hb200_weight_i8_quantize_dev(3, 128, p, 128, None, C.byref(h)) == 0
        assert L.hb200_weight_i8_free(h) == 0
    assert L.hb200_weight_i8_upload_dev(0, 128, None, 128, None, None, C.byref(h)) == 0 and L.hb200_weight_i8_free(h) == 0


def test_memory_of_another_device_is_refused(hb):
    import torch
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    with pytest.raises(hb.Hb200Error, match="device 1"):
        hb.WeightI8.quantize_dev(torch.ones(4, 128, device="cuda:1"))
    with pytest.raises(hb.Hb200Error, match="device 1"):
        hb.WeightI8.upload_dev(torch.ones(4, 128, dtype=torch.int8, device="cuda:1"), torch.ones(4, device="cuda:1"))
