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


def test_a_call_that_runs_out_of_memory_leaves_no_error_behind(hb):
    """The host-buffer product of a size whose output (2.2 TB) no device holds: refused by the allocator, and neither the next launch of
    torch nor the library's own takes the error for its own."""
    import torch
    from hearth_b200 import lib
    rows, tok = 8388480, 65535
    W = hb.WeightI8.upload_dev(torch.ones(rows, 1, dtype=torch.int8, device="cuda"), torch.ones(rows, device="cuda"))
    x, out = np.ones(tok, dtype=np.float32), np.zeros(1, dtype=np.float32)
    assert lib.load().hb200_matmul_i8(W._h, x.ctypes.data, tok, out.ctypes.data) == -6  # (before anything is written to `out`)
    torch.ones(3, device="cuda").add_(1)
    W.free()
    W = hb.WeightI8.upload(np.ones((3, 128), dtype=np.int8), np.ones(3, dtype=np.float32))
    assert lib.load().hb200_matmul_i8(W._h, np.ones(128, dtype=np.float32).ctypes.data, 1, (got := np.zeros(3, dtype=np.float32)).ctypes.data) == 0
    assert (got == np.float32(np.float32(127 * 128) * (np.float32(1) / np.float32(127)))).all()
    W.free()


def test_objects_of_a_slot_that_moved_to_another_device_are_refused(hb):
    """An object outlives hb200_shutdown; its slot may then be bound to another device.  Here the object's own record of its device (the
    second int behind the handle) is changed instead: every call that would read it there is refused, freeing is not."""
    import torch
    W, A, B = hb.WeightI8.quantize_dev(torch.ones(4, 128, device="cuda")), hb.ActI8(2, 128), hb.ActI8(2, 128)
    x, q, s = torch.ones(2, 128, device="cuda"), torch.ones(4, 128, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    w, out = torch.ones(128, device="cuda"), torch.full((2, 4), 5.0, device="cuda")
    B.quantize(x, 2)
    for h in (W, A):
        record = C.c_int.from_address(h._p + 4)
        assert record.value == h.device
        record.value = h.device + 1
    calls = [lambda: A.quantize(x, 2), lambda: A.add_rms_norm(x, w, 1e-6, 2), lambda: A.silu_mul(x, x, 2), lambda: A.load(q, s, 2), lambda: A.store(q, s, 2),
             lambda: A.dequantize(x, 2), lambda: W.store(q, s), lambda: hb.matmul_i8_dev(W, A, 2, out), lambda: hb.matmul_i8_dev(W, B, 2, out),
             lambda: hb.matmul_i8(W, np.ones((2, 128), dtype=np.float32))]
    for i, call in enumerate(calls):
        with pytest.raises(hb.Hb200Error, match="device"):
            call()
            pytest.fail(f"call {i} was accepted")
    assert (out == 5).all()
    for h in (W, A, B):
        h.free()
