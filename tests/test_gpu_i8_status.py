"""GPU tests of what the 8-bit product reports when a bounded wait on the device has run out."""
import os
import subprocess
import sys

import numpy as np
import pytest

import i8_ref as R
from test_bounds_build import ROOT, bounds_lib
from test_gpu_peers import _build_rank

pytestmark = pytest.mark.gpu


def test_the_host_buffer_product_reports_an_expired_wait(hb):
    """An expired wait stands in the slot's status word (here that of a rank whose neighbour never launches): the next call that
    waits for the device must return it, not a success, and the one after it runs as ever."""
    import torch
    rng = np.random.default_rng(7)
    q, s = rng.integers(-128, 128, size=(70, 300)).astype(np.int8), rng.random(70).astype(np.float32)
    x = rng.standard_normal((40, 300)).astype(np.float32)
    qx, sx = R.round_rows(x)
    want = R.product(q, s, qx, sx)
    W = hb.WeightI8.upload(q, s)
    dev = torch.device("cuda:0")
    bufs = [hb.PeerBuffer.alloc(33) for _ in range(2)]
    batch, acts, Ws = _build_rank(hb, torch, dev, 0, 2, 1, bufs, True, specs=[(8, 33, 256)])
    try:
        batch.launch()
        torch.cuda.synchronize()
        with pytest.raises(hb.Hb200Error) as e:
            hb.matmul_i8(W, x)
        assert e.value.code == -9
        hb.check_status()  # reported once
        assert (np.abs(hb.matmul_i8(W, x) - want) <= R.PRODUCT_RTOL * np.abs(want)).all()
    finally:
        batch.free()
        for h in [*acts.values(), *Ws, W]:
            h.free()
        for b in bufs:
            b.close()


def test_a_cta_without_sums_keeps_its_whole_cluster_from_storing():
    """Of the CTAs that finish a tile together, each in turn reports a wait that ran out (the debug build's self-test: nothing does,
    and every sum is complete): its neighbours must leave the outputs as they were, too."""
    code = ("from hearth_b200 import api, lib; api.init(0); l = lib.load(); rc = l.hb200_bounds_selftest(); "
            "assert rc == 0, (rc, l.hb200_last_error()); assert api.matmul_i8_kernel(200, 2048, 9) == 'i8_tcgen05_n16_split'; print('selftest ok')")
    p = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=dict(os.environ, HB200_LIB=bounds_lib()), capture_output=True, text=True, timeout=600)
    assert p.returncode == 0 and "selftest ok" in p.stdout, (p.stdout + p.stderr)[-2000:]
