"""GPU tests: calls of the 8-bit linear path on another slot's objects leave the current slot as it was (two slots on one GPU)."""
import numpy as np
import pytest

from hearth_b200 import synth

pytestmark = pytest.mark.gpu

TOK, COLS, ROWS = 5, 256, 70


def _calls(hb, torch, W, A, x):
    """Every call that takes an object."""
    out, v = torch.empty(TOK, ROWS, device="cuda"), torch.empty(TOK, COLS, device="cuda")
    q, s = torch.zeros(TOK, COLS, dtype=torch.int8, device="cuda"), torch.ones(TOK, device="cuda")
    wq, ws, w = torch.empty(ROWS, COLS, dtype=torch.int8, device="cuda"), torch.empty(ROWS, device="cuda"), torch.ones(COLS, device="cuda")
    return {
        "quantize": lambda: A.quantize(x, TOK),
        "add_rms_norm": lambda: A.add_rms_norm(x, w, 1e-6, TOK),
        "silu_mul": lambda: A.silu_mul(x, x, TOK),
        "load": lambda: A.load(q, s, TOK),
        "store": lambda: A.store(q, s, TOK),
        "dequantize": lambda: A.dequantize(v, TOK),
        "weight store": lambda: W.store(wq, ws),
        "product": lambda: hb.matmul_i8_dev(W, A, TOK, out),
        "host product": lambda: hb.matmul_i8(W, x.cpu().numpy()),
        "refused product": lambda: pytest.raises(hb.Hb200Error, hb.matmul_i8_dev, W, A, TOK + 1, torch.empty(TOK + 1, ROWS, device="cuda")),
        "activation free": lambda: A.free(),
        "weight free": lambda: W.free(),
    }


def test_the_current_slot_stays(hb, oracle):
    import torch
    x = torch.randn(TOK, COLS, device="cuda")
    hb.init_multi(devices=[0, 0])
    try:
        hb.set_slot(0)
        W0 = hb.WeightI8.quantize_dev(torch.randn(ROWS, COLS, device="cuda"))
        packed = synth.weights(8, ROWS, COLS, seed=3)
        B0 = hb.Weight.upload(8, ROWS, COLS, packed)
        hb.set_slot(1)
        W1, A1 = hb.WeightI8.quantize_dev(torch.randn(ROWS, COLS, device="cuda")), hb.ActI8(TOK, COLS)
        hb.set_slot(0)
        for name, call in _calls(hb, torch, W1, A1, x).items():
            call()
            A, B = hb.ActI8(TOK, COLS), hb.Act(1, COLS)  # in slot 0, which set_slot selected
            A.quantize(x, TOK)
            try:
                hb.matmul_i8_dev(W0, A, TOK, torch.empty(TOK, ROWS, device="cuda"))
                B.quantize(1, x_dev=x[:1].contiguous())
                hb.dot_rows_dev(B0, B, 1, torch.empty(1, ROWS, device="cuda"))
            except hb.Hb200Error as e:
                pytest.fail(f"after {name}: {e}")
            A.free(); B.free()
            hb.set_slot(0)
        W0.free(); B0.free()
    finally:
        hb.set_slot(0)


def test_creating_in_the_current_slot_only(hb):
    """Calls on slot 0's objects from slot 1: what is created next belongs to slot 1."""
    import torch
    hb.init_multi(devices=[0, 0])
    x = torch.randn(TOK, COLS, device="cuda")
    try:
        hb.set_slot(0)
        A0, W0 = hb.ActI8(TOK, COLS), hb.WeightI8.upload(np.ones((ROWS, COLS), dtype=np.int8), np.ones(ROWS, dtype=np.float32))
        hb.set_slot(1)
        A0.quantize(x, TOK)
        A1 = hb.ActI8(TOK, COLS)
        with pytest.raises(hb.Hb200Error, match="slot"):
            hb.matmul_i8_dev(W0, A1, TOK, torch.empty(TOK, ROWS, device="cuda"))
        for h in (A0, A1, W0):
            h.free()
    finally:
        hb.set_slot(0)
