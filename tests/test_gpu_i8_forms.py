"""GPU tests of the 8-bit linear path: forms of its calls that the header allows, at the sizes where each kernel variant runs (integers
exactly, sums in 64 bits, against i8_ref.py)."""
import numpy as np
import pytest

import i8_ref as R
from test_gpu_i8 import EPS, NORM_RTOL, PRODUCTS, SILU_V, _cuda, _product_case, _read, _rng

pytestmark = pytest.mark.gpu

# one CTA per row with one to eight float4s a thread, a cluster per row, rows that are read twice; aligned and odd widths
NORM_ROWS = [(1, 1), (3, 129), (5, 4099), (9, 5120), (3, 17408), (2, 65533), (300, 257), (260, 4096), (256, 20000), (65, 33000), (66, 33001)]


@pytest.mark.parametrize("seq,cols", NORM_ROWS)
@pytest.mark.parametrize("form", ["into x", "into x, no residual", "new, no residual", "into the residual, odd stride"])
def test_norm_sums_go_where_the_header_allows(hb, seq, cols, form):
    import torch
    rng = _rng(seq, cols, 71)
    x = rng.standard_normal((seq, cols)).astype(np.float32)
    r = None if "no residual" in form else (3 * rng.standard_normal((seq, cols))).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(cols)).astype(np.float32)
    h, want_q, want_s = R.add_rms_norm(x, r, w, EPS)
    pad = 3 if "odd" in form else 0
    xd = torch.full((seq, cols + pad), 9.0, device="cuda")
    xd[:, :cols] = _cuda(x)
    rd = None
    if r is not None:
        rd = torch.full((seq, cols + pad), 9.0, device="cuda")
        rd[:, :cols] = _cuda(r)
    target = xd if form.startswith("into x") else rd if form.startswith("into the residual") else torch.empty(seq, cols + pad, device="cuda")
    A = hb.ActI8(seq, cols)
    A.add_rms_norm(xd[:, :cols], _cuda(w), EPS, seq, residual_dev=None if rd is None else rd[:, :cols], sum_dev=target[:, :cols])
    q, s = _read(hb, A, seq)
    got = target.cpu().numpy()
    assert np.array_equal(got[:, :cols].view(np.uint32), h.view(np.uint32)) and (pad == 0 or (got[:, cols:] == 9).all())
    assert np.array_equal(q, want_q)
    assert (np.abs(s - want_s) <= NORM_RTOL * np.abs(want_s)).all()
    if target is not xd:
        assert np.array_equal(xd[:, :cols].cpu().numpy(), x)
    A.free()


@pytest.mark.parametrize("seq,cols,rows", PRODUCTS)
def test_products_accumulate_at_odd_strides(hb, seq, cols, rows):
    """The shapes of test_product, which run every kernel variant: onto rows an odd number of values apart, with values around them."""
    import torch
    W, A, want = _product_case(hb, seq, cols, rows, 5)
    base = _rng(seq, rows).standard_normal((seq, rows)).astype(np.float32) * np.float32(np.abs(want).mean())
    ld = rows + 1 + rows % 2 * 2
    ld += 1 - ld % 2
    out = torch.full((seq + 2, ld), 77.0, device="cuda")
    out[1:-1, :rows] = _cuda(base)
    hb.matmul_i8_dev(W, A, seq, out[1:-1, :rows], accumulate=True)
    got = out.cpu().numpy()
    hb.check_status()
    # the product within three roundings of its own, the addition one of the sum
    assert (np.abs(got[1:-1, :rows] - (base + want)) <= 1.01 * R.U * np.abs(base + want) + R.PRODUCT_RTOL * 1.01 * np.abs(want)).all()
    assert (got[0] == 77).all() and (got[-1] == 77).all() and (got[:, rows:] == 77).all()
    A.free(); W.free()


def test_host_products_of_two_widths_in_turn(hb):
    """What the host-buffer product keeps is made anew as widths alternate and token counts grow and shrink."""
    rng = _rng(91)
    parts = []
    for rows, cols in ((200, 300), (130, 1000)):
        q, s = rng.integers(-128, 128, size=(rows, cols)).astype(np.int8), rng.random(rows).astype(np.float32)
        parts.append((hb.WeightI8.upload(q, s), q, s))
    for seq in (3, 90, 1, 20, 150, 2):
        for W, q, s in parts:
            x = rng.standard_normal((seq, q.shape[1])).astype(np.float32)
            want = R.product(q, s, *R.round_rows(x))
            assert (np.abs(hb.matmul_i8(W, x) - want) <= R.PRODUCT_RTOL * np.abs(want)).all()
    for W, _, _ in parts:
        W.free()


# 32 MiB of input and more: lines marked to leave L2 first, with four or eight float4s a thread and with rows read twice
LARGE = [(2100, 4096), (4200, 2048), (500, 17408), (300, 30000), (260, 33000), (1700, 5003)]


@pytest.mark.parametrize("seq,cols", LARGE)
def test_large_row_calls(hb, seq, cols):
    import torch
    rng = _rng(seq, cols, 17)
    x, y = (3 * rng.standard_normal((seq, cols))).astype(np.float32), rng.standard_normal((seq, cols)).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(cols)).astype(np.float32)
    A, xd, yd = hb.ActI8(seq, cols), _cuda(x), _cuda(y)
    A.quantize(xd, seq)
    q, s = _read(hb, A, seq)
    want_q, want_s = R.round_rows(x)
    assert np.array_equal(q, want_q) and np.array_equal(s, want_s)
    v = torch.empty(seq, cols, device="cuda")
    A.dequantize(v, seq)
    assert np.array_equal(v.cpu().numpy(), want_q.astype(np.float32) * want_s[:, None])
    A.silu_mul(xd, yd, seq)
    q, s = _read(hb, A, seq)
    e = R.silu_mul64(x, y)
    a = np.abs(e).max(axis=1)
    r = e * 127 / a[:, None]
    assert (np.abs(s - a / 127) <= (SILU_V + 1.01 * R.U) * a / 127).all()
    assert (np.abs(q - r) <= 0.5 + np.abs(r) * (2 * SILU_V + 2.1 * R.U)).all()
    h, want_q, want_s = R.add_rms_norm(x, y, w, EPS)
    A.add_rms_norm(xd, _cuda(w), EPS, seq, residual_dev=yd, sum_dev=yd)
    q, s = _read(hb, A, seq)
    assert np.array_equal(yd.cpu().numpy(), h) and np.array_equal(q, want_q)
    assert (np.abs(s - want_s) <= NORM_RTOL * np.abs(want_s)).all()
    A.free()


def test_the_checks_in_python_serve_the_same_calls(hb, monkeypatch):
    """Without the compiled calls the results are the same bits."""
    import torch
    seq, d, ffn = 20, 512, 640
    W1, W2 = hb.WeightI8.quantize_dev(torch.randn(2 * ffn, d, device="cuda")), hb.WeightI8.quantize_dev(torch.randn(d, ffn, device="cuda"))
    A1, A2 = hb.ActI8(seq, d), hb.ActI8(seq, ffn)
    x, res, w = torch.randn(seq, d, device="cuda"), torch.randn(seq, d, device="cuda"), torch.rand(d, device="cuda")

    def layer():
        h, gu, v = torch.empty(seq, d, device="cuda"), torch.empty(seq, 2 * ffn, device="cuda"), torch.empty(seq, ffn, device="cuda")
        A1.add_rms_norm(x, w, EPS, seq, residual_dev=res, sum_dev=h)
        hb.matmul_i8_dev(W1, A1, seq, gu)
        A2.silu_mul(gu[:, :ffn], gu[:, ffn:], seq)
        A2.dequantize(v, seq)
        hb.matmul_i8_dev(W2, A2, seq, h, accumulate=True)
        A1.quantize(h, seq)
        hb.matmul_i8_dev(W1, A1, seq, gu)
        return h, gu, v

    want = layer()
    monkeypatch.setattr(hb, "_fast", hb._ChecksInPython)
    for a, b in zip(layer(), want):
        assert torch.equal(a, b)
    for o in (W1, W2, A1, A2):
        o.free()
