"""GPU tests of the 8-bit linear path against the numpy restatement in i8_ref.py (integers exactly, sums in 64 bits)."""
import numpy as np
import pytest

import i8_ref as R

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _rng(*key):
    return np.random.default_rng(sum((i + 1) * 7919 * int(k) for i, k in enumerate(key)) + 11)


def _cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _ints(rng, rows, cols):
    q = rng.integers(-128, 128, size=(rows, cols)).astype(np.int8)
    return q


def _read(hb, act, seq):
    """Values and scales of an activation, host."""
    import torch
    q = torch.empty(seq, act.n_cols, dtype=torch.int8, device="cuda")
    s = torch.empty(seq, device="cuda")
    act.store(q, s, seq)
    return q.cpu().numpy(), s.cpu().numpy()


# ---------------------------------------------------------------------------------- rounding to 8 bits

ROWS = [(1, 1), (1, 5), (2, 31), (3, 128), (7, 129), (1, 4096), (5, 4099), (9, 5120), (1, 12288), (3, 17408), (2, 32768), (2, 32772), (1, 65536), (2, 65533),
        (300, 257), (260, 4096), (257, 8192), (256, 20000), (90, 17000), (100, 12288), (65, 33000), (1000, 2050), (64, 6272)]


@pytest.mark.parametrize("seq,cols", ROWS)
def test_quantize_integers_are_exact(hb, seq, cols):
    x = _rng(seq, cols).standard_normal((seq, cols)).astype(np.float32) * 3
    A = hb.ActI8(seq, cols)
    A.quantize(_cuda(x), seq)
    q, s = _read(hb, A, seq)
    want_q, want_s = R.round_rows(x)
    assert np.array_equal(q, want_q)
    assert np.array_equal(s.view(np.uint32), want_s.view(np.uint32))
    import torch
    v = torch.empty(seq, cols, device="cuda")
    A.dequantize(v, seq)
    assert np.array_equal(v.cpu().numpy(), want_q.astype(np.float32) * want_s[:, None])
    A.free()


def test_quantize_special_rows(hb):
    x = _rng(1).standard_normal((8, 300)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-36)     # below the smallest row maximum: zeros
    x[2, 299] = np.inf
    x[3, 0] = np.nan
    x[4, 7] = -np.inf
    x[5] *= np.float32(1e37)
    x[6] = 0
    x[6, 5] = np.float32(2.0 ** -100)
    A = hb.ActI8(8, 300)
    A.quantize(_cuda(x), 8)
    q, s = _read(hb, A, 8)
    want_q, want_s = R.round_rows(x)
    assert np.array_equal(q, want_q)
    assert np.array_equal(np.isnan(s), np.isnan(want_s)) and np.isnan(s).tolist() == [False, False, True, True, True, False, False, False]
    assert np.array_equal(s[~np.isnan(s)], want_s[~np.isnan(s)])
    assert q[6, 5] == 127
    A.free()


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("ld", [100, 101, 104])
def test_quantize_strides_and_alignment(hb, shift, ld):
    import torch
    x = _rng(shift, ld).standard_normal((6, 100)).astype(np.float32)
    buf = torch.full((6 * ld + shift + 8,), 7.0, device="cuda")
    view = buf[shift:shift + 6 * ld].view(6, ld)[:, :100]
    view.copy_(_cuda(x))
    A = hb.ActI8(6, 100)
    A.quantize(view, 6)
    q, _ = _read(hb, A, 6)
    assert np.array_equal(q, R.round_rows(x)[0])
    out = torch.full((6 * ld + shift + 8,), 9.0, device="cuda")
    A.dequantize(out[shift:shift + 6 * ld].view(6, ld)[:, :100], 6)
    got = out.cpu().numpy()
    rows = got[shift:shift + 6 * ld].reshape(6, ld)
    want_q, want_s = R.round_rows(x)
    assert np.array_equal(rows[:, :100], want_q.astype(np.float32) * want_s[:, None])
    assert (rows[:, 100:] == 9).all() and (got[:shift] == 9).all() and (got[shift + 6 * ld:] == 9).all()
    A.free()


def test_rows_behind_the_last_are_left(hb):
    import torch
    rng = _rng(5)
    x, y = rng.standard_normal((20, 500)).astype(np.float32), rng.standard_normal((3, 500)).astype(np.float32)
    A = hb.ActI8(20, 500)
    A.quantize(_cuda(x), 20)
    A.quantize(_cuda(y), 3)
    q, s = _read(hb, A, 20)
    want_q, want_s = R.round_rows(np.concatenate([y, x[3:]]))
    assert np.array_equal(q, want_q) and np.array_equal(s, want_s)
    v = torch.full((20, 500), 5.0, device="cuda")
    A.dequantize(v, 3)
    assert (v[3:] == 5).all()
    A.quantize(_cuda(x), 0)  # nothing to do
    A.quantize(_cuda(y[0]), 1)  # one row as a vector
    assert np.array_equal(_read(hb, A, 20)[0], want_q)
    A.free()


@pytest.mark.parametrize("rows,cols,ld,shift", [(11, 77, 77, 0), (11, 77, 80, 0), (5, 128, 128, 1), (3, 2048, 2064, 0), (6, 2100, 2112, 16), (1, 4097, 4100, 0),
                                                (9, 16, 16, 0), (2, 1, 1, 3)])
def test_load_and_store_round_trip(hb, rows, cols, ld, shift):
    import torch
    q = _ints(_rng(ld, rows), rows, cols)
    s = _rng(ld, 2).random(rows).astype(np.float32)
    buf = torch.zeros(rows * ld + shift, dtype=torch.int8, device="cuda")[shift:].view(rows, ld)
    buf[:, :cols] = _cuda(q)
    A = hb.ActI8(16, cols)
    A.load(buf[:, :cols], _cuda(s), rows)
    got_q, got_s = _read(hb, A, rows)
    assert np.array_equal(got_q, q) and np.array_equal(got_s, s)
    flat = torch.full((rows * ld + shift,), 3, dtype=torch.int8, device="cuda")
    back = flat[shift:].view(rows, ld)
    A.store(back[:, :cols], None, rows)
    assert np.array_equal(back[:, :cols].cpu().numpy(), q) and (back[:, cols:] == 3).all() and (flat[:shift] == 3).all()
    only = torch.zeros(rows, device="cuda")
    A.store(None, only, rows)
    assert np.array_equal(only.cpu().numpy(), s)
    A.free()


# ---------------------------------------------------------------------------------- norm

# Sum of squares of positive terms: at most 64 fused additions in a thread, then ten levels of halving: (64 + 10) U; the
# mean's division and the addition of eps U each, the square root halves that and adds U, reciprocal, a / 127 and the last
# product U each: (76 / 2 + 4) U.
NORM_RTOL = 42.5 * R.U


@pytest.mark.parametrize("seq,cols", ROWS)
@pytest.mark.parametrize("form", ["residual", "plain", "in_place"])
def test_add_rms_norm(hb, seq, cols, form):
    import torch
    rng = _rng(seq, cols, 3)
    x = rng.standard_normal((seq, cols)).astype(np.float32)
    r = None if form == "plain" else (4 * rng.standard_normal((seq, cols))).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(cols)).astype(np.float32)
    h, want_q, want_s = R.add_rms_norm(x, r, w, EPS)
    A = hb.ActI8(seq, cols)
    xd, rd, wd = _cuda(x), None if r is None else _cuda(r), _cuda(w)
    sum_dev = None if form == "plain" else rd if form == "in_place" else torch.empty_like(xd)
    A.add_rms_norm(xd, wd, EPS, seq, residual_dev=rd, sum_dev=sum_dev)
    q, s = _read(hb, A, seq)
    if sum_dev is not None:
        assert np.array_equal(sum_dev.cpu().numpy().view(np.uint32), h.view(np.uint32))
    assert np.array_equal(q, want_q)
    assert (np.abs(s - want_s) <= NORM_RTOL * np.abs(want_s)).all()
    A.free()


def test_add_rms_norm_special_rows(hb):
    import torch
    x = _rng(8).standard_normal((6, 200)).astype(np.float32)
    r = _rng(9).standard_normal((6, 200)).astype(np.float32)
    x[0] = 0; r[0] = 0
    x[1, 4] = np.nan
    r[2, 199] = np.inf
    x[3] = np.float32(1e25)   # h^2 leaves f32: NaN, not a silent zero
    x[4] = -r[4]              # cancels to an all-zero row
    w = np.ones(200, dtype=np.float32)
    A = hb.ActI8(6, 200)
    s_dev = torch.empty(6, 200, device="cuda")
    A.add_rms_norm(_cuda(x), _cuda(w), EPS, 6, residual_dev=_cuda(r), sum_dev=s_dev)
    q, s = _read(hb, A, 6)
    assert np.isnan(s).tolist() == [False, True, True, True, False, False]
    assert (q[:5] == 0).all() and s[0] == 0 and s[4] == 0
    h, want_q, want_s = R.add_rms_norm(x, r, w, EPS)
    assert np.array_equal(q[5], want_q[5]) and abs(s[5] - want_s[5]) <= NORM_RTOL * want_s[5]
    assert np.array_equal(s_dev.cpu().numpy(), h, equal_nan=True)
    A.free()


# ---------------------------------------------------------------------------------- gated activation

# expf within 1 ulp (2 U) where exp(-g) counts, then 1 + e, the division, the product: v within 5 U of the exact value (a
# gate below about -87 makes exp(-g) overflow: v is a zero where the exact value is below 1e-35, far under a step).
SILU_V = 5.0 * R.U


@pytest.mark.parametrize("seq,cols", ROWS)
@pytest.mark.parametrize("packed", [False, True])
def test_silu_mul(hb, seq, cols, packed):
    rng = _rng(seq, cols, 4)
    g = (3 * rng.standard_normal((seq, cols))).astype(np.float32)
    u = rng.standard_normal((seq, cols)).astype(np.float32)
    A = hb.ActI8(seq, cols)
    if packed:
        both = _cuda(np.concatenate([g, u], axis=1))
        A.silu_mul(both[:, :cols], both[:, cols:], seq)
    else:
        A.silu_mul(_cuda(g), _cuda(u), seq)
    q, s = _read(hb, A, seq)
    v = R.silu_mul64(g, u)
    a = np.abs(v).max(axis=1)
    # scale: a is within SILU_V, a / 127 adds U
    assert (np.abs(s - a / 127) <= (SILU_V + 1.01 * R.U) * a / 127).all()
    # 127 / a and the product add U each; then half a step
    r = v * 127 / a[:, None]
    assert (np.abs(q - r) <= 0.5 + np.abs(r) * (2 * SILU_V + 2.1 * R.U)).all()
    A.free()


def test_silu_mul_extremes(hb):
    g = np.array([[-200.0, 200.0, -88.0, 0.0, 30.0]], dtype=np.float32).repeat(3, 0)
    u = np.array([[5.0, 1.0, 1.0, 9.0, -1.0]], dtype=np.float32).repeat(3, 0)
    u[1] = 0
    g[2, 1] = np.nan
    A = hb.ActI8(3, 5)
    A.silu_mul(_cuda(g), _cuda(u), 3)
    q, s = _read(hb, A, 3)
    assert q[0].tolist() == [0, 127, 0, 0, -19] and s[1] == 0 and (q[1:] == 0).all() and np.isnan(s[2])
    A.free()


# ---------------------------------------------------------------------------------- product

PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 4096, 300), (2, 129, 127), (8, 64, 1), (15, 100, 257), (16, 2048, 256), (17, 640, 130), (31, 1, 129),
            (32, 5120, 512), (33, 300, 64), (64, 1152, 384), (65, 1000, 200), (77, 2050, 1024), (128, 512, 128), (129, 2048, 384), (200, 4097, 129),
            (256, 256, 256), (257, 384, 300), (300, 1111, 777), (513, 384, 700), (1000, 896, 515), (1024, 1024, 2048), (2049, 130, 1025),
            (2600, 1411, 2100), (2333, 2049, 2900), (1025, 3333, 2700), (5003, 1665, 1153)]


def _product_case(hb, seq, cols, rows, key=0):
    rng = _rng(seq, cols, rows, key)
    qw, qx = _ints(rng, rows, cols), _ints(rng, seq, cols)
    sw, sx = (rng.random(rows) + 0.01).astype(np.float32), (rng.random(seq) + 0.01).astype(np.float32)
    W = hb.WeightI8.upload(qw, sw)
    A = hb.ActI8(seq, cols)
    A.load(_cuda(qx), _cuda(sx), seq)
    return W, A, R.product(qw, sw, qx, sx)


@pytest.mark.parametrize("seq,cols,rows", PRODUCTS)
def test_product(hb, seq, cols, rows):
    import torch
    W, A, want = _product_case(hb, seq, cols, rows)
    out = torch.full((seq + 2, rows + 3), 77.0, device="cuda")
    hb.matmul_i8_dev(W, A, seq, out[1:seq + 1, :rows])
    got = out.cpu().numpy()
    hb.check_status()
    assert (np.abs(got[1:-1, :rows] - want) <= R.PRODUCT_RTOL * np.abs(want)).all()
    assert (got[0] == 77).all() and (got[-1] == 77).all() and (got[:, rows:] == 77).all()
    # an aligned, tight output gives the same bits
    tight = torch.empty(seq, rows, device="cuda")
    hb.matmul_i8_dev(W, A, seq, tight)
    assert np.array_equal(tight.cpu().numpy(), got[1:-1, :rows])
    A.free(); W.free()


@pytest.mark.parametrize("seq,cols,rows", [(1, 4096, 300), (5, 100, 129), (40, 1024, 256), (300, 513, 260), (700, 256, 512)])
def test_product_accumulates(hb, seq, cols, rows):
    import torch
    W, A, want = _product_case(hb, seq, cols, rows, 1)
    base = _rng(seq).standard_normal((seq, rows)).astype(np.float32) * np.float32(np.abs(want).mean())
    for extra in (0, 1):
        out = torch.zeros(seq, rows + extra, device="cuda")
        out[:, :rows] = _cuda(base)
        hb.matmul_i8_dev(W, A, seq, out[:, :rows], accumulate=True)
        got = out[:, :rows].cpu().numpy()
        assert (np.abs(got - (base + want)) <= 1.01 * R.U * np.abs(base + want) + R.PRODUCT_RTOL * 1.01 * np.abs(want)).all()
    A.free(); W.free()


@pytest.mark.parametrize("seq", [1, 20, 300])
def test_product_at_the_widest_sum_is_exact(hb, seq):
    """65536 columns of -128 x -128: the sum is 2^30."""
    import torch
    cols, rows = 65536, 130
    qw, qx = np.full((rows, cols), -128, dtype=np.int8), np.full((seq, cols), -128, dtype=np.int8)
    qw[5, ::2] = 127
    W = hb.WeightI8.upload(qw, np.ones(rows, dtype=np.float32))
    A = hb.ActI8(seq, cols)
    A.load(_cuda(qx), _cuda(np.ones(seq, dtype=np.float32)), seq)
    out = torch.empty(seq, rows, device="cuda")
    hb.matmul_i8_dev(W, A, seq, out)
    got = out.cpu().numpy()
    assert (np.delete(got, 5, axis=1) == 2.0 ** 30).all()
    assert (got[:, 5] == np.float32(32768 * 128 * 128 - 32768 * 127 * 128)).all()
    A.free(); W.free()


def test_fewer_tokens_than_the_activation_holds(hb):
    import torch
    W, A, want = _product_case(hb, 130, 700, 200, 2)
    for seq in (1, 9, 16, 33, 70, 129):
        out = torch.full((130, 200), 4.0, device="cuda")
        hb.matmul_i8_dev(W, A, seq, out)
        got = out.cpu().numpy()
        assert (np.abs(got[:seq] - want[:seq]) <= R.PRODUCT_RTOL * np.abs(want[:seq])).all() and (got[seq:] == 4).all()
    out.fill_(4.0)
    hb.matmul_i8_dev(W, A, 0, out)
    assert (out == 4).all()
    A.free(); W.free()


def test_a_bad_token_spoils_only_itself(hb):
    import torch
    x = _rng(21).standard_normal((40, 600)).astype(np.float32)
    x[7, 3] = np.nan
    x[20, 599] = np.inf
    x[30] = 0
    W = hb.WeightI8.quantize_dev(_cuda(_rng(22).standard_normal((150, 600)).astype(np.float32)))
    A = hb.ActI8(40, 600)
    A.quantize(_cuda(x), 40)
    out = torch.empty(40, 150, device="cuda")
    hb.matmul_i8_dev(W, A, 40, out)
    got = out.cpu().numpy()
    bad = np.isnan(got)
    assert bad[[7, 20]].all() and not np.delete(bad, [7, 20], axis=0).any() and (got[30] == 0).all()
    A.free(); W.free()


# ---------------------------------------------------------------------------------- weights

@pytest.mark.parametrize("rows,cols", [(1, 1), (130, 77), (257, 513), (300, 4100)])
def test_weight_forms_agree(hb, rows, cols):
    import torch
    rng = _rng(rows, cols)
    w = rng.standard_normal((rows, cols)).astype(np.float32)
    q, s = R.round_rows(w)
    wide = torch.zeros(rows, cols + 5, device="cuda")
    wide[:, :cols] = _cuda(w)
    wide_q = torch.zeros(rows, cols + 3, dtype=torch.int8, device="cuda")
    wide_q[:, :cols] = _cuda(q)
    made = [hb.WeightI8.upload(q, s), hb.WeightI8.upload_dev(wide_q[:, :cols], _cuda(s)), hb.WeightI8.quantize_dev(wide[:, :cols])]
    lo, hi = rows // 3, rows
    made.append(hb.WeightI8.upload(q, s, rows=(lo, hi)))
    for W in made:
        a, b = (lo, hi) if W.n_rows != rows else (0, rows)
        got_q = torch.empty(b - a, cols, dtype=torch.int8, device="cuda")
        got_s = torch.empty(b - a, device="cuda")
        W.store(got_q, got_s)
        assert np.array_equal(got_q.cpu().numpy(), q[a:b]) and np.array_equal(got_s.cpu().numpy(), s[a:b])
        assert W.n_cols == cols and W.resident_bytes >= (b - a) * cols
        W.free()
    empty = hb.WeightI8.upload(q, s, rows=(1, 1) if rows > 1 else (0, 0))
    A = hb.ActI8(2, cols)
    hb.matmul_i8_dev(empty, A, 2, torch.empty(2, 1, device="cuda"))
    A.free(); empty.free()


# ---------------------------------------------------------------------------------- as they are used together

def _layer(hb, x, res, up_down, norm_w, A1, A2, bufs, seq):
    """norm with the residual's addition -> gate|up -> gated activation -> down, added onto the residual."""
    W1, W2 = up_down
    gu, stream_sum = bufs
    ffn = W2.n_cols
    A1.add_rms_norm(x, norm_w, EPS, seq, residual_dev=res, sum_dev=stream_sum)
    hb.matmul_i8_dev(W1, A1, seq, gu)
    A2.silu_mul(gu[:, :ffn], gu[:, ffn:], seq)
    hb.matmul_i8_dev(W2, A2, seq, stream_sum, accumulate=True)


def _layer_setup(hb, seq, d, ffn):
    import torch
    rng = _rng(seq, d, ffn)
    x, res = rng.standard_normal((seq, d)).astype(np.float32), rng.standard_normal((seq, d)).astype(np.float32)
    w1, w2 = (rng.standard_normal((2 * ffn, d)) / np.sqrt(d)).astype(np.float32), (rng.standard_normal((d, ffn)) / np.sqrt(ffn)).astype(np.float32)
    nw = (1 + 0.1 * rng.standard_normal(d)).astype(np.float32)
    W = (hb.WeightI8.quantize_dev(_cuda(w1)), hb.WeightI8.quantize_dev(_cuda(w2)))
    A = (hb.ActI8(seq, d), hb.ActI8(seq, ffn))
    bufs = (torch.empty(seq, 2 * ffn, device="cuda"), torch.empty(seq, d, device="cuda"))
    h, q, s = R.add_rms_norm(x, res, nw, EPS)
    q1, s1 = R.round_rows(w1)
    gu = R.product(q1, s1, q, s)
    v = R.silu_mul64(gu[:, :ffn].astype(np.float32), gu[:, ffn:].astype(np.float32))
    a = np.abs(v).max(axis=1, keepdims=True)
    q2, s2 = R.round_rows(w2)
    want = h + R.product(q2, s2, np.rint(v * 127 / a), (a[:, 0] / 127))
    # a value next to a border may go the other way (the float32 chain in front of it is off by some 1e-6): one step of
    # one product each, at most a handful of the row's
    slack = 4 * 127 * s2.max() * a / 127
    return x, res, W, nw, A, bufs, want, slack


@pytest.mark.parametrize("seq,d,ffn", [(1, 256, 640), (3, 513, 1000), (40, 1024, 2048), (300, 384, 1152)])
def test_layer_runs_together(hb, seq, d, ffn):
    x, res, W, nw, A, bufs, want, slack = _layer_setup(hb, seq, d, ffn)
    _layer(hb, _cuda(x), _cuda(res), W, _cuda(nw), A[0], A[1], bufs, seq)
    got = bufs[1].cpu().numpy()
    assert (np.abs(got - want) <= slack + 1e-5 * np.abs(want)).all()
    for h in W + A:
        h.free()


@pytest.mark.parametrize("seq", [1, 40, 300])
def test_captured_and_replayed_with_new_inputs(hb, seq):
    import torch
    x, res, W, nw, A, bufs, want, _ = _layer_setup(hb, seq, 512, 1024)
    xd, rd, nd = _cuda(x), _cuda(res), _cuda(nw)
    _layer(hb, xd, rd, W, nd, A[0], A[1], bufs, seq)
    first = bufs[1].clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        _layer(hb, xd, rd, W, nd, A[0], A[1], bufs, seq)
    bufs[1].zero_()
    for _ in range(5):
        g.replay()
    assert torch.equal(bufs[1], first)
    xd.mul_(-0.5)
    g.replay()
    second = bufs[1].clone()
    _layer(hb, xd, rd, W, nd, A[0], A[1], bufs, seq)
    assert torch.equal(bufs[1], second) and not torch.equal(first, second)
    hb.check_status()
    for h in W + A:
        h.free()


def test_products_on_several_streams_read_one_activation(hb):
    import torch
    cols = 2048
    W = [_product_case(hb, 1, cols, 384 + 128 * i, i) for i in range(3)]
    W, drop = [w for w, _, _ in W], [a for _, a, _ in W]
    for a in drop:
        a.free()
    x = _cuda(_rng(77).standard_normal((33, cols)).astype(np.float32))
    A = hb.ActI8(33, cols)
    A.quantize(x, 33)
    want = []
    for w in W:
        out = torch.empty(33, w.n_rows, device="cuda")
        hb.matmul_i8_dev(w, A, 33, out)
        want.append(out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in W]
    outs = [torch.zeros_like(o) for o in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for w, o, st in zip(W, outs, streams):
            hb.matmul_i8_dev(w, A, 33, o, stream=st)
    torch.cuda.synchronize()
    for o, e in zip(outs, want):
        assert torch.equal(o, e)
    A.free()
    for w in W:
        w.free()


def test_back_to_back_calls_on_changing_inputs(hb):
    """The kernels start ahead of their predecessors' ends; what they read must not."""
    import torch
    cols, rows = 1024, 640
    W = hb.WeightI8.quantize_dev(_cuda(_rng(31).standard_normal((rows, cols)).astype(np.float32)))
    A = hb.ActI8(24, cols)
    xs = [torch.randn(24, cols, device="cuda") * (i + 1) for i in range(16)]
    slow = []
    for x in xs:
        out = torch.empty(24, rows, device="cuda")
        A.quantize(x, 24)
        torch.cuda.synchronize()
        hb.matmul_i8_dev(W, A, 24, out)
        torch.cuda.synchronize()
        slow.append(out)
    for _ in range(3):
        fast = []
        for x in xs:
            out = torch.empty(24, rows, device="cuda")
            A.quantize(x, 24)
            hb.matmul_i8_dev(W, A, 24, out)
            fast.append(out)
        torch.cuda.synchronize()
        for a, b in zip(slow, fast):
            assert torch.equal(a, b)
    A.free(); W.free()


def test_host_buffer_product(hb):
    rng = _rng(55)
    q, s = _ints(rng, 200, 300), rng.random(200).astype(np.float32)
    W = hb.WeightI8.upload(q, s)
    for seq in (3, 1, 50):
        x = rng.standard_normal((seq, 300)).astype(np.float32)
        qx, sx = R.round_rows(x)
        want = R.product(q, s, qx, sx)
        assert (np.abs(hb.matmul_i8(W, x) - want) <= R.PRODUCT_RTOL * np.abs(want)).all()
    assert hb.matmul_i8(W, np.zeros(300, dtype=np.float32)).shape == (200,)
    with pytest.raises(hb.Hb200Error):
        hb.matmul_i8(W, np.zeros(301, dtype=np.float32))
    W.free()


def test_refusals(hb):
    import torch
    E = hb.Hb200Error
    W = hb.WeightI8.quantize_dev(torch.randn(64, 96, device="cuda"))
    A = hb.ActI8(4, 96)
    x, w = torch.randn(4, 96, device="cuda"), torch.ones(96, device="cuda")
    out = torch.full((4, 64), 6.0, device="cuda")
    A.quantize(x, 4)
    bad = [
        lambda: A.quantize(x, 5),                                          # beyond the capacity
        lambda: A.quantize(x[:, :95], 4),                                  # too narrow
        lambda: A.quantize(x.cpu(), 4),
        lambda: A.quantize(x.half(), 4),
        lambda: A.quantize(x.t().contiguous().t(), 4),                     # columns not adjacent
        lambda: A.quantize(x[:1].expand(4, 96), 4),                        # rows on top of one another
        lambda: A.quantize(None, 4),
        lambda: A.add_rms_norm(x, w, 0.0, 4),
        lambda: A.add_rms_norm(x, w, float("nan"), 4),
        lambda: A.add_rms_norm(x, w, -1e-6, 4),
        lambda: A.add_rms_norm(x, w[:95], 1e-6, 4),
        lambda: A.add_rms_norm(x, w, 1e-6, 4, residual_dev=torch.zeros(4, 100, device="cuda")[:, :96]),
        lambda: A.add_rms_norm(x, w, 1e-6, 4, sum_dev=torch.empty(3, 96, device="cuda")),
        lambda: A.silu_mul(x, torch.zeros(4, 100, device="cuda")[:, :96], 4),
        lambda: A.silu_mul(x, x[:, :90], 4),
        lambda: A.load(torch.zeros(4, 96, device="cuda"), torch.zeros(4, device="cuda"), 4),
        lambda: A.load(torch.zeros(4, 96, dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda"), 4),
        lambda: A.dequantize(torch.empty(4, 95, device="cuda"), 4),
        lambda: A.store(None, None, 4),
        lambda: hb.matmul_i8_dev(W, A, 5, out),
        lambda: hb.matmul_i8_dev(W, A, 4, out[:, :63]),
        lambda: hb.matmul_i8_dev(W, A, 4, out[:3]),
        lambda: hb.WeightI8.upload(np.zeros((2, 3), dtype=np.int8), np.zeros(3, dtype=np.float32)),
        lambda: hb.WeightI8.upload(np.zeros((2, 3), dtype=np.float32), np.zeros(2, dtype=np.float32)),
        lambda: hb.WeightI8.upload(np.zeros((2, 3), dtype=np.int8), np.zeros(2, dtype=np.float32), rows=(1, 3)),
        lambda: hb.WeightI8.quantize_dev(torch.zeros(2, 65537, device="cuda")),
        lambda: hb.ActI8(4, 65537),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(E):
            call()
            pytest.fail(f"call {i} was accepted")
    other = hb.ActI8(4, 128)
    with pytest.raises(E):
        hb.matmul_i8_dev(W, other, 4, out)
    assert (out == 6).all()
    for h in (W, A, other):
        h.free()


def test_objects_of_two_slots(hb):
    """Two slots on one device: objects work from whichever slot is current, and do not mix."""
    import torch
    hb.init_multi(devices=[0, 0])
    try:
        hb.set_slot(1)
        x = torch.randn(5, 200, device="cuda")
        W1, A1 = hb.WeightI8.quantize_dev(torch.randn(70, 200, device="cuda")), hb.ActI8(5, 200)
        hb.set_slot(0)
        A0 = hb.ActI8(5, 200)
        out, out_host = torch.empty(5, 70, device="cuda"), None
        A1.quantize(x, 5)
        hb.matmul_i8_dev(W1, A1, 5, out)
        out_host = hb.matmul_i8(W1, x.cpu().numpy())
        assert np.array_equal(out.cpu().numpy(), out_host)
        A0.quantize(x, 5)
        with pytest.raises(hb.Hb200Error):
            hb.matmul_i8_dev(W1, A0, 5, out)
        for h in (W1, A1, A0):
            h.free()
    finally:
        hb.set_slot(0)


# ---------------------------------------------------------------------------------- order, graphs, far offsets

def test_captured_behind_copies_and_beside_another_stream(hb):
    """A graph whose calls follow a copy node and join a forked stream: the early start of the kernels must not outrun
    either."""
    import torch
    cols, rows, seq = 1536, 520, 30
    W = hb.WeightI8.quantize_dev(_cuda(_rng(41).standard_normal((rows, cols)).astype(np.float32)))
    A, B = hb.ActI8(seq, cols), hb.ActI8(seq, cols)
    src = [torch.randn(seq, cols, device="cuda") for _ in range(6)]
    xa, xb = torch.zeros(seq, cols, device="cuda"), torch.zeros(seq, cols, device="cuda")
    oa, ob = torch.zeros(seq, rows, device="cuda"), torch.zeros(seq, rows, device="cuda")
    pick = torch.zeros(seq, cols, device="cuda")

    def step(side):
        main = torch.cuda.current_stream()
        xa.copy_(pick)                       # a copy node in front of the first call
        side.wait_stream(main)
        with torch.cuda.stream(side):
            torch.mul(pick, 2.0, out=xb)
            B.quantize(xb, seq)
            hb.matmul_i8_dev(W, B, seq, ob)
        A.quantize(xa, seq)
        hb.matmul_i8_dev(W, A, seq, oa)
        main.wait_stream(side)
        oa.add_(ob)
        A.quantize(xa, seq)
        hb.matmul_i8_dev(W, A, seq, oa, accumulate=True)

    side, st = torch.cuda.Stream(), torch.cuda.Stream()
    want = []
    for s in src:
        pick.copy_(s)
        torch.cuda.synchronize()
        step(side)
        torch.cuda.synchronize()
        want.append(oa.clone())
    g = torch.cuda.CUDAGraph()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=st):
        step(side)
    for _ in range(3):
        for s, e in zip(src, want):
            pick.copy_(s)
            g.replay()
            assert torch.equal(oa, e)
    for h in (W, A, B):
        h.free()


def test_two_graphs_of_the_same_weight(hb):
    """Two captured products of one weight, replayed on two streams at once: a call keeps no scratch."""
    import torch
    cols, rows = 4096, 1024
    W = hb.WeightI8.quantize_dev(torch.randn(rows, cols, device="cuda"))
    parts = []
    for seq in (1, 40):
        A, x, out = hb.ActI8(seq, cols), torch.randn(seq, cols, device="cuda"), torch.empty(seq, rows, device="cuda")
        A.quantize(x, seq)
        hb.matmul_i8_dev(W, A, seq, out)
        want, st, g = out.clone(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=st):
            for _ in range(20):
                A.quantize(x, seq)
                hb.matmul_i8_dev(W, A, seq, out)
        parts.append((A, out, want, st, g))
    torch.cuda.synchronize()
    for _ in range(5):
        for _, out, _, st, g in parts:
            with torch.cuda.stream(st):
                out.zero_()
                g.replay()
    torch.cuda.synchronize()
    for A, out, want, _, _ in parts:
        assert torch.equal(out, want)
        A.free()
    W.free()


def test_offsets_past_32_bits(hb):
    """An activation plane of 2.1 GB, inputs and outputs of more than 2^31 values: the last tokens come out right."""
    import torch
    seq, cols, rows = 65535, 33000, 150
    x = torch.zeros(seq, cols, device="cuda")
    tail = _rng(61).standard_normal((7, cols)).astype(np.float32)
    x[-7:] = _cuda(tail)
    A = hb.ActI8(seq, cols)
    A.quantize(x, seq)
    q, s = R.round_rows(tail)
    qw = _ints(_rng(62), rows, cols)
    sw = np.full(rows, 1e-3, dtype=np.float32)
    W = hb.WeightI8.upload(qw, sw)
    out = torch.empty(seq, rows, device="cuda")
    hb.matmul_i8_dev(W, A, seq, out)
    want = R.product(qw, sw, q, s)
    assert (np.abs(out[-7:].cpu().numpy() - want) <= R.PRODUCT_RTOL * np.abs(want)).all() and not out[:-7].any()
    A.dequantize(x, seq)
    assert np.array_equal(x[-7:].cpu().numpy(), q.astype(np.float32) * s[:, None])
    A.free(); W.free()
    del x, out
    rows, cols = 40000, 64
    qw, qx = _ints(_rng(63), rows, cols), _ints(_rng(64), 3, cols)
    W = hb.WeightI8.upload(qw, np.ones(rows, dtype=np.float32))
    A = hb.ActI8(seq, cols)
    A.load(torch.zeros(seq, cols, dtype=torch.int8, device="cuda"), torch.ones(seq, device="cuda"), seq)
    rows_q = torch.zeros(seq, cols, dtype=torch.int8, device="cuda")
    rows_q[-3:] = _cuda(qx)
    A.load(rows_q, torch.ones(seq, device="cuda"), seq)
    out = torch.empty(seq, rows, device="cuda")
    hb.matmul_i8_dev(W, A, seq, out)
    assert np.array_equal(out[-3:].cpu().numpy(), (qx.astype(np.int64) @ qw.astype(np.int64).T).astype(np.float32))
    assert not out[-10000:-3].any()
    hb.check_status()
    A.free(); W.free()


def test_every_kernel_variant_is_covered_by_a_shape_above(hb):
    names = {hb.matmul_i8_kernel(n, k, m) for m, k, n in PRODUCTS}
    assert names == {"i8_tcgen05_n16", "i8_tcgen05_n16_split", "i8_tcgen05_n32", "i8_tcgen05_n32_split", "i8_tcgen05_n64", "i8_tcgen05_n64_split",
                     "i8_tcgen05_pair_n128", "i8_tcgen05_pair_n256"}, names
