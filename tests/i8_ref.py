"""Plain numpy restatement of the 8-bit linear path (include/hb200.h), with the rounding steps its header fixes."""
import numpy as np

MIN_MAX = np.float32(2.0 ** -100)
U = 2.0 ** -24  # half a step of float32, relative


def round_rows(v):
    """float32 rows -> (int8 rows, float32 scales): every step one float32 operation."""
    v = np.asarray(v, dtype=np.float32)
    with np.errstate(all="ignore"):
        a = np.abs(v).max(axis=1)
        bad = ~np.isfinite(v).all(axis=1)
        live = ~bad & (a >= MIN_MAX)
        inv = np.where(live, np.float32(127) / np.where(live, a, np.float32(1)), np.float32(0)).astype(np.float32)
        q = np.rint(np.where(live[:, None], v, np.float32(0)) * inv[:, None]).astype(np.int8)
        scale = np.where(live, a / np.float32(127), np.float32(0)).astype(np.float32)
    scale[bad] = np.nan
    return q, scale


def add_rms_norm(x, residual, weight, eps):
    """(h float32, int8 rows, scales in float64)."""
    with np.errstate(all="ignore"):
        h = x if residual is None else (x + residual).astype(np.float32)
        q, base = round_rows((weight[None, :] * h).astype(np.float32))
        mean = (h.astype(np.float64) ** 2).mean(axis=1)
        scale = base.astype(np.float64) / np.sqrt(mean + np.float64(np.float32(eps)))
    return h, q, scale


def silu_mul64(gate, up):
    g = gate.astype(np.float64)
    with np.errstate(all="ignore"):
        return g / (1.0 + np.exp(-g)) * up.astype(np.float64)


def product(q_w, s_w, q_x, s_x):
    """float64 [tokens, rows] from int8 operands and float32 scales."""
    acc = q_x.astype(np.int64) @ q_w.astype(np.int64).T if q_x.size < 1 << 16 else (q_x.astype(np.float64) @ q_w.astype(np.float64).T)
    return acc.astype(np.float64) * s_w.astype(np.float64)[None, :] * s_x.astype(np.float64)[:, None]


# (float)acc is off by U, the two multiplications by U each, relative to the product: 3 U and terms of the order U^2.
PRODUCT_RTOL = 3.01 * U
