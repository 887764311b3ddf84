"""Microscaled rows and their operators in 64 bits: what clipenc_op_*_mx compute, from the definitions alone (test infrastructure).

Block of 32 values v: X = clamp(floor(log2 max|v|) - emax, -127, 127); elements v / 2^X to the nearest value of the format, a tie to
the even code, larger ones to the largest; a block with an infinity or a NaN is NaN."""
import math

import numpy as np

BLOCK = 32
EMAX = {"e2m1": 2, "e4m3": 8}


def grid(fmt):
    """The format's non-negative values in the order of their codes."""
    if fmt == "e2m1":
        return np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    return np.array([c / 8 * 2.0 ** -6 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)])


def nearest_code(a, fmt):
    """Codes of a >= 0."""
    g = grid(fmt)
    hi = np.clip(np.searchsorted(g, a, side="left"), 1, len(g) - 1)
    lo = hi - 1
    below, above = a - g[lo], g[hi] - a
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return np.where(up, hi, lo)


def padded(cols):
    return -(-cols // 128) * 128


def quantize(x, fmt):
    """(codes [rows, kp] with the sign on top, scale bytes [rows, kp / 32]) of float64 rows."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    v = np.zeros((rows, padded(cols)))
    v[:, :cols] = x
    v = v.reshape(rows, -1, BLOCK)
    fine = np.isfinite(v).all(-1)
    v = np.where(fine[..., None], v, 0.0)
    most = np.abs(v).max(-1)
    e = np.where(most > 0, np.frexp(most)[1] - 1 - EMAX[fmt], -127)
    e = np.clip(e, -127, 127)
    s = np.ldexp(v, -e[..., None])
    sign_bit = 8 if fmt == "e2m1" else 128
    codes = nearest_code(np.abs(s), fmt) | np.where(np.signbit(s), sign_bit, 0)
    return codes.reshape(rows, -1).astype(np.uint8), np.where(fine, e + 127, 255).astype(np.uint8)


def pack(codes, fmt):
    return codes if fmt != "e2m1" else (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def values(codes, scale, fmt, cols):
    """What (codes, scale) stand for, float64 [rows, cols]."""
    g = grid("e2m1" if fmt == "e2m1" else "e4m3")
    top = 8 if fmt == "e2m1" else 128
    mag = np.append(g, [np.nan])[codes & (top - 1)] if fmt != "e2m1" else g[codes & 7]
    v = np.where(codes & top, -mag, mag)
    if fmt == "e4m3_row":
        return (v * np.asarray(scale, dtype=np.float64)[:, None])[:, :cols]
    unit = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(int) - 127))
    return (v.reshape(len(v), -1, BLOCK) * unit[..., None]).reshape(len(v), -1)[:, :cols]


def unpack(data, fmt):
    if fmt != "e2m1":
        return data
    return np.stack([data & 15, data >> 4], -1).reshape(len(data), -1)


def norm(h, gamma, beta, kind, eps):
    """float64 rows h -> the norm's y."""
    h = np.asarray(h, dtype=np.float64)
    if kind == "layer":
        h = h - h.mean(1, keepdims=True)
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * gamma
    return y if beta is None else y + beta


def activate(u, act):
    if act == "gelu":
        return 0.5 * u * np.vectorize(math.erfc)(-u / math.sqrt(2.0))
    return u * 0.5 * (1 + np.tanh(0.851 * u)) if act == "quick_gelu" else u      # sigmoid(1.702 u)


def linear(a, w, bias, act, residual):
    """(result, sum of the products' magnitudes) of float64 operands."""
    u = a @ w.T
    size = np.abs(a) @ np.abs(w).T
    if bias is not None:
        u, size = u + bias, size + np.abs(bias)
    y = activate(u, act)
    return (y if residual is None else y + residual), size
