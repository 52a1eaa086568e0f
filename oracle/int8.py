"""Rows of 8-bit whole numbers with a scale each, and products of them, from the definition. Test infrastructure only."""
import numpy as np


def quantize(x):
    """x [rows, columns], f32 values -> the whole numbers and the f32 scales of the rows.

    127 x / A in 64 bits, then put on the right side of a border by the remainder 254 x - 2 q A, which 53 bits hold exactly."""
    x = x.astype(np.float64)
    finite = np.isfinite(x).all(axis=1)
    most = np.where(finite, np.abs(np.where(np.isfinite(x), x, 0)).max(axis=1), np.nan)
    a = np.where(finite & (most > 0), most, 1.0)[:, None]
    x = np.where(finite[:, None], x, 0.0)
    q = np.rint(127.0 * (x / a))
    off = 254.0 * x - 2.0 * q * a
    q = np.where((off > a) | ((off == a) & (q % 2 != 0)), q + 1, np.where((off < -a) | ((off == -a) & (q % 2 != 0)), q - 1, q))
    return q.astype(np.int8), most.astype(np.float32) / np.float32(127)


def product(q, scales, weights, weight_scales, bias=None):
    """y[t, n] = scales[t] weight_scales[n] sum over k of q[t, k] weights[n, k], in 64 bits."""
    with np.errstate(invalid="ignore"):
        y = (q.astype(np.float64) @ weights.astype(np.float64).T) * scales.astype(np.float64)[:, None] * weight_scales.astype(np.float64)
    return y if bias is None else y + bias.astype(np.float64)
