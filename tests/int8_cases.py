"""Inputs, tolerances and checks that the tests of products in 8-bit integers share.

Tolerances. u = 2^-24. The sums are exact; one is rounded to f32, multiplied with two scales and added to the bias: three roundings of the
product and one of the sum of both, then half a step of the result's type."""
import numpy as np

from group_norm_cases import HALF_STEP, TINY, U
from helium_amd.int8 import pitch
from oracle import int8 as oracle

# tokens, inputs, channels
SMALL = [(1, 1, 1), (1, 16, 5), (3, 17, 16), (16, 64, 33), (2, 300, 70), (17, 130, 17), (40, 96, 64), (64, 257, 40)]


def inputs(tokens, columns, channels, bias, seed):
    """Quantised operands, padded, their scales and the bias. The whole numbers go to their ends, -127 and 127."""
    rng = np.random.default_rng(seed)

    def matrix(rows):
        q = np.zeros((rows, pitch(columns)), np.int8)
        q[:, :columns] = np.clip(np.rint(rng.standard_normal((rows, columns)) * 50), -127, 127)
        return q

    scales = lambda rows: np.exp(rng.standard_normal(rows)).astype(np.float32)  # noqa: E731
    host = {"x": matrix(tokens), "x_scales": scales(tokens), "weights": matrix(channels), "weight_scales": scales(channels)}
    return dict(host, bias=(100 * rng.standard_normal(channels)).astype(np.float32) if bias else None)


def check(host, dtype, y):
    """y: f32 values"""
    args = host["x"], host["x_scales"], host["weights"], host["weight_scales"]
    product = oracle.product(*args)
    want = oracle.product(*args, host["bias"])
    off = 3 * U * np.abs(product) + U * np.abs(want)
    off = off + HALF_STEP[dtype] * 1.01 * (np.abs(want) + off) + TINY[dtype]
    wrong = ~(np.abs(y - want) <= off)
    if dtype == "f16":   # (its largest value is 65504, its step there 32: what is 65520 or more rounds to infinity, within the sum's error of that either way)
        wrong &= ~(np.isinf(y) & (np.sign(y) == np.sign(want)) & (np.abs(want) * (1 + 4 * U) >= 65520))
    assert not wrong.any(), (int(wrong.sum()), np.argwhere(wrong)[0], y[wrong][0], want[wrong][0])
