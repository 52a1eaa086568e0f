"""Inputs, tolerances and checks that the tests of gradient clipping share.

Tolerances. u = 2^-24. Sums of squares are f64: the norm is off by its rounding to f32. The factor rounds to f32, its product with a value
too, and that to the result's type."""
import numpy as np

from group_norm_cases import HALF_STEP, TINY, U, to_f32, to_storage
from oracle import gradient_clip as oracle

# sizes and types of a group
GROUPS = [
    ([1], ["f32"]),
    ([5, 0, 7, 8, 1, 4096], ["f32", "bf16", "f16", "bf16", "f16", "f32"]),
    ([8192, 8193, 4095, 16384, 3], ["bf16", "f16", "f32", "bf16", "bf16"]),
    ([20000, 1, 30001], ["f32", "f32", "f16"]),
    ([3] * 70 + [9000] + [2] * 70, ["bf16"] * 141),   # two launches' addresses
]


def inputs(sizes, dtypes, size, seed):
    rng = np.random.default_rng(seed)
    host = [to_storage(size * rng.standard_normal(n), d) for n, d in zip(sizes, dtypes)]
    return host, [to_f32(h, d) for h, d in zip(host, dtypes)]


def check_norm(values, norm):
    want = oracle.norm(values)
    assert abs(norm - want) <= 1.01 * U * want + 2.0 ** -149, (norm, want)


def check(dtypes, values, most, got, norm=None):
    want, n = oracle.clip(values, most)
    if norm is not None:
        check_norm(values, norm)
    for k, (g, w, d) in enumerate(zip(got, want, dtypes)):
        off = 2.01 * U * np.abs(w)
        off = off + (HALF_STEP[d] * 1.01 * (np.abs(w) + off) if d != "f32" else 0) + TINY[d]
        wrong = ~(np.abs(to_f32(g, d) - w) <= off)
        assert not wrong.any(), (k, d, int(wrong.sum()), to_f32(g, d)[wrong][0], w[wrong][0])
        if n <= most:
            assert np.array_equal(to_f32(g, d), values[k])
