"""Inputs, tolerances and runners that the group norm tests share.

Tolerances. u = 2^-24. A sum of f32 values here is a chain of at most a few hundred additions (a thread's pixels and channels,
then the workgroup's rows, then the parts of a sample, then the samples), so its error is at most DEPTH u times the sum of the
absolute values. exp and the reciprocal in a sigmoid are off by a few u, and exp by |z| u more, the rounding of its argument.
A result that is stored in 16 bits is off by half a step of that type on top."""
import numpy as np

from oracle import group_norm as oracle
from oracle import numerics as nm

U = 2.0 ** -24
DEPTH = 1024
HALF_STEP = {"f32": U, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # 24, 8 and 11 significant bits
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -24}
EPSILON = 1e-5

# batch, pixels, channels, groups
SHAPES = [
    (1, 1, 1, 1),         # one value: variance zero
    (1, 1, 64, 8),        # one pixel
    (2, 49, 32, 8),
    (3, 37, 30, 5),       # six channels to a group, rows of no whole vector
    (2, 65, 21, 7),       # odd channels: single elements
    (2, 100, 48, 16),     # three channels to a group: vectors span groups
    (1, 130, 40, 40),     # every channel a group
    (2, 33, 264, 1),      # one group of all channels
    (5, 64, 128, 32),
    (1, 7, 2560, 4),      # more vectors in a pixel than threads stand side by side
    (1, 3000, 16, 4),     # several workgroups along the pixels
    (2, 2049, 24, 6),     # the last of them with one pixel
]

# wide groups, that no workgroup holds a pixel of with one vector to a thread
WIDE = [((1, 10, 10244, 1), "f32"), ((1, 3, 12288, 1), "f16"), ((2, 2, 16384, 1), "bf16"),
        ((1, 5, 16380, 4), "bf16"), ((1, 2, 16001, 1), "f32")]
# the widest of them: one vector of each column is all that a thread holds
WIDEST = [((1, 10, 16384, 1), "f32"), ((4, 64, 15368, 1), "f32"), ((1, 10, 16383, 1), "f32"), ((1, 10, 16129, 1), "bf16")]


def to_storage(x, dtype):
    x = np.asarray(x, np.float32)
    return x if dtype == "f32" else nm.f32_to_bf16_bits(x) if dtype == "bf16" else x.astype(np.float16).view(np.uint16)


def to_f32(bits, dtype):
    return bits if dtype == "f32" else nm.bf16_bits_to_f32(bits) if dtype == "bf16" else bits.view(np.float16).astype(np.float32)


def inputs(shape, dtype, param_dtype, activation, seed):
    """Storage arrays by name, and the same as f32. The statistics are f32 and belong to x but for the pixels that are moved out
    of the neighbourhood of relu's corner, where 32 and 64 bits may not agree on the side."""
    n, p, c, groups = shape
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, p, c)) * (0.5 + np.abs(rng.standard_normal(c))) + 2.0 * rng.standard_normal(c)
    host = {"x": to_storage(x, dtype), "dy": to_storage(rng.standard_normal((n, p, c)), dtype),
            "gamma": to_storage(1 + 0.3 * rng.standard_normal(c), param_dtype), "beta": to_storage(0.3 * rng.standard_normal(c), param_dtype)}
    values = lambda: {k: to_f32(v, param_dtype if k in ("gamma", "beta") else dtype) for k, v in host.items()}  # noqa: E731
    mean, rstd = (v.astype(np.float32) for v in oracle.statistics(values()["x"], groups, EPSILON))
    for _ in range(8):
        v = values()
        z = oracle.normalised(v["x"], mean, rstd, v["gamma"], v["beta"])[1]
        near = np.abs(z) < 1e-3
        if activation != "relu" or not near.any():
            break
        host["x"] = to_storage(np.where(near, v["x"] + 0.25 * (1 + np.abs(v["x"])), v["x"]), dtype)
    v = values()
    assert activation != "relu" or (np.abs(oracle.normalised(v["x"], mean, rstd, v["gamma"], v["beta"])[1]) > 1e-4).all()
    return host, v, mean, rstd


def check_forward(shape, dtype, activation, v, y, mean, rstd):
    n, p, c, groups = shape
    want, wmean, wrstd = oracle.forward(v["x"], v["gamma"], v["beta"], groups, activation, EPSILON)
    size = oracle.statistics(np.abs(v["x"]), groups, EPSILON)[0]          # mean |x| per group
    if mean is not None:
        # the variance: relative to itself, and the square of the mean's error on top
        mean_off = DEPTH * U * size
        variance = wrstd ** -2.0 - EPSILON
        assert (np.abs(mean - wmean) <= mean_off).all(), np.abs(mean - wmean).max()
        assert (np.abs(rstd / wrstd - 1) <= 4 * U + DEPTH * U * variance * wrstd ** 2 + 0.5 * mean_off ** 2 * wrstd ** 2 + 2 * U).all()
    xh, z = oracle.normalised(v["x"], wmean, wrstd, v["gamma"], v["beta"])
    spread = lambda a: oracle._spread(a, c)  # noqa: E731
    gamma = np.abs(v["gamma"].astype(np.float64))
    off_z = gamma * spread(wrstd) * (DEPTH * U * spread(size) + 2 * U * np.abs(v["x"])) + np.abs(xh) * gamma * (DEPTH + 8) * U + 4 * U * np.abs(z)
    off = 1.1 * off_z + (np.abs(want) * (16 + 2 * np.abs(z)) * U if activation == "silu" else 0)
    off = off + HALF_STEP[dtype] * 1.01 * (np.abs(want) + off) + TINY[dtype]
    wrong = np.abs(y - want) > off
    assert not wrong.any(), (int(wrong.sum()), np.argwhere(wrong)[0], y[wrong][0], want[wrong][0])


def check_backward(shape, dtype, activation, v, mean, rstd, dx, dgamma, dbeta):
    n, p, c, groups = shape
    want, wgamma, wbeta = oracle.backward(v["dy"], v["x"], v["gamma"], v["beta"], mean, rstd, activation)
    gamma, dy = np.abs(v["gamma"].astype(np.float64)), np.abs(v["dy"].astype(np.float64))
    spread = lambda a: oracle._spread(np.asarray(a, np.float64), c)  # noqa: E731
    xh, z = oracle.normalised(v["x"], mean, rstd, v["gamma"], v["beta"])
    off_xh = 3 * U * spread(rstd) * (np.abs(v["x"]) + np.abs(spread(mean)))
    off_z = gamma * off_xh + 3 * U * (np.abs(z) + np.abs(xh) * gamma)
    off_dz = dy * ((24 + 2 * np.abs(z)) * U + off_z) if activation == "silu" else 2 * U * dy   # (|slope| and its own slope are below 1.1)
    size = 1.1 * dy
    group_mean = lambda a: spread(a.reshape(n, p, groups, c // groups).mean(axis=(1, 3)))  # noqa: E731
    terms = gamma * size + group_mean(gamma * size) + np.abs(xh) * group_mean(gamma * size * np.abs(xh))
    offs = gamma * off_dz + group_mean(gamma * off_dz) + np.abs(xh) * group_mean(gamma * (off_dz * np.abs(xh) + size * off_xh)) + off_xh * group_mean(gamma * size * np.abs(xh))
    off = spread(rstd) * (DEPTH * U * terms + offs)
    off = off + HALF_STEP[dtype] * 1.01 * (np.abs(want) + off) + TINY[dtype]
    wrong = np.abs(dx - want) > off
    assert not wrong.any(), (int(wrong.sum()), np.argwhere(wrong)[0], dx[wrong][0], want[wrong][0], off[wrong][0])
    total = lambda a: a.sum(axis=(0, 1))  # noqa: E731
    assert (np.abs(dbeta - wbeta) <= DEPTH * U * total(size) + total(off_dz)).all()
    assert (np.abs(dgamma - wgamma) <= DEPTH * U * total(size * np.abs(xh)) + total(off_dz * np.abs(xh) + size * off_xh)).all()
