"""Inputs, tolerances and checks that the tests of rms norm and of quantised rows share.

Tolerances. u = 2^-24. A lane adds up at most 64 squares, and a tree or 16 waves in a row join the lanes: no sum of a row is a chain of
more than DEPTH additions. A result that is stored in 16 bits is off by half a step of that type on top."""
import numpy as np

from group_norm_cases import HALF_STEP, TINY, U, to_f32, to_storage
from oracle import rms_norm as oracle

DEPTH = 96
EPSILON = 1e-5

# rows, columns
SHAPES = [(1, 1), (3, 2), (5, 3), (2, 7), (9, 8), (70, 21), (3, 64), (17, 100), (4, 256), (33, 257), (6, 510), (2, 1203), (3, 2056), (1, 4096), (2, 4100)]
LARGE = [(1, 32768), (2, 32767), (1500, 1203), (3000, 512), (1100, 4096), (1200, 2867), (5000, 64), (20000, 20), (1030, 8192), (1027, 12290)]
# x's type, the residual's
TYPES = [("f32", None), ("f32", "f32"), ("bf16", None), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]


def inputs(rows, columns, dtype, residual, param_dtype, seed):
    """Storage arrays by name, and the same as f32; h and rstd as a forward pass leaves them."""
    rng = np.random.default_rng(seed)
    size = np.exp(0.5 * rng.standard_normal(columns))
    stream = residual or dtype
    host = {"x": to_storage(rng.standard_normal((rows, columns)) * size, dtype), "dy": to_storage(rng.standard_normal((rows, columns)), dtype),
            "gamma": to_storage(1 + 0.3 * rng.standard_normal(columns), param_dtype)}
    types = {"x": dtype, "dy": dtype, "gamma": param_dtype}
    if residual:
        host["residual"] = to_storage(2 * rng.standard_normal((rows, columns)), residual)
        host["dh"] = to_storage(rng.standard_normal((rows, columns)), residual)
        types["residual"] = types["dh"] = residual
    v = {k: to_f32(a, types[k]) for k, a in host.items()}
    # the sum in f32, rounded to the stream's type
    host["h"] = to_storage(v["x"] + v["residual"], stream) if residual else host["x"]
    v["h"] = to_f32(host["h"], stream)
    host["rstd"] = v["rstd"] = oracle.rstd(v["h"], EPSILON).astype(np.float32)
    return host, v


def within(got, want, off, what):
    wrong = ~(np.abs(got - want) <= off)
    assert not wrong.any(), (what, int(wrong.sum()), np.argwhere(wrong)[0], got[wrong][0], want[wrong][0], np.broadcast_to(off, want.shape)[wrong][0])


def rounded(off, want, dtype):
    return off + HALF_STEP[dtype] * 1.01 * (np.abs(want) + off) + TINY[dtype]


def check_forward(dtype, v, y, rstd=None):
    want, wrstd = oracle.forward(v["h"], v["gamma"], EPSILON)
    # the sum is off by DEPTH u of itself, its root by half that; the root, the division and the mean round
    if rstd is not None:
        within(rstd, wrstd, (DEPTH / 2 + 4) * U * wrstd, "rstd")
    within(y, want, rounded((DEPTH / 2 + 8) * U * np.abs(want), want, dtype), "y")


def check_quantized_norm(v, q, scales):
    columns = v["h"].shape[1]
    want, _ = oracle.forward(v["h"], v["gamma"], EPSILON)
    most = np.abs(want).max(axis=1)
    within(scales, most / 127, (DEPTH / 2 + 12) * U * most / 127, "scales")
    # h gamma, its reciprocal's and the quotient's rounding: 127 (1 + 4 u) at most, so that a whole number is half a step and 127 * 4 u off
    quotient = 127 * want / np.where(most > 0, most, 1)[:, None]
    within(q[:, :columns].astype(np.float64), quotient, 0.5 + 127 * 6 * U, "q")
    assert np.abs(q[:, :columns].astype(int)).max() <= 127 and not q[:, columns:].any()


def check_backward(dtype, residual, v, dx, dresidual, dgamma, rows_per_block):
    """rows_per_block: how many rows a workgroup's lane adds up for dgamma."""
    dh = v.get("dh") if dx is None or residual else None
    want, wgamma = oracle.backward(v["dy"], v["h"], v["gamma"], v["rstd"], dh)
    xh = np.abs(v["h"].astype(np.float64) * v["rstd"][:, None])
    dy, gamma, rstd = np.abs(v["dy"].astype(np.float64)), np.abs(v["gamma"].astype(np.float64)), v["rstd"].astype(np.float64)[:, None]
    mean = (dy * gamma * xh).mean(axis=1, keepdims=True)
    off = rstd * (3 * U * dy * gamma + (DEPTH + 8) * U * xh * mean) + 3 * U * np.abs(want) + (U * np.abs(v["dh"]) if dh is not None else 0)
    if dx is not None:
        within(dx, want, rounded(off, want, dtype), "dx")
    if dresidual is not None:
        within(dresidual, want, rounded(off, want, residual), "dresidual")
    # a lane's rows, the lanes and waves side by side (10 at most), then 16 chains over 512 workgroups
    depth = rows_per_block + 10 + 32 + 16 + 4
    within(dgamma, wgamma, depth * U * (dy * xh).sum(axis=0), "dgamma")


# rows, columns, x's type, the residual's, epsilon: several rows to a wave, to a workgroup, one row to a workgroup
BEYOND = [(9, 20, "f32", None, 1e-5), (70, 21, "bf16", "f32", 0.0), (3, 64, "f32", "f32", 0.0), (7, 300, "bf16", "bf16", 1e-5), (9, 700, "f32", None, 0.0),
          (5, 1203, "bf16", "f32", 0.0), (4, 1203, "f32", "f32", 1e-5), (5, 2056, "bf16", None, 0.0)]


def beyond(rows, columns, dtype, residual, epsilon, seed):
    """Rows whose squares or sums of squares f32 cannot hold, too large and, without an epsilon, too small ones, between ordinary rows; gamma is f32."""
    host, v = inputs(rows, columns, dtype, residual, "f32", seed)
    sizes = np.array([1, 3e17, 1, 1e19, 1e25, 1e37] if epsilon else [1, 1e-15, 3e18, 1e-25, 1e-34, 1, 1e36])[np.arange(rows) % (6 if epsilon else 7), None]
    for k, t in (("x", dtype), ("residual", residual)):
        if t:
            host[k] = to_storage(v[k] * sizes, t)
            v[k] = to_f32(host[k], t)
    stream = residual or dtype
    host["h"] = to_storage(v["x"] + v["residual"], stream) if residual else host["x"]
    v["h"] = to_f32(host["h"], stream)
    assert np.isfinite(v["h"]).all() and (np.abs(v["h"]).max(axis=1) > 0).all()
    return host, v


def check_beyond(dtype, v, epsilon, y, rstd):
    """As check_forward has it: the factor that the values are taken times is a power of two."""
    want, wrstd = oracle.forward(v["h"], v["gamma"], epsilon)
    assert wrstd.min() > 2.0 ** -125 and wrstd.max() < 2.0 ** 126
    within(rstd, wrstd, (DEPTH / 2 + 4) * U * wrstd, "rstd")
    within(y, want, rounded((DEPTH / 2 + 8) * U * np.abs(want), want, dtype), "y")


def check_quantized_beyond(v, epsilon, q, scales):
    want, _ = oracle.forward(v["h"], v["gamma"], epsilon)
    most = np.abs(want).max(axis=1)
    within(scales, most / 127, (DEPTH / 2 + 12) * U * most / 127, "scales")
    within(q[:, :v["h"].shape[1]].astype(np.float64), 127 * want / most[:, None], 0.5 + 127 * 6 * U, "q")
