"""Inputs and tolerances that the tests of orthogonalised updates share.

Tolerance. The iteration is a polynomial of degree 3125 whose worst-case error bound says nothing, so the measure of how far rounding
may take a result is the documented arithmetic itself, done by the oracle in numpy on the same input (oracle.muon.modelled): the
kernels' sums run in another order, so their errors are of that size but not those. Allowed: 4 times that error in the 2-norm, plus
1e-6 of the result (f32 sums of other lengths) and the rounding of the stored type; and no element further off than 8 times what
the 2-norm allows on average (errors are sums of many roundings; 8 standard deviations do not occur)."""
import numpy as np

from group_norm_cases import HALF_STEP, TINY, to_f32, to_storage  # noqa: F401
from oracle import muon as oracle

# rows, columns
SHAPES = [(1, 1), (1, 7), (9, 1), (3, 5), (8, 8), (31, 33), (64, 64), (65, 40), (130, 20), (40, 200), (128, 128), (129, 257)]


def runs_of(muon):
    return [int(r) for r in muon.description.split("\nruns ")[1].split("\n")[0].split(",")]


def matrix(shape, kind, seed):
    rng = np.random.default_rng(seed)
    r, c = shape
    if kind == "zero":
        return np.zeros(shape)
    if kind == "low_rank":   # one direction only, in noise of 1e-3
        return np.outer(rng.standard_normal(r), rng.standard_normal(c)) + 1e-3 * rng.standard_normal(shape)
    if kind == "one_entry":
        u = np.zeros(shape)
        u[r // 2, c // 2] = -3.0
        return u
    return rng.standard_normal(shape)


def check(got, u, dtype, split, steps=5, runs=None):
    """`got` f32, `u` the matrix as the kernel saw it, `runs` how its steps were taken."""
    want = oracle.orthogonalize(u, steps)
    off = np.linalg.norm(oracle.modelled(u, split, steps, runs) - want)
    size = np.linalg.norm(want)
    allowed = 4 * off + 1e-6 * size + HALF_STEP[dtype] * size + TINY[dtype] * np.sqrt(want.size)
    far = np.linalg.norm(got - want)
    assert far <= allowed, (far, allowed, size)
    each = 8 * (4 * off + 1e-6 * size) / np.sqrt(want.size) + HALF_STEP[dtype] * np.abs(want) * 1.01 + TINY[dtype]
    # (a matrix with few entries that are not zero has nothing to average over: all of the error may be in one of them)
    each = each if np.count_nonzero(want) > 64 else np.maximum(each, allowed)
    wrong = np.abs(got - want) > each
    assert not wrong.any(), (int(wrong.sum()), np.argwhere(wrong)[0], got[wrong][0], want[wrong][0])


def check_rounded_once(got, u, dtype, steps=5):
    """`got` is the exact result as well as its type holds it: each value off by half a step of the type, and by what five steps with
    f32 products are off (below 1e-5 of the result's norm) on top."""
    want = oracle.orthogonalize(u, steps)
    size = np.linalg.norm(want)
    far = np.linalg.norm(got - want)
    assert far <= (HALF_STEP[dtype] + 1e-5) * size + TINY[dtype] * np.sqrt(want.size), (far / size, HALF_STEP[dtype])


def f32_products(u, steps=5):
    """The definition in f32, products and all: what an implementation without matrix cores of 16 bits gives."""
    a, b, c = (np.float32(v) for v in oracle.COEFFICIENTS)
    tall = u.shape[0] > u.shape[1]
    x = np.ascontiguousarray(u.T if tall else u, np.float32)
    x = x / np.float32(np.sqrt((x.astype(np.float64) ** 2).sum()) + oracle.NORM_FLOOR)
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.T if tall else x


def spectra(shape, seed):
    """Matrices whose errors are magnified in different ways."""
    rng = np.random.default_rng(seed)
    r, c = shape
    noise, few = rng.standard_normal(shape), 0.35 * rng.standard_normal((r, 8)) @ rng.standard_normal((8, c))
    u, _, vt = np.linalg.svd(rng.standard_normal(shape), full_matrices=False)
    weak = np.where(np.arange(r)[:, None] % 2, noise, 1e-3 * noise)
    return {"noise": noise, "few directions": noise + few, "few strong directions": noise + 4 * few, "decades": (u * np.logspace(0, -3, min(shape))) @ vt, "weak rows": weak}
