"""Orthogonalised updates by Newton-Schulz products and the optimizer step built on them, from the definition, in 64 bits; and the
arithmetic that the kernels document, in 32 bits, as a measure of how far rounding may take them. Test infrastructure only."""
import numpy as np

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NORM_FLOOR = 1e-7


def orthogonalize(u, steps=5):
    a, b, c = COEFFICIENTS
    x = np.asarray(u, np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (np.sqrt((x * x).sum()) + NORM_FLOOR)
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.T if tall else x


def singular_values_after(s, steps=5):
    """What the iteration makes of singular values of a matrix of norm 1."""
    a, b, c = COEFFICIENTS
    for _ in range(steps):
        s = a * s + b * s ** 3 + c * s ** 5
    return s


def step(gradient, momentum, weight, learning_rate, mu, weight_decay, nesterov, steps=5):
    """New weight and new momentum."""
    g, w = np.asarray(gradient, np.float64), np.asarray(weight, np.float64)
    m = mu * np.asarray(momentum, np.float64) + g
    o = orthogonalize(g + mu * m if nesterov else m, steps)
    return (1 - learning_rate * weight_decay) * w - learning_rate * np.sqrt(max(1.0, g.shape[0] / g.shape[1])) * o, m


def _parts(x, scale, count):
    high = (x * np.float32(scale)).astype(np.float16).astype(np.float32)
    low = (x * np.float32(scale) - high).astype(np.float16).astype(np.float32)
    return high, low if count == 2 else np.zeros_like(low), (high + low) / np.float32(scale)


def _product(p, q):
    return p[0] @ q[0].T + (p[0] @ q[1].T + p[1] @ q[0].T)


def modelled(u, split, steps=5, runs=None):
    """orthogonalize() with operands of one or two f16 parts and f32 sums. `runs`: how many steps at a time are taken on the
    smaller side (A = X X^T, A <- Q A Q with Q = a I + b A + c A A, X <- the product of the Q's times X); one by one unless given."""
    a, b, c = (np.float32(v) for v in COEFFICIENTS)
    sx, sa, sq = np.float32(4096), np.float32(8192), [None, np.float32(8192), np.float32(4096), np.float32(1024)]
    count = 2 if split else 1
    x = np.asarray(u, np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = (x / (np.sqrt((x * x).sum()) + NORM_FLOOR)).astype(np.float32)
    turned = lambda p: [np.ascontiguousarray(v.T) for v in p[:2]]  # noqa: E731
    symmetric = lambda v: np.tril(v) + np.tril(v, -1).T  # noqa: E731
    assert sum(runs or [1] * steps) == steps
    for run in runs or [1] * steps:
        xp = _parts(x, sx, count)
        ap = _parts(symmetric(_product(xp, xp) / (sx * sx)), sa, count)
        for j in range(run):
            bp = _parts(symmetric(b * ap[2] + c * _product(ap, ap) / (sa * sa)), sa, count)
            if j == 0:
                qp = bp
            elif j == 1:
                q = symmetric(a * a * np.eye(len(x), dtype=np.float32) + a * qp[2] + a * bp[2] + _product(bp, qp) / (sa * sa))
                qp = _parts(q, sq[2], count)
            else:
                qp = _parts(symmetric(a * qp[2] + _product(bp, qp) / (sa * sq[j])), sq[j + 1], count)
            if j + 1 < run:
                cp = _parts(symmetric(a * ap[2] + _product(bp, ap) / (sa * sa)), sa, count)
                ap = _parts(symmetric(a * cp[2] + _product(cp, bp) / (sa * sa)), sa, count)
        x = a * xp[2] + _product(bp, turned(xp)) / (sa * sx) if run == 1 else _product(qp, turned(xp)) / (sq[run] * sx)
    x = _parts(x, sx, 2)[2]
    return x.T if tall else x
