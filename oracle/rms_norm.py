"""Root-mean-square norm over rows and its gradients, from the definition, in 64 bits. Test infrastructure only."""
import numpy as np


def rstd(h, epsilon):
    """h [rows, columns] -> 1 / sqrt(mean of squares + epsilon), [rows]."""
    h = h.astype(np.float64)
    return 1.0 / np.sqrt((h * h).mean(axis=1) + epsilon)


def forward(h, gamma, epsilon):
    r = rstd(h, epsilon)
    return h.astype(np.float64) * r[:, None] * gamma.astype(np.float64), r


def backward(dy, h, gamma, rstd, dh=None):
    """The gradients of h and gamma; rstd counts as that of h."""
    xh = h.astype(np.float64) * rstd.astype(np.float64)[:, None]
    dy = dy.astype(np.float64)
    flow = dy * gamma.astype(np.float64)
    dx = rstd.astype(np.float64)[:, None] * (flow - xh * (flow * xh).mean(axis=1, keepdims=True))
    return dx if dh is None else dx + dh.astype(np.float64), (dy * xh).sum(axis=0)
