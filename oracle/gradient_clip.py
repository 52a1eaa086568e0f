"""The norm of all gradients together and clipping, from the definition, in 64 bits. Test infrastructure only."""
import numpy as np


def norm(gradients):
    return np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in gradients))


def clip(gradients, most):
    n = norm(gradients)
    return [g.astype(np.float64) * min(1.0, most / (n + 1e-6)) for g in gradients], n
