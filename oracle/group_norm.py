"""Group norm with an activation and its gradients, from the definition, in 64 bits. Test infrastructure only."""
import numpy as np


def _spread(per_group, channels):
    """[batch, groups] -> [batch, 1, channels]"""
    return np.repeat(per_group, channels // per_group.shape[1], axis=1)[:, None, :]


def statistics(x, groups, epsilon):
    """x [batch, pixels, channels] -> mean and 1 / sqrt(variance + epsilon), both [batch, groups]."""
    n, p, c = x.shape
    v = x.astype(np.float64).reshape(n, p, groups, c // groups)
    mean = v.mean(axis=(1, 3))
    variance = ((v - mean[:, None, :, None]) ** 2).mean(axis=(1, 3))
    return mean, 1.0 / np.sqrt(variance + epsilon)


def _sigmoid(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z))


def activate(z, activation):
    return {"none": lambda: z, "relu": lambda: np.maximum(z, 0.0), "silu": lambda: z * _sigmoid(z)}[activation]()


def slope(z, activation):
    s = _sigmoid(z)
    return {"none": lambda: np.ones_like(z), "relu": lambda: (z > 0).astype(np.float64), "silu": lambda: s + z * s * (1 - s)}[activation]()


def normalised(x, mean, rstd, gamma, beta):
    """xh and z = gamma * xh + beta."""
    c = x.shape[2]
    xh = (x.astype(np.float64) - _spread(mean.astype(np.float64), c)) * _spread(rstd.astype(np.float64), c)
    return xh, xh * gamma.astype(np.float64) + beta.astype(np.float64)


def forward(x, gamma, beta, groups, activation, epsilon):
    mean, rstd = statistics(x, groups, epsilon)
    return activate(normalised(x, mean, rstd, gamma, beta)[1], activation), mean, rstd


def backward(dy, x, gamma, beta, mean, rstd, activation):
    """dx, dgamma, dbeta; mean and rstd count as the statistics of x."""
    n, p, c = x.shape
    groups = mean.shape[1]
    xh, z = normalised(x, mean, rstd, gamma, beta)
    dz = dy.astype(np.float64) * slope(z, activation)
    flow = dz * gamma.astype(np.float64)
    per_group = lambda v: _spread(v.reshape(n, p, groups, c // groups).mean(axis=(1, 3)), c)  # noqa: E731
    dx = _spread(rstd.astype(np.float64), c) * (flow - per_group(flow) - xh * per_group(flow * xh))
    return dx, (dz * xh).sum(axis=(0, 1)), dz.sum(axis=(0, 1))
