"""The model of harness/norm_classifier.py in 64 bits, with torch's derivatives on the CPU, and the comparison of what a model took with it."""
import numpy as np
import torch

from harness import norm_classifier

BATCH, EXTENT, CHANNELS, GROUPS, CLASSES = 4, 9, [5, 16, 20], 4, 7  # (data gradients of 16 bits take input channels in eights)


def batch():
    rng = np.random.default_rng(3)
    images = rng.standard_normal([BATCH, EXTENT, EXTENT, CHANNELS[0]]).astype(np.float32)
    return images, np.eye(CLASSES, dtype=np.float32)[rng.integers(0, CLASSES, BATCH)]


def reference(filters, gammas, betas, linear, images, one_hot):
    """The loss and all gradients in 64 bits."""
    leaves = [torch.tensor(np.asarray(v, np.float64), requires_grad=True) for v in (*filters, *gammas, *betas, linear)]
    n = len(filters)
    x = torch.tensor(images.astype(np.float64))
    for k in range(n):
        x = torch.nn.functional.conv2d(x.permute(0, 3, 1, 2), leaves[k].permute(0, 3, 1, 2), padding=1).permute(0, 2, 3, 1)
        c = x.shape[3]
        g = x.reshape(BATCH, EXTENT * EXTENT, GROUPS, c // GROUPS)
        centred = g - g.mean((1, 3), keepdim=True)
        x = (centred / torch.sqrt((centred ** 2).mean((1, 3), keepdim=True) + 1e-5)).reshape(x.shape) * leaves[n + k] + leaves[2 * n + k]
        x = x * torch.sigmoid(x) if k == norm_classifier.SILU_STAGE else torch.relu(x)
    logits = x.mean((1, 2)) @ leaves[-1]
    loss = -(torch.log_softmax(logits, 1) * torch.tensor(one_hot.astype(np.float64))).sum() / BATCH
    loss.backward()
    return loss.item(), [v.grad.numpy() for v in leaves]


def values(model):
    """The filters, gammas, betas and the linear layer as they are."""
    shapes = [(s.filter_shape[0], 3, 3, s.filter_shape[1] // 9) for s in model.stages]
    return ([s.filter.to_numpy().reshape(f) for s, f in zip(model.stages, shapes)], [s.gamma.to_numpy() for s in model.stages],
            [s.beta.to_numpy() for s in model.stages], model.linear.to_numpy().reshape(CHANNELS[-1], CLASSES))


def close(got, want, rel, what):
    got, want = np.asarray(got, np.float64).reshape(-1), np.asarray(want, np.float64).reshape(-1)
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= rel, f"{what}: {off:.2e} of its norm, {rel:.0e} allowed"


def check_gradients(model, loss, images, one_hot):
    """Of an f32 model. Sums of up to 4 * 81 products in each of four layers: 1e-4 of a gradient's norm is over a hundred roundings of each
    value."""
    want_loss, want = reference(*values(model), images, one_hot)
    assert abs(loss - want_loss) <= 1e-5 * abs(want_loss)
    n = len(model.stages)
    for k, s in enumerate(model.stages):
        close(s.filter_gradient.to_numpy(), want[k], 1e-4, f"filter {k}")
        close(s.d_gamma.to_numpy(), want[n + k], 1e-4, f"gamma {k}")
        close(s.d_beta.to_numpy(), want[2 * n + k], 1e-4, f"beta {k}")
