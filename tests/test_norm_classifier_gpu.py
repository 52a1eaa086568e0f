"""Group norm and Muon in a training step: harness/norm_classifier.py against the same model in 64 bits (torch's derivatives on the
CPU for everything but the optimizer's orthogonalised update, which is the oracle's)."""
import numpy as np
import pytest

from harness import autodiff as ad
from harness import norm_classifier
from helium_amd.backend import Tensor
from oracle import muon as oracle_muon
from norm_classifier_cases import BATCH, CHANNELS, CLASSES, EXTENT, GROUPS, batch, check_gradients, close, reference, values

pytestmark = pytest.mark.gpu

RATE, MU, DECAY, OTHER = 0.02, 0.95, 0.01, 0.1


def make(dtype, **more):
    model = norm_classifier.Classifier(BATCH, EXTENT, CHANNELS, GROUPS, CLASSES, dtype=dtype, learning_rate=RATE, momentum=MU, weight_decay=DECAY,
                                       other_rate=OTHER, **more)
    images, one_hot = batch()
    return (model, images, one_hot, Tensor.from_numpy(ad._to_storage(images, dtype), dtype, images.size),
            Tensor.from_numpy(one_hot, "f32", one_hot.size))


def test_the_gradients_of_f32():
    model, images, one_hot, image, labels = make("f32")
    check_gradients(model, model.gradients(image, labels), images, one_hot)


def test_three_steps_of_f32():
    """Each step is held to what 64 bits make of the parameters it began with and the gradients it took."""
    model, images, one_hot, image, labels = make("f32")
    for _ in range(3):
        before = values(model)
        momenta = [s.momentum.to_numpy().reshape(s.filter_shape) for s in model.stages]
        want_loss, want = reference(*before, images, one_hot)
        loss = model.step(image, labels)
        assert abs(loss - want_loss) <= 1e-5 * abs(want_loss)
        filters, gammas, betas, linear = values(model)
        n = len(model.stages)
        for k, s in enumerate(model.stages):
            # (the gradient as the device has it: an orthogonalised update may turn on its smallest singular values)
            weight, momentum = oracle_muon.step(s.filter_gradient.to_numpy().reshape(s.filter_shape), momenta[k], before[0][k].reshape(s.filter_shape),
                                                RATE, MU, DECAY, True)
            close(s.momentum.to_numpy(), momentum, 1e-6, f"momentum {k}")
            # (an update is RATE * 0.7 .. 1.2 per singular value, next to weights of about 1: 2e-5 of it shrinks to 1e-6)
            close(filters[k], weight, 1e-6, f"filter {k}")
            close(gammas[k] - before[1][k], -OTHER * want[n + k], 1e-3, f"gamma {k}")
            close(betas[k] - before[2][k], -OTHER * want[2 * n + k], 1e-3, f"beta {k}")
        close(linear - before[3], -OTHER * want[-1], 1e-3, "linear layer")


def trained(filters, gammas, betas, linear, images, one_hot, steps):
    """The losses of that many steps in 64 bits."""
    n, losses, momenta = len(filters), [], [np.zeros((f.shape[0], f[0].size)) for f in filters]
    for _ in range(steps):
        loss, g = reference(filters, gammas, betas, linear, images, one_hot)
        losses.append(loss)
        new = [oracle_muon.step(g[k].reshape(momenta[k].shape), momenta[k], filters[k].reshape(momenta[k].shape), RATE, MU, DECAY, True) for k in range(n)]
        momenta = [m for _, m in new]
        filters = [w.reshape(f.shape) for (w, _), f in zip(new, filters)]
        gammas, betas = [v - OTHER * d for v, d in zip(gammas, g[n:])], [v - OTHER * d for v, d in zip(betas, g[2 * n:])]
        linear = linear - OTHER * g[-1]
    return losses


@pytest.mark.parametrize("dtype, precision", [("bf16", "f32_f32"), ("f16", "f16_f32"), ("bf16", "f16_f32")])
def test_it_learns(dtype, precision):
    """Four images of random labels are learnt as in 64 bits, and two models of one seed go the same way to the last bit. An activation passes half a
    dozen roundings of at most 2^-8 on its way to the loss, and the path's own errors are of the same order: 5% of the loss."""
    losses = []
    for _ in range(2):
        model, images, one_hot, image, labels = make(dtype, precision=precision)
        start = values(model)
        losses.append([model.step(image, labels) for _ in range(12)])
    want = trained(*start, images, one_hot, 12)
    assert losses[0] == losses[1]
    assert all(abs(got - w) <= 0.05 * w for got, w in zip(losses[0], want)), (losses[0], want)
    assert all(b < a for a, b in zip(losses[0], losses[0][1:])), losses[0]
