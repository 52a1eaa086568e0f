"""The classifier of harness/norm_classifier.py with its gradients clipped: each step is held to what 64 bits make of the parameters it began with."""
import numpy as np
import pytest

from harness import autodiff as ad
from harness import norm_classifier
from helium_amd.backend import Tensor
from norm_classifier_cases import BATCH, CHANNELS, CLASSES, EXTENT, GROUPS, batch, close, reference, values
from oracle import gradient_clip as oracle
from oracle import muon as oracle_muon

pytestmark = pytest.mark.gpu

RATE, MU, DECAY, OTHER = 0.02, 0.95, 0.01, 0.1


@pytest.mark.parametrize("max_norm", [0.05, 1e3])
def test_two_steps(max_norm):
    model = norm_classifier.Classifier(BATCH, EXTENT, CHANNELS, GROUPS, CLASSES, dtype="f32", learning_rate=RATE, momentum=MU, weight_decay=DECAY,
                                       other_rate=OTHER, max_norm=max_norm)
    images, one_hot = batch()
    image, labels = Tensor.from_numpy(ad._to_storage(images, "f32"), "f32", images.size), Tensor.from_numpy(one_hot, "f32", one_hot.size)
    for _ in range(2):
        before = values(model)
        momenta = [s.momentum.to_numpy().reshape(s.filter_shape) for s in model.stages]
        want_loss, want = reference(*before, images, one_hot)
        n = len(model.stages)
        # (in the model's order: filters, then gamma and beta of each stage, then the linear layer)
        want = want[:n] + [g for k in range(n) for g in (want[n + k], want[2 * n + k])] + want[3 * n:]
        clipped, norm = oracle.clip(want, max_norm)
        loss = model.step(image, labels)
        assert abs(loss - want_loss) <= 1e-5 * abs(want_loss)
        # gradients are off by 1e-4 of their norm at most (test_norm_classifier_gpu.py), their norm together by no more
        assert abs(float(model.norm.to_numpy()[0]) - norm) <= 1e-4 * norm
        assert (norm > max_norm) == (max_norm < 1)
        for got, w in zip(model.all_gradients(), clipped):
            close(got.to_numpy(), w, 2e-4, "a clipped gradient")
        filters, gammas, betas, linear = values(model)
        for k, s in enumerate(model.stages):
            weight, momentum = oracle_muon.step(s.filter_gradient.to_numpy().reshape(s.filter_shape), momenta[k], before[0][k].reshape(s.filter_shape),
                                                RATE, MU, DECAY, True)
            close(s.momentum.to_numpy(), momentum, 1e-6, f"momentum {k}")
            close(filters[k], weight, 1e-6, f"filter {k}")
            # (differences of parameters near one, each rounded to 2^-24: of a step of OTHER times the gradient)
            for new, old, g in ((gammas[k], before[1][k], clipped[n + 2 * k]), (betas[k], before[2][k], clipped[n + 2 * k + 1])):
                close(new - old, -OTHER * g, 1e-3 + 2.0 ** -23 * np.sqrt(g.size) / (OTHER * np.linalg.norm(g)), f"stage {k}")
        close(linear - before[3], -OTHER * clipped[-1].reshape(before[3].shape), 1e-3 + 2.0 ** -23 * np.linalg.norm(before[3]) / (OTHER * np.linalg.norm(clipped[-1])), "linear layer")
