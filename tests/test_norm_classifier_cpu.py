"""The graphs of harness/norm_classifier.py plan, and their gradients are those of the same model in 64 bits, with the oracle running the graphs
and the operators. No device."""
import numpy as np
import pytest

from harness import norm_classifier
from helium_amd.backend import Plan
from oracle import group_norm as oracle_norm
from oracle import helium_ir as oracle_ir
from norm_classifier_cases import BATCH, CHANNELS, CLASSES, EXTENT, GROUPS, batch, check_gradients


class Held:
    """What stands for a device tensor: its values."""

    def __init__(self, values):
        self.values = np.asarray(values, np.float32).reshape(-1).copy()

    @classmethod
    def from_numpy(cls, storage, dtype, length=None):
        assert dtype == "f32" and length in (None, np.asarray(storage).size)
        return cls(storage)

    def to_numpy(self):
        return self.values


class Norm:
    """GroupNorm's calls, by the oracle."""

    def __init__(self, batch, pixels, channels, groups, dtype, activation):
        self.shape, self.channels, self.groups, self.activation = (batch, pixels, channels), channels, groups, activation

    def forward(self, x, gamma, beta, y, mean, rstd):
        out = oracle_norm.forward(x.values.reshape(self.shape), gamma.values, beta.values, self.groups, self.activation, 1e-5)
        for to, v in zip((y, mean, rstd), out):
            to.values[:] = v.reshape(-1)

    def backward(self, dy, x, gamma, beta, mean, rstd, dx, dgamma, dbeta):
        at = (self.shape[0], self.groups)
        out = oracle_norm.backward(dy.values.reshape(self.shape), x.values.reshape(self.shape), gamma.values, beta.values, mean.values.reshape(at),
                                   rstd.values.reshape(at), self.activation)
        for to, v in zip((dx, dgamma, dbeta), out):
            to.values[:] = v.reshape(-1)


def run(graph, feeds):
    shapes = {n["id"]: n["shape"] for n in graph.nodes if n["id"] in feeds}
    host = {i: t.values.reshape(shapes[i]) for i, t in feeds.items()}
    graph.optimize()
    return {o: Held(v) for o, v in oracle_ir.plan_outputs(graph.nodes, host, Plan(graph).steps).items()}


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(norm_classifier, "Tensor", Held)
    monkeypatch.setattr(norm_classifier, "GroupNorm", Norm)
    monkeypatch.setattr(norm_classifier, "execute_graph", run)
    monkeypatch.setattr(norm_classifier.device, "synchronize", lambda: None)
    return norm_classifier.Classifier(BATCH, EXTENT, CHANNELS, GROUPS, CLASSES, dtype="f32")


def test_the_gradients(model):
    images, one_hot = batch()
    check_gradients(model, model.gradients(Held(images), Held(one_hot)), images, one_hot)
