"""A small image classifier with group norm whose filters are trained with Muon: what the two operators look like beside the graphs
that `execute_graph` runs.

    image -> [3x3 convolution -> group norm -> silu or relu] x stages -> average over pixels -> linear layer -> cross-entropy

The convolutions, the loss and their gradients are recorded helium-ir graphs; group norm (forward and backward) and the optimizer
step of the filters are calls on the tensors those graphs read and write. Group norm, unlike the batch norm of harness/resnet.py, has
no running statistics and one behaviour in training and use, and its gradients here are its own rules instead of the some sixty recorded ops.
The other parameters (gamma, beta, the linear layer) are trained by plain gradient steps, as a matrix's orthogonalised update
has no meaning for vectors.

Everything that one step makes stays on the device; only the loss comes back. `execute_graph` works on streams of the library's own, the operators on the
caller's (here the default one), so the two wait for each other with device.synchronize() at every change.
"""
import numpy as np

from helium_amd import GroupNorm, Muon, device
from helium_amd.backend import Tensor, execute_graph

from . import autodiff as ad

SILU_STAGE = 0  # the first stage takes silu, the others relu


class Stage:
    """One convolution and its group norm."""

    def __init__(self, rng, batch, extent, in_channels, out_channels, groups, dtype, activation, first):
        self.dtype, self.first = dtype, first
        pixels = extent * extent
        conv = {"in_channels": in_channels, "out_channels": out_channels, "kernel_size": [3, 3]}
        image, flow, filt = [batch, extent, extent, in_channels], [batch, extent, extent, out_channels], [out_channels, 3, 3, in_channels]
        self.norm = GroupNorm(batch, pixels, out_channels, groups, dtype, activation=activation)
        self.filter_shape = (out_channels, 9 * in_channels)

        # y = conv(x, filter)
        G = ad.Graph()
        x, w = ad.Raw(G, G.g.new_input(image, dtype)), ad.Raw(G, G.g.new_input(filt, "f32"))
        self.forward_graph, self.forward_in = G.g, (x.node, w.node)
        self.forward_out = G.g.new_output(x.conv2d(w.into_data_type(dtype), conv).node)

        # the filter's gradient and, but for the first stage, the image's
        G = ad.Graph()
        f, x = ad.Raw(G, G.g.new_input(flow, dtype)), ad.Raw(G, G.g.new_input(image, dtype))
        self.backward_graph, self.backward_in = G.g, (f.node, x.node)
        self.d_filter = G.g.new_output(f.conv2d_backward_filter(x, conv).into_data_type(dtype).node)
        if not first:
            w = ad.Raw(G, G.g.new_input(filt, "f32"))
            self.backward_in += (w.node,)
            self.d_image = G.g.new_output(f.conv2d_backward_data(w.into_data_type(dtype), conv, [extent, extent]).into_data_type(dtype).node)

        def tensor(values, kind="f32"):
            return Tensor.from_numpy(ad._to_storage(values, kind), kind, int(np.asarray(values).size))

        weights = rng.standard_normal(filt) / np.sqrt(9 * in_channels)
        self.filter, self.momentum = tensor(weights), tensor(np.zeros(filt))
        self.gamma, self.beta = tensor(np.ones(out_channels)), tensor(np.zeros(out_channels))
        # what the calls write: the activation, the statistics its gradient reads, and the gradients
        self.out, self.flow = tensor(np.zeros(flow), dtype), tensor(np.zeros(flow), dtype)
        self.mean, self.rstd = tensor(np.zeros([batch, groups])), tensor(np.zeros([batch, groups]))
        self.d_gamma, self.d_beta = tensor(np.zeros(out_channels)), tensor(np.zeros(out_channels))

    def forward(self, image):
        self.image = image
        self.conv_out = execute_graph(self.forward_graph, dict(zip(self.forward_in, (image, self.filter))))[self.forward_out]
        device.synchronize()
        self.norm.forward(self.conv_out, self.gamma, self.beta, self.out, self.mean, self.rstd)
        device.synchronize()
        return self.out

    def backward(self, d_out):
        """Sets the parameters' gradients; returns the image's, None for the first stage."""
        device.synchronize()
        self.norm.backward(d_out, self.conv_out, self.gamma, self.beta, self.mean, self.rstd, self.flow, self.d_gamma, self.d_beta)
        device.synchronize()
        got = execute_graph(self.backward_graph, dict(zip(self.backward_in, (self.flow, self.image, self.filter))))
        self.filter_gradient = got[self.d_filter]
        return None if self.first else got[self.d_image]


class Classifier:
    """channels: of the image, then of each stage's result. dtype: of images, activations and flows; parameters are f32."""

    def __init__(self, batch, extent, channels, groups, classes, dtype="bf16", precision="f32_f32", seed=66, learning_rate=0.02,
                 momentum=0.95, weight_decay=0.01, other_rate=0.1):
        rng = np.random.default_rng(seed)
        self.dtype, self.settings = dtype, dict(learning_rate=learning_rate, momentum=momentum, weight_decay=weight_decay)
        self.stages = [Stage(rng, batch, extent, i, o, groups, dtype, "silu" if k == SILU_STAGE else "relu", k == 0)
                       for k, (i, o) in enumerate(zip(channels, channels[1:]))]
        self.muon = Muon([s.filter_shape for s in self.stages], dtype, precision)
        last = channels[-1]
        weights = rng.standard_normal([last, classes]) / np.sqrt(last)
        self.linear = Tensor.from_numpy(weights.astype(np.float32), "f32", weights.size)

        # the loss, its gradient at the last activation, and the linear layer's step
        G = ad.Graph()
        shape = [batch, extent, extent, last]
        activation = ad.Param(ad.Tensor(ad.Raw(G, G.g.new_input(shape, dtype))))
        linear = ad.Param(ad.Tensor(ad.Raw(G, G.g.new_input([last, classes], "f32"))))
        labels = ad.Tensor(ad.Raw(G, G.g.new_input([batch, classes], "f32")))
        self.head_in = (activation.value.raw.node, linear.value.raw.node, labels.raw.node)
        pooled = activation.value.to_data_type("f32").reshape([batch, extent * extent, last]).swap_dims(1, 2).reduce_mean(1).reshape([batch, last])
        loss = ad.cross_entropy_loss(pooled.matmul(linear.value, "f32_f32"), labels)
        grads = loss.backward()
        self.head_graph = G.g
        self.loss = G.g.new_output(loss.raw.node)
        self.d_activation = G.g.new_output(grads[activation.id].into_data_type(dtype).node)
        self.new_linear = G.g.new_output((ad.Tensor(linear.value.raw) - ad.Tensor(grads[linear.id]) * other_rate).raw.node)
        self.head_feeds = {n: Tensor.from_numpy(a, "f32", a.size) for n, a in G.feeds.items()}

        # the step of gamma and beta of all stages
        G = ad.Graph()
        self.affine_in, self.affine_out = [], []
        for s in self.stages:
            for _ in ("gamma", "beta"):
                value, gradient = (ad.Tensor(ad.Raw(G, G.g.new_input([s.norm.channels], "f32"))) for _ in range(2))
                self.affine_in += [value.raw.node, gradient.raw.node]
                self.affine_out.append(G.g.new_output((value - gradient * other_rate).raw.node))
        self.affine_graph = G.g
        self.affine_feeds = {n: Tensor.from_numpy(a, "f32", a.size) for n, a in G.feeds.items()}

    def graphs(self):
        return [g for s in self.stages for g in (s.forward_graph, s.backward_graph)] + [self.head_graph, self.affine_graph]

    def gradients(self, image, labels):
        """The loss, with the gradients left where step() finds them. image: a Tensor of `dtype`; labels: f32, one row per image."""
        x = image
        for s in self.stages:
            x = s.forward(x)
        got = execute_graph(self.head_graph, {**self.head_feeds, **dict(zip(self.head_in, (x, self.linear, labels)))})
        flow, self.next_linear = got[self.d_activation], got[self.new_linear]
        for s in reversed(self.stages):
            flow = s.backward(flow)
        return float(got[self.loss].to_numpy()[0])

    def step(self, image, labels):
        """One training step; returns the loss before it."""
        loss = self.gradients(image, labels)
        feeds = [t for s in self.stages for t in (s.gamma, s.d_gamma, s.beta, s.d_beta)]
        got = execute_graph(self.affine_graph, {**self.affine_feeds, **dict(zip(self.affine_in, feeds))})
        device.synchronize()
        filters, momenta = [s.filter for s in self.stages], [s.momentum for s in self.stages]
        self.muon.step([s.filter_gradient for s in self.stages], momenta, filters, momenta, filters, **self.settings)
        device.synchronize()
        for k, s in enumerate(self.stages):
            s.gamma, s.beta = got[self.affine_out[2 * k]], got[self.affine_out[2 * k + 1]]
        self.linear = self.next_linear
        return loss


def main(steps=20):
    """Trains on random images until it knows them by heart."""
    rng = np.random.default_rng(1)
    batch, extent, classes = 32, 16, 10
    model = Classifier(batch, extent, [16, 64, 128, 128], 8, classes)
    images = rng.standard_normal([batch, extent, extent, 16])
    one_hot = np.eye(classes, dtype=np.float32)[rng.integers(0, classes, batch)]
    image, labels = Tensor.from_numpy(ad._to_storage(images, "bf16"), "bf16", images.size), Tensor.from_numpy(one_hot, "f32", one_hot.size)
    for k in range(steps):
        print(f"step {k}: loss {model.step(image, labels):.4f}", flush=True)


if __name__ == "__main__":
    main()
