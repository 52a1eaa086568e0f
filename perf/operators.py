"""Group norm with its activation (channels last, forward and backward) and Muon's orthogonalised updates, as cases that can
be timed: `listed()` names them, `draw()` makes more of the same kinds and ranges, `prepare()` makes what a training
program has in hand before the call and `run()` is one pass.

The kinds:
  norm      y = act(gamma * (x - mean) / sqrt(var + epsilon) + beta) over groups of channels of [batch, pixels, channels],
            and the statistics that the backward pass reads
  norm_back the gradients of x, gamma and beta
  ortho     matrices of a group replaced by their orthogonalised forms: five Newton-Schulz steps from U / |U|
  muon      one optimizer step of a group of matrices: momenta, orthogonalised updates and weights
"""
import functools
import math

import torch

own = False

EPSILON = 1e-5
NORM_FLOOR = 1e-7                    # added to a matrix's norm before the division
A, B, C = 3.4445, -4.7750, 2.0315    # one step: X <- A X + (B S + C S S) X with S = X X^T
STEPS = 5
RATE, MOMENTUM, DECAY = 0.02, 0.95, 0.01
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}

# the filters of the image classifier that harness/resnet.py records (width 32, 1000 classes), as rows of one output channel
# each: the head, then per stage two blocks and the shortcut, then the 1x1 convolution to the classes
CLASSIFIER = "32x147," + ",".join(
    "%dx%d,%dx%d,%dx%d,%dx%d,%dx%d" % (2 * c, 9 * c, 2 * c, 18 * c, 2 * c, c, 2 * c, 18 * c, 2 * c, 18 * c) for c in (32, 64, 128, 256)
) + ",1000x512"


def listed():
    return [
        # serving one image: the last stage's activation, where the call's latency is all
        {"name": "norm_one_image", "kind": "norm", "batch": 1, "pixels": 49, "channels": 512, "groups": 32, "dtype": "bf16", "act": "silu"},
        # the benchmark's normalised activation, batch 64 at 56 x 56
        {"name": "norm_block", "kind": "norm", "batch": 64, "pixels": 3136, "channels": 256, "groups": 32, "dtype": "bf16", "act": "relu"},
        # f32 at extents that nothing divides, five channels to a group
        {"name": "norm_ragged_f32", "kind": "norm", "batch": 5, "pixels": 1517, "channels": 150, "groups": 30, "dtype": "f32", "act": "silu"},
        # two large images: groups far larger than what stays on the chip
        {"name": "norm_large_image", "kind": "norm", "batch": 2, "pixels": 262144, "channels": 128, "groups": 32, "dtype": "bf16", "act": "silu"},
        # the gradient of the benchmark's activation
        {"name": "norm_back_block", "kind": "norm_back", "batch": 64, "pixels": 3136, "channels": 256, "groups": 32, "dtype": "bf16", "act": "silu"},
        # a small training step in f32, bound by launches
        {"name": "norm_back_small_f32", "kind": "norm_back", "batch": 8, "pixels": 64, "channels": 256, "groups": 16, "dtype": "f32", "act": "silu"},
        # f16 with six channels to a group and odd extents
        {"name": "norm_back_ragged_f16", "kind": "norm_back", "batch": 3, "pixels": 2867, "channels": 102, "groups": 17, "dtype": "f16", "act": "none"},
        # one 3x3 filter of 64 channels: fifteen small products, one after the other
        {"name": "ortho_filter_f32", "kind": "ortho", "shapes": "64x576", "dtype": "f32"},
        # tall and odd extents: a classifier's last layer and a layer that no tile divides
        {"name": "ortho_ragged_f32", "kind": "ortho", "shapes": "1000x512,777x1203", "dtype": "f32"},
        # a large layer in mixed precision: the products are the bound
        {"name": "ortho_square_bf16", "kind": "ortho", "shapes": "4096x4096", "dtype": "bf16"},
        # the optimizer step of the whole image classifier, f32 gradients
        {"name": "muon_classifier_f32", "kind": "muon", "shapes": CLASSIFIER, "dtype": "f32"},
        # two layers of a wide perceptron: 16-bit gradients, f32 weights
        {"name": "muon_layers_bf16", "kind": "muon", "shapes": "4096x1024,1024x4096", "dtype": "bf16"},
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_back", "ortho", "muon"])
    if kind in ("norm", "norm_back"):
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        most = 51_380_224 // (2 if dtype == "f32" else 1)
        groups, width = _log(rng, 1, 64), _log(rng, 1, 64)
        if rng.random() < 0.6:
            groups, width = 1 << (groups.bit_length() - 1), 1 << (width.bit_length() - 1)
        channels = groups * width
        # (relu's gradient is not continuous: where 32 and 64 bits put an argument on different sides of zero no two
        # gradients agree, so gradients are drawn with the other activations)
        act = rng.choice(["none", "relu", "silu"]) if kind == "norm" else rng.choice(["none", "silu"])
        batch = _log(rng, 1, min(128, max(1, most // channels)))
        pixels = _log(rng, 1, max(1, min(262144, most // (channels * batch))))
        # (a group of very few values has next to no gradient: what is left of it is rounding)
        return {"kind": kind, "batch": batch, "pixels": max(pixels, -(-16 // width)), "channels": channels, "groups": groups, "dtype": dtype, "act": act}
    count, shapes, cost = _log(rng, 1, 12), [], 0
    while len(shapes) < count:
        rows, cols = _log(rng, 8, 4096), _log(rng, 8, 4096)
        if rng.random() < 0.5:
            rows, cols = -(-rows // 32) * 32, -(-cols // 32) * 32
        cost += min(rows, cols) * rows * cols
        if shapes and cost > 4096 * 4096 * 1024:
            break
        shapes.append("%dx%d" % (rows, cols))
    return {"kind": kind, "shapes": ",".join(shapes), "dtype": rng.choice(["f32", "bf16", "f16"])}


def _shapes(case):
    return tuple(tuple(int(d) for d in s.split("x")) for s in case["shapes"].split(","))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    dtype = TORCH[case["dtype"]]
    if case["kind"] in ("norm", "norm_back"):
        n, p, c, groups = (case[k] for k in ("batch", "pixels", "channels", "groups"))
        # a convolution's output: every channel has a scale and an offset of its own
        x = (normal(n, p, c) * (0.5 + normal(c).abs()) + 0.5 * normal(c)).to(dtype)
        s = {"case": case, "x": x, "gamma": 1.0 + 0.2 * normal(c), "beta": 0.2 * normal(c)}
        if case["kind"] == "norm":
            s["y"] = torch.empty_like(x)
            s["mean"], s["rstd"] = torch.empty(2, n, groups, device="cuda")
            return s
        s["dy"] = (0.01 * normal(n, p, c)).to(dtype) if dtype != torch.float16 else normal(n, p, c).to(dtype)
        xg = x.float().view(n, p, groups, c // groups)
        s["mean"] = xg.mean((1, 3))
        s["rstd"] = (xg.var((1, 3), unbiased=False) + EPSILON).rsqrt()
        s["dx"], s["dgamma"], s["dbeta"] = torch.empty_like(x), torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
        return s
    shapes = _shapes(case)
    # a gradient: a few strong directions in noise
    few = lambda r, c: normal(r, 8) @ normal(8, c) * 0.35  # noqa: E731
    s = {"case": case, "shapes": shapes, "grads": [(1e-3 * (normal(r, c) + few(r, c))).to(dtype) for r, c in shapes]}
    if case["kind"] == "ortho":
        s["out"] = [torch.empty_like(x) for x in s["grads"]]
        return s
    s["weights"] = [normal(r, c) / math.sqrt(c) for r, c in shapes]
    s["momenta"] = [1e-2 * normal(r, c) for r, c in shapes]
    s["new_weights"] = [torch.empty_like(w) for w in s["weights"]]
    s["new_momenta"] = [torch.empty_like(w) for w in s["weights"]]
    return s


# ---- the plain form: 32 bits, one elementary operation after the other -----------------------------------------------
def _normalised(x, mean, rstd, groups):
    n, p, c = x.shape
    return ((x.float().view(n, p, groups, c // groups) - mean.view(n, 1, groups, 1)) * rstd.view(n, 1, groups, 1)).view(n, p, c)


def _plain_norm(s):
    case, x = s["case"], s["x"]
    n, p, c = x.shape
    groups = case["groups"]
    xg = x.float().view(n, p, groups, c // groups)
    mean = xg.mean((1, 3))
    rstd = 1.0 / torch.sqrt((xg - mean.view(n, 1, groups, 1)).square().mean((1, 3)) + EPSILON)
    z = _normalised(x, mean, rstd, groups) * s["gamma"] + s["beta"]
    y = {"none": lambda: z, "relu": lambda: z.clamp(min=0.0), "silu": lambda: z / (1.0 + torch.exp(-z))}[case["act"]]()
    return {"y": y.to(x.dtype), "mean": mean, "rstd": rstd}


def _plain_norm_back(s):
    case, x = s["case"], s["x"]
    n, p, c = x.shape
    groups = case["groups"]
    d = c // groups
    xh = _normalised(x, s["mean"], s["rstd"], groups)
    dz = s["dy"].float()
    if case["act"] == "silu":
        z = xh * s["gamma"] + s["beta"]
        sig = 1.0 / (1.0 + torch.exp(-z))
        dz = dz * (sig * (1.0 + z * (1.0 - sig)))
    elif case["act"] == "relu":
        dz = dz * (xh * s["gamma"] + s["beta"] > 0)
    flow = dz * s["gamma"]
    s1 = flow.view(n, p, groups, d).mean((1, 3)).view(n, 1, groups, 1)
    s2 = (flow * xh).view(n, p, groups, d).mean((1, 3)).view(n, 1, groups, 1)
    dx = (flow.view(n, p, groups, d) - (s1 + xh.view(n, p, groups, d) * s2)) * s["rstd"].view(n, 1, groups, 1)
    return {"dx": dx.view(n, p, c).to(x.dtype), "dgamma": (dz * xh).sum((0, 1)), "dbeta": dz.sum((0, 1))}


def _step(x, _):
    s = x @ x.T
    return A * x + (B * s + C * (s @ s)) @ x


def _plain_ortho(u):
    """U in 32 bits -> its orthogonalised form in 32 bits."""
    x = u.T if u.shape[0] > u.shape[1] else u
    x = functools.reduce(_step, range(STEPS), x / (torch.sqrt((x * x).sum()) + NORM_FLOOR))
    return x.T if u.shape[0] > u.shape[1] else x


def _plain_muon(grad, momentum, weight):
    rows, cols = grad.shape
    g = grad.float()
    m = MOMENTUM * momentum + g
    o = _plain_ortho(g + MOMENTUM * m)
    return (1.0 - RATE * DECAY) * weight - RATE * math.sqrt(max(1.0, rows / cols)) * o, m


# ---- the framework's operators ------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _group_norm(batch, pixels, channels, groups, dtype, act):
    import helium_amd as ha

    return ha.GroupNorm(batch, pixels, channels, groups, dtype, activation=act, epsilon=EPSILON)


@functools.lru_cache(maxsize=16)
def _muon(shapes, dtype, results):
    """Products as exact as the type of the results asks for."""
    import helium_amd as ha

    return ha.Muon(shapes, dtype, precision="f32_f32" if results == "f32" else "f16_f32", steps=STEPS)


def _at(tensors):
    return [t.data_ptr() for t in tensors]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "norm":
            return _plain_norm(s)
        if kind == "norm_back":
            return _plain_norm_back(s)
        if kind == "ortho":
            return [_plain_ortho(u.float()).to(u.dtype) for u in s["grads"]]
        done = [_plain_muon(*gmw) for gmw in zip(s["grads"], s["momenta"], s["weights"])]
        return {"weights": [w for w, _ in done], "momenta": [m for _, m in done]}
    if kind in ("norm", "norm_back"):
        op = _group_norm(*(case[k] for k in ("batch", "pixels", "channels", "groups", "dtype", "act")))
        x, gamma, beta, mean, rstd = _at(s[k] for k in ("x", "gamma", "beta", "mean", "rstd"))
        if kind == "norm":
            op.forward(x, gamma, beta, s["y"].data_ptr(), mean, rstd)
            return {k: s[k] for k in ("y", "mean", "rstd")}
        op.backward(s["dy"].data_ptr(), x, gamma, beta, mean, rstd, *_at(s[k] for k in ("dx", "dgamma", "dbeta")))
        return {k: s[k] for k in ("dx", "dgamma", "dbeta")}
    op = _muon(s["shapes"], case["dtype"], case["dtype"] if kind == "ortho" else "f32")
    if kind == "ortho":
        op.orthogonalize(_at(s["grads"]), _at(s["out"]))
        return s["out"]
    op.step(_at(s["grads"]), _at(s["momenta"]), _at(s["weights"]), _at(s["new_momenta"]), _at(s["new_weights"]),
            learning_rate=RATE, momentum=MOMENTUM, weight_decay=DECAY, nesterov=True)
    return {"weights": s["new_weights"], "momenta": s["new_momenta"]}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] in ("norm", "norm_back"):
        n, p, c, groups = (case[k] for k in ("batch", "pixels", "channels", "groups"))
        tensors, per_element = (2, 8) if case["kind"] == "norm" else (3, 18)
        return {"bytes": tensors * n * p * c * SIZE[case["dtype"]] + 8 * n * groups + (8 if case["kind"] == "norm" else 16) * c,
                "flops": per_element * n * p * c}
    flops = bytes_ = 0
    for rows, cols in _shapes(case):
        m, n = min(rows, cols), max(rows, cols)
        # the two products whose result is symmetric count half
        flops += STEPS * (m * m * n + m * m * m + 2 * m * m * n)
        bytes_ += rows * cols * (SIZE[case["dtype"]] + (SIZE[case["dtype"]] if case["kind"] == "ortho" else 16))
    return {"bytes": bytes_, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _exact_norm(s):
    case, x = s["case"], s["x"].double()
    n, p, c = x.shape
    groups = case["groups"]
    rows = x.reshape(n, p, groups, -1).permute(0, 2, 1, 3).reshape(n, groups, -1)
    var, mean = torch.var_mean(rows, dim=2, correction=0)
    std = torch.sqrt(var + EPSILON)
    spread = lambda v: v.repeat_interleave(c // groups, dim=1)[:, None, :]  # noqa: E731
    z = torch.addcmul(s["beta"].double(), (x - spread(mean)) / spread(std), s["gamma"].double())
    y = z if case["act"] == "none" else torch.where(z > 0, z, 0.0) if case["act"] == "relu" else z * torch.sigmoid(z)
    return {"y": y, "mean": mean, "rstd": std.reciprocal()}


def _exact_norm_back(s):
    """The chain rule through the statistics that the call is given, which count as the data's own."""
    case, x = s["case"], s["x"].double()
    n, p, c = x.shape
    groups = case["groups"]
    spread = lambda v: v.double().repeat_interleave(c // groups, dim=1)[:, None, :]  # noqa: E731
    rstd, gamma = spread(s["rstd"]), s["gamma"].double()
    xh = (x - spread(s["mean"])) * rstd
    z = xh * gamma + s["beta"].double()
    slope = {"none": lambda: 1.0, "relu": lambda: (z > 0).double(), "silu": lambda: torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)}[case["act"]]()
    dz = s["dy"].double() * slope
    dbeta_n, dgamma_n = dz.sum(1), (dz * xh).sum(1)
    of_group = lambda v: (v * gamma).reshape(n, groups, -1).sum(2) / (p * c // groups)  # noqa: E731
    dx = rstd * (gamma * dz - spread(of_group(dbeta_n)) - xh * spread(of_group(dgamma_n)))
    return {"dx": dx, "dgamma": dgamma_n.sum(0), "dbeta": dbeta_n.sum(0)}


def _exact_ortho(u):
    """(In Horner's form, X <- (a + (b + c S) S) X, on the smaller side.)"""
    wide = u if u.shape[0] <= u.shape[1] else u.mT
    x = wide / (torch.linalg.vector_norm(wide) + NORM_FLOOR)
    one = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        s = x.matmul(x.mT)
        x = torch.addmm(A * one, torch.add(B * one, s, alpha=C), s).matmul(x)
    return x if u.shape[0] <= u.shape[1] else x.mT


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(s)
    if case["kind"] == "norm_back":
        return _exact_norm_back(s)
    if case["kind"] == "ortho":
        return [_exact_ortho(u.double()) for u in s["grads"]]
    weights, momenta = [], []
    for g, m, w in zip(s["grads"], s["momenta"], s["weights"]):
        new = MOMENTUM * m.double() + g.double()
        scale = RATE * max(1.0, g.shape[0] / g.shape[1]) ** 0.5
        momenta.append(new)
        weights.append(w.double() - RATE * DECAY * w.double() - scale * _exact_ortho(g.double() + MOMENTUM * new))
    return {"weights": weights, "momenta": momenta}
