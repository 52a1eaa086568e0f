"""Root-mean-square norm with its residual, products in 8-bit integers and gradient clipping, as cases that can be timed:
`listed()` names them, `draw()` makes more of the same kinds and ranges, `prepare()` makes what a program has in hand before the
call and `run()` is one pass.

The kinds:
  norm       h = x + residual, y = gamma h / sqrt(mean(h^2) + epsilon) for every row, and what the backward pass reads
  norm_back  the gradients of h (the residual's own gradient added) and of gamma
  linear     rows quantised to 8 bits with a scale each, times weights of 8 bits with a scale for each channel
  layer      the norm with its output in 8 bits, and the product that reads it
  clip       the norm of all gradients together, and the gradients scaled down to it
"""
import functools
import math

import torch

own = False

EPSILON = 1e-5
NORM_FLOOR = 1e-6   # added to the gradients' norm before the division
MOST_NORM = 1.0
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}

# the parameters of the image classifier that harness/resnet.py records (width 32, 1000 classes): the head, then per stage two blocks and
# the shortcut, each filter with the two vectors of its normalisation, then the 1x1 convolution to the classes
CLASSIFIER = "32x147,32,32," + ",".join(
    "%dx%d,%d,%d,%dx%d,%d,%d,%dx%d,%d,%d,%dx%d,%d,%d,%dx%d,%d,%d" % tuple(
        v for i in (9 * c, 18 * c, c, 18 * c, 18 * c) for v in (2 * c, i, 2 * c, 2 * c)) for c in (32, 64, 128, 256)
) + ",1000x512,1000"


def listed():
    return [
        # serving one token: a row of a residual stream, where the call's latency is all
        {"name": "norm_token", "kind": "norm", "rows": 1, "columns": 4096, "dtype": "bf16", "residual": "bf16"},
        # a prompt's or a training step's residual stream
        {"name": "norm_prompt", "kind": "norm", "rows": 8192, "columns": 4096, "dtype": "bf16", "residual": "bf16"},
        # f32 at extents that nothing divides, no residual
        {"name": "norm_ragged_f32", "kind": "norm", "rows": 777, "columns": 1203, "dtype": "f32", "residual": "none"},
        # the training step's gradients of the same stream
        {"name": "norm_back_prompt", "kind": "norm_back", "rows": 8192, "columns": 4096, "dtype": "bf16", "residual": "bf16"},
        # mixed precision: a branch in f16 beside a residual stream in f32, odd extents
        {"name": "norm_back_ragged_f16", "kind": "norm_back", "rows": 1517, "columns": 2867, "dtype": "f16", "residual": "f32"},
        # one token through one layer: reading the weights is all
        {"name": "linear_token", "kind": "linear", "tokens": 1, "inputs": 4096, "channels": 4096, "dtype": "bf16", "bias": False},
        # a batch of sequences that take a token each, into a wide layer
        {"name": "linear_batch_f16", "kind": "linear", "tokens": 48, "inputs": 4096, "channels": 16384, "dtype": "f16", "bias": True},
        # a whole prompt: the matrix units are the bound
        {"name": "linear_prompt", "kind": "linear", "tokens": 4096, "inputs": 4096, "channels": 4096, "dtype": "bf16", "bias": False},
        # f32 activations, extents that nothing divides
        {"name": "linear_ragged_f32", "kind": "linear", "tokens": 333, "inputs": 1203, "channels": 777, "dtype": "f32", "bias": True},
        # a residual stream's norm straight into 8 bits, and the layer behind it
        {"name": "layer_prompt", "kind": "layer", "tokens": 2048, "inputs": 4096, "channels": 8192, "dtype": "bf16", "residual": "bf16"},
        # the gradients of the whole image classifier: 65 small tensors
        {"name": "clip_classifier_f32", "kind": "clip", "shapes": CLASSIFIER, "dtype": "f32", "clips": True},
        # the gradients of twenty-four wide layers
        {"name": "clip_layers_bf16", "kind": "clip", "shapes": ",".join(["4096x4096"] * 24), "dtype": "bf16", "clips": True},
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _extent(rng, low, high):
    """Half of them as wide as layers are, multiples of 64 from there on, the others odd or even as they come."""
    n = _log(rng, low, high)
    return min(high, -(-n // 64) * 64) if rng.random() < 0.5 and n >= 64 else n


def draw(rng):
    kind = rng.choice(["norm", "norm_back", "linear", "linear", "layer", "clip"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind in ("norm", "norm_back"):
        # (gradients of a row of very few values are next to nothing but rounding)
        columns = _extent(rng, 8 if kind == "norm" else 32, 16384)
        most = 8192 * 4096 // (2 if dtype == "f32" else 1)
        residual = rng.choice(["none", dtype, "f32"])
        most //= 2 if residual == "f32" and dtype != "f32" else 1
        return {"kind": kind, "rows": _log(rng, 1, min(32768, most // columns)), "columns": columns, "dtype": dtype, "residual": residual}
    if kind in ("linear", "layer"):
        inputs, channels = _extent(rng, 16, 16384), _extent(rng, 16, 16384)
        tokens = _log(rng, 1, max(1, min(8192, 4096 ** 3 // (inputs * channels))))
        if kind == "linear":
            return {"kind": kind, "tokens": tokens, "inputs": inputs, "channels": channels, "dtype": dtype, "bias": rng.random() < 0.5}
        # (a norm's values are on the border of two whole numbers now and then: results of 16 bits do not show on which side)
        dtype = "f16" if dtype == "f16" else "bf16"
        return {"kind": kind, "tokens": tokens, "inputs": inputs, "channels": channels, "dtype": dtype, "residual": rng.choice(["none", dtype, "f32"])}
    count, shapes, left = _log(rng, 1, 200), [], 24 * 4096 * 4096 // (2 if dtype == "f32" else 1)
    while len(shapes) < count and left > 0:
        n = rng.choice([1, 2, 3])
        size = min(left, _log(rng, 1, 4096) * (_log(rng, 1, 4096) if n > 1 else 1))
        left -= size
        shapes.append(str(size))
    return {"kind": kind, "shapes": ",".join(shapes), "dtype": dtype, "clips": rng.random() < 0.7}


def _sizes(case):
    return tuple(math.prod(int(d) for d in s.split("x")) for s in case["shapes"].split(","))


def _pitch(inputs):
    """Bytes of a quantised row: padded with zeros to whole vectors."""
    return -(-inputs // 16) * 16


def _activations(normal, rows, columns):
    """Rows of different sizes, with a few channels that are much larger than the others, as trained layers have them."""
    wide = torch.where(normal(columns) > 2.5, 8.0, 1.0) * (0.5 + normal(columns).abs())
    return normal(rows, columns) * wide * torch.exp(0.3 * normal(rows, 1))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    dtype, kind = TORCH[case["dtype"]], case["kind"]
    s = {"case": case}
    if kind == "clip":
        sizes = _sizes(case)
        total = sum(sizes)
        # (norms of about 20 or a half, as far as the least values of f16 go)
        size = (20.0 if case["clips"] else 0.5) / math.sqrt(total)
        s["gradients"] = [(size * normal(n)).to(dtype) for n in sizes]
        # a trainer's gradients lie in one buffer, each on a border of 256 bytes
        at, end = [], 0
        for n in sizes:
            at.append(end)
            end += -(-n // 128) * 128
        s["flat"] = torch.zeros(end, dtype=dtype, device="cuda")
        s["clipped"] = [s["flat"][a:a + n] for a, n in zip(at, sizes)]
        s["norm"] = torch.zeros(1, device="cuda")
        return s
    rows, columns = (case["rows"], case["columns"]) if "rows" in case else (case["tokens"], case["inputs"])
    if kind in ("norm", "norm_back", "layer"):
        stream = dtype if case["residual"] == "none" else TORCH[case["residual"]]
        s["gamma"] = 1.0 + 0.3 * normal(columns)
        if kind == "norm_back":
            h = _activations(normal, rows, columns).to(stream)
            s["h"], s["rstd"] = h, (h.float().square().mean(1) + EPSILON).rsqrt()
            s["dy"] = ((1.0 if dtype == torch.float16 else 0.01) * normal(rows, columns)).to(dtype)
            s["dx"], s["dgamma"] = torch.empty(rows, columns, dtype=dtype, device="cuda"), torch.empty(columns, device="cuda")
            if case["residual"] != "none":
                s["dh"] = ((1.0 if dtype == torch.float16 else 0.01) * normal(rows, columns)).to(stream)
                if stream != dtype:
                    s["dresidual"] = torch.empty_like(h)
            return s
        s["x"] = _activations(normal, rows, columns).to(dtype)
        if case["residual"] != "none":
            s["residual"] = (2.0 * _activations(normal, rows, columns)).to(stream)
            s["h"] = torch.empty_like(s["residual"])
        if kind == "norm":
            s["y"], s["rstd"] = torch.empty_like(s["x"]), torch.empty(rows, device="cuda")
            return s
    else:
        s["x"] = _activations(normal, rows, columns).to(dtype)
    # the weights, quantised once: rows of one output channel each, with a scale for each
    channels = case["channels"]
    w = normal(channels, columns) * (0.5 + normal(channels, 1).abs()) / math.sqrt(columns)
    s["weight_scales"] = w.abs().amax(1) / 127.0
    s["weights"] = torch.zeros(channels, _pitch(columns), dtype=torch.int8, device="cuda")
    s["weights"][:, :columns] = torch.round(w / s["weight_scales"][:, None]).to(torch.int8)
    s["bias"] = 0.5 * normal(channels) if case.get("bias") else None
    # what the call works in: the quantised rows and their scales
    s["q"], s["scales"] = torch.zeros(rows, _pitch(columns), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    s["out"] = torch.empty(rows, channels, dtype=dtype, device="cuda")
    return s


# ---- the plain form: 32 bits, one elementary operation after the other -----------------------------------------------
def _plain_stream(s):
    """h in its own type: what later layers read is what is normalised."""
    return (s["x"].float() + s["residual"].float()).to(s["residual"].dtype) if "residual" in s else s["x"]


def _plain_rms(h, gamma):
    rstd = 1.0 / torch.sqrt(h.float().square().mean(1) + EPSILON)
    return h.float() * rstd[:, None] * gamma, rstd


def _plain_norm(s):
    h = _plain_stream(s)
    y, rstd = _plain_rms(h, s["gamma"])
    return {"y": y.to(s["x"].dtype), "rstd": rstd, **({"h": h} if "residual" in s else {})}


def _plain_norm_back(s):
    rstd = s["rstd"][:, None]
    xh, dy = s["h"].float() * rstd, s["dy"].float()
    flow = dy * s["gamma"]
    dx = rstd * (flow - xh * (flow * xh).mean(1, keepdim=True))
    dx = dx + s["dh"].float() if "dh" in s else dx
    more = {"dresidual": dx.to(s["h"].dtype)} if "dresidual" in s else {}
    return {"dx": dx.to(s["dy"].dtype), "dgamma": (dy * xh).sum(0), **more}


def _plain_quantize(x):
    """Whole numbers and the scale of each row: x = scale q. (In 64 bits: the quotients lie next to a border now and then.)"""
    most = x.double().abs().amax(1)
    q = torch.round(x.double() * 127.0 / torch.where(most > 0, most, 1.0)[:, None])
    return q.float(), (most / 127.0).float()


def _plain_product(s, q, scales):
    """(Sums of products of whole numbers: nearly all below 2^24, where f32 has them exactly.)"""
    weights = s["weights"][:, :q.shape[1]].float()
    y = (q @ weights.T) * scales[:, None] * s["weight_scales"]
    y = y if s["bias"] is None else y + s["bias"]
    return y.to(s["out"].dtype)


def _plain_clip(s):
    norm = torch.sqrt(torch.stack([g.float().square().sum() for g in s["gradients"]]).double().sum())
    by = (MOST_NORM / (norm + NORM_FLOOR)).clamp(max=1.0).float()
    flat = torch.zeros_like(s["flat"])
    starts = [c.storage_offset() for c in s["clipped"]]
    [flat[a:a + g.numel()].copy_(g.float() * by) for a, g in zip(starts, s["gradients"])]
    return {"clipped": flat, "norm": norm.float()[None]}


# ---- the framework's operators ------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _rms_norm(columns, dtype, residual, output):
    import helium_amd as ha

    return ha.RmsNorm(columns, dtype, residual_dtype=None if residual == "none" else residual, output=output, epsilon=EPSILON)


@functools.lru_cache(maxsize=None)
def _quantize(columns, dtype):
    import helium_amd as ha

    return ha.QuantizeRows(columns, dtype)


@functools.lru_cache(maxsize=None)
def _product(inputs, channels, dtype):
    import helium_amd as ha

    return ha.Int8Matmul(inputs, channels, dtype)


@functools.lru_cache(maxsize=16)
def _clip(sizes, dtype):
    import helium_amd as ha

    return ha.GradientClip(sizes, dtype)


def _at(*tensors):
    return [None if t is None else t.data_ptr() for t in tensors]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "norm":
            return _plain_norm(s)
        if kind == "norm_back":
            return _plain_norm_back(s)
        if kind == "clip":
            return _plain_clip(s)
        if kind == "linear":
            return _plain_product(s, *_plain_quantize(s["x"]))
        h = _plain_stream(s)
        y = _plain_product(s, *_plain_quantize(_plain_rms(h, s["gamma"])[0]))
        return {"y": y, "h": h} if "residual" in s else {"y": y}
    if kind == "clip":
        _clip(_sizes(case), case["dtype"]).clip(_at(*s["gradients"]), _at(*s["clipped"]), MOST_NORM, s["norm"].data_ptr())
        return {"clipped": s["flat"], "norm": s["norm"]}
    if kind == "norm":
        op = _rms_norm(case["columns"], case["dtype"], case["residual"], "same")
        x, gamma, y, residual, h, rstd = _at(*(s.get(k) for k in ("x", "gamma", "y", "residual", "h", "rstd")))
        op.forward(case["rows"], x, gamma, y, residual=residual, new_residual=h, rstd=rstd)
        return {k: s[k] for k in ("y", "rstd", "h") if k in s}
    if kind == "norm_back":
        op = _rms_norm(case["columns"], case["dtype"], case["residual"], "same")
        dy, h, gamma, rstd, dx, dgamma, dh, dresidual = _at(*(s.get(k) for k in ("dy", "h", "gamma", "rstd", "dx", "dgamma", "dh", "dresidual")))
        op.backward(case["rows"], dy, h, gamma, rstd, dx, dgamma, dh=dh, dresidual=dresidual)
        return {k: s[k] for k in ("dx", "dgamma", "dresidual") if k in s}
    tokens, inputs = case["tokens"], case["inputs"]
    x, q, scales, weights, weight_scales, bias, out = _at(*(s[k] for k in ("x", "q", "scales", "weights", "weight_scales", "bias", "out")))
    if kind == "linear":
        _quantize(inputs, case["dtype"]).quantize(tokens, x, q, scales)
    else:
        gamma, residual, h = _at(*(s.get(k) for k in ("gamma", "residual", "h")))
        _rms_norm(inputs, case["dtype"], case["residual"], "i8").forward(tokens, x, gamma, q, residual=residual, new_residual=h, scales=scales)
    _product(inputs, case["channels"], case["dtype"]).multiply(tokens, q, scales, weights, weight_scales, out, bias=bias)
    return s["out"] if kind == "linear" else {"y": s["out"], "h": s["h"]} if "residual" in s else {"y": s["out"]}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "clip":
        n = sum(_sizes(case))
        return {"bytes": 2 * n * size + 4, "flops": 3 * n}
    stream = 0 if case.get("residual", "none") == "none" else SIZE[case["residual"]]
    if kind in ("norm", "norm_back"):
        n, columns = case["rows"] * case["columns"], case["columns"]
        if kind == "norm":
            return {"bytes": n * (2 * size + 2 * stream) + 4 * columns + 4 * case["rows"], "flops": 5 * n}
        # dy, h and the residual's gradient in, the gradients out
        apart = stream if stream and case["residual"] != case["dtype"] else 0
        return {"bytes": n * (2 * size + (stream or size) + stream + apart) + 8 * columns + 4 * case["rows"], "flops": 10 * n}
    m, k, n = case["tokens"], case["inputs"], case["channels"]
    bytes_ = m * k * size + 2 * m * k * stream + n * k + 4 * n + m * n * size + (4 * n if case.get("bias") else 0) + (4 * k if kind == "layer" else 0)
    return {"bytes": bytes_, "flops": 2 * m * n * k}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _exact_h(s):
    if "residual" not in s:
        return s["x"].double()
    return torch.add(s["x"].double(), s["residual"].double()).to(s["residual"].dtype).double()


def _exact_y(s, h):
    size = torch.sqrt(torch.linalg.vecdot(h, h) / h.shape[1] + EPSILON)
    return torch.einsum("rc,c->rc", h / size[:, None], s["gamma"].double()), size.reciprocal()


def _exact_product(s, y):
    step = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / 127.0
    whole = torch.nan_to_num(y / step[:, None], nan=0.0).round()
    w = s["weights"][:, :y.shape[1]].double().mul(s["weight_scales"].double()[:, None])
    out = torch.mm(whole * step[:, None], w.T.contiguous())
    return out if s["bias"] is None else out.add(s["bias"].double())


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "linear":
        return _exact_product(s, s["x"].double())
    if kind in ("norm", "layer"):
        h = _exact_h(s)
        y, rstd = _exact_y(s, h)
        got = {"y": y, "rstd": rstd} if kind == "norm" else {"y": _exact_product(s, y)}
        return {**got, "h": h} if "residual" in s else got
    if kind == "norm_back":
        # the chain rule through rstd, which the call is given and which counts as the row's own
        h, dy, gamma, r = s["h"].double(), s["dy"].double(), s["gamma"].double(), s["rstd"].double()
        through = torch.linalg.vecdot(dy * gamma, h) * r ** 3 / h.shape[1]
        dh = torch.addcmul(dy * gamma * r[:, None], h, through[:, None], value=-1.0)
        dh = dh + s["dh"].double() if "dh" in s else dh
        got = {"dx": dh, "dgamma": torch.mv((dy * h).T, r)}
        return {**got, "dresidual": dh} if "dresidual" in s else got
    parts = torch.cat([g.double().norm()[None] for g in s["gradients"]])
    norm = torch.linalg.vector_norm(parts)
    by = min(1.0, MOST_NORM / (norm.item() + NORM_FLOOR))
    flat = torch.zeros_like(s["flat"], dtype=torch.float64)
    for place, g in zip(s["clipped"], s["gradients"]):
        flat[place.storage_offset():place.storage_offset() + g.numel()] = g.double() * by
    return {"clipped": flat, "norm": norm[None]}
