"""Group norm through the C ABI on the GPU against the 64-bit oracle."""
import numpy as np
import pytest

import helium_amd as ha
from group_norm_cases import EPSILON, SHAPES, WIDE, WIDEST, check_backward, check_forward, inputs, to_f32, to_storage
from oracle import group_norm as oracle

pytestmark = pytest.mark.gpu

LARGE = [
    (1, 49, 512, 32),
    (8, 784, 128, 32),
    (3, 3136, 64, 8),
    (2, 1517, 150, 30),
    (1, 20000, 48, 4),    # a sample that no workgroup holds
    (2, 5000, 320, 32),
    (40, 9, 512, 32),
]


def device(a, offset=0):
    """A copy on the GPU, `offset` bytes into its allocation, with a margin behind it."""
    b = ha.DeviceBuffer(offset + a.nbytes + 64)
    b.fill_u8(0xEE)
    whole = np.full(b.nbytes, 0xEE, np.uint8)
    whole[offset:offset + a.nbytes] = np.ascontiguousarray(a).reshape(-1).view(np.uint8)
    b.upload(whole)
    return b, offset


def address(d):
    return d[0].ptr.value + d[1]


def back(d, like):
    out = d[0].read(d[1], like.dtype, like.size).reshape(like.shape)
    assert (d[0].read(d[1] + like.nbytes, np.uint8, 64) == 0xEE).all(), "written past the end"
    return out


def empty(shape, dtype, offset=0):
    return device(np.full(shape, 0xEE, np.uint8).astype(dtype) if dtype == np.uint8 else np.zeros(shape, dtype), offset)


def run_forward(norm, shape, host, stats=True, in_place=False, offset=0, stream=None):
    n, p, c, groups = shape
    x, gamma, beta = device(host["x"], offset), device(host["gamma"]), device(host["beta"])
    y = x if in_place else empty(host["x"].shape, host["x"].dtype, offset)
    mean, rstd = empty((n, groups), np.float32), empty((n, groups), np.float32)
    norm.forward(address(x), address(gamma), address(beta), address(y), *((address(mean), address(rstd)) if stats else ()), stream=stream)
    if stream is not None:
        stream.synchronize()
    like = np.zeros((n, groups), np.float32)
    return back(y, host["x"]), back(mean, like), back(rstd, like)


def run_backward(norm, shape, host, mean, rstd, into=None):
    n, p, c, groups = shape
    d = {k: device(host[k]) for k in ("dy", "x", "gamma", "beta")}
    d["mean"], d["rstd"] = device(mean), device(rstd)
    dx = empty(host["x"].shape, host["x"].dtype) if into is None else d[into]
    dgamma, dbeta = empty((c,), np.float32), empty((c,), np.float32)
    norm.backward(*[address(d[k]) for k in ("dy", "x", "gamma", "beta", "mean", "rstd")], address(dx), address(dgamma), address(dbeta))
    like = np.zeros(c, np.float32)
    return back(dx, host["x"]), back(dgamma, like), back(dbeta, like)


@pytest.mark.parametrize("activation", ["none", "relu", "silu"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES + LARGE)
def test_forward_and_backward_match_the_oracle(gpu, shape, dtype, activation):
    param_dtype = dtype if shape[1] % 2 else "f32"
    norm = ha.GroupNorm(*shape, dtype, param_dtype=param_dtype, activation=activation, epsilon=EPSILON)
    host, v, mean, rstd = inputs(shape, dtype, param_dtype, activation, seed=shape[1])
    y, got_mean, got_rstd = run_forward(norm, shape, host)
    check_forward(shape, dtype, activation, v, to_f32(y, dtype), got_mean, got_rstd)
    dx, dgamma, dbeta = run_backward(norm, shape, host, mean, rstd)
    check_backward(shape, dtype, activation, v, mean, rstd, to_f32(dx, dtype), dgamma, dbeta)


@pytest.mark.parametrize("parts", ["0", "1"])
@pytest.mark.parametrize("shape,dtype", [((5000, 1, 64, 8), "bf16"), ((1025, 3, 40, 5), "f16"), ((300000, 1, 8, 2), "f32"), ((1 << 22, 1, 2, 1), "f32")])
def test_many_samples_of_few_pixels_match_the_oracle(gpu, monkeypatch, shape, dtype, parts):
    monkeypatch.setenv("HELIUM_HIP_NORM_PARTS", parts)
    norm = ha.GroupNorm(*shape, dtype, activation="silu", epsilon=EPSILON)
    host, v, mean, rstd = inputs(shape, dtype, "f32", "silu", seed=15)
    y, got_mean, got_rstd = run_forward(norm, shape, host)
    check_forward(shape, dtype, "silu", v, to_f32(y, dtype), got_mean, got_rstd)
    dx, dgamma, dbeta = run_backward(norm, shape, host, mean, rstd)
    check_backward(shape, dtype, "silu", v, mean, rstd, to_f32(dx, dtype), dgamma, dbeta)


@pytest.mark.parametrize("shape,dtype", WIDE + WIDEST)
def test_wide_groups_match_the_oracle(gpu, shape, dtype):
    norm = ha.GroupNorm(*shape, dtype, activation="silu", epsilon=EPSILON)
    host, v, mean, rstd = inputs(shape, dtype, "f32", "silu", seed=13)
    y, got_mean, got_rstd = run_forward(norm, shape, host)
    check_forward(shape, dtype, "silu", v, to_f32(y, dtype), got_mean, got_rstd)
    dx, dgamma, dbeta = run_backward(norm, shape, host, mean, rstd)
    check_backward(shape, dtype, "silu", v, mean, rstd, to_f32(dx, dtype), dgamma, dbeta)


@pytest.mark.parametrize("shape", [(2, 49, 32, 8), (1, 20000, 48, 4)])
def test_results_may_take_an_operands_place_and_statistics_may_be_left_out(gpu, shape):
    norm = ha.GroupNorm(*shape, "bf16", activation="silu", epsilon=EPSILON)
    host, v, mean, rstd = inputs(shape, "bf16", "f32", "silu", seed=1)
    want = run_forward(norm, shape, host)
    y, no_mean, no_rstd = run_forward(norm, shape, host, stats=False, in_place=True)
    assert np.array_equal(y, want[0]) and not no_mean.any() and not no_rstd.any()
    apart = run_backward(norm, shape, host, mean, rstd)
    for into in ("dy", "x"):
        for a, b in zip(run_backward(norm, shape, host, mean, rstd, into=into), apart):
            assert np.array_equal(a, b)


def test_operands_need_no_more_than_their_vectors_alignment(gpu):
    """Pixels of 6 bytes: vectors of two bytes, at any even address."""
    shape = (2, 100, 3, 1)
    norm = ha.GroupNorm(*shape, "bf16", epsilon=EPSILON)
    host, v, _, _ = inputs(shape, "bf16", "f32", "none", seed=2)
    y, mean, rstd = run_forward(norm, shape, host, offset=2)
    check_forward(shape, "bf16", "none", v, to_f32(y, "bf16"), mean, rstd)


def test_a_large_mean_leaves_the_variance_its_digits(gpu):
    """Values of 1000 +- 1: E[x^2] - E[x]^2 in f32 would be off by 0.1."""
    shape = (2, 5000, 16, 2)
    rng = np.random.default_rng(3)
    x = (1000 + rng.standard_normal(shape[:3])).astype(np.float32)
    host = {"x": x, "gamma": np.ones(16, np.float32), "beta": np.zeros(16, np.float32)}
    y, mean, rstd = run_forward(ha.GroupNorm(*shape, "f32", epsilon=EPSILON), shape, host)
    wmean, wrstd = oracle.statistics(x, 2, EPSILON)
    # rounding of the mean: 1000 * 2^-24 * (chain of additions, far below 100 here); its square is what the variance sees
    assert np.abs(mean - wmean).max() < 1000 * 100 * 2.0 ** -24
    assert np.abs(rstd / wrstd - 1).max() < 1e-4


@pytest.mark.parametrize("shape", [(3, 50, 32, 4), (3, 6000, 16, 2)])
def test_a_sample_that_is_not_finite_stays_by_itself(gpu, shape):
    host, v, _, _ = inputs(shape, "f32", "f32", "silu", seed=4)
    norm = ha.GroupNorm(*shape, "f32", activation="silu", epsilon=EPSILON)
    clean = run_forward(norm, shape, host)
    d = shape[2] // shape[3]
    for bad in (np.nan, np.inf, -np.inf):
        spoilt = dict(host, x=host["x"].copy())
        spoilt["x"][1, 7, 0] = bad
        y, mean, rstd = run_forward(norm, shape, spoilt)
        assert np.isnan(y[1, :, :d]).all() and np.isnan(rstd[1, 0])
        y[1, :, :d], clean_y = clean[0][1, :, :d], clean[0]
        assert np.array_equal(y, clean_y)


def test_an_empty_batch_has_gradients_of_zero(gpu):
    norm = ha.GroupNorm(0, 9, 70, 7, "f32")
    norm.forward(None, None, None, None)
    dgamma, dbeta = device(np.ones(70, np.float32)), device(np.ones(70, np.float32))
    norm.backward(None, None, None, None, None, None, None, address(dgamma), address(dbeta))
    like = np.zeros(70, np.float32)
    assert not back(dgamma, like).any() and not back(dbeta, like).any()


def test_results_are_the_same_from_call_to_call_and_from_stream_to_stream(gpu):
    shape = (8, 784, 128, 32)
    norm = ha.GroupNorm(*shape, "bf16", activation="relu", epsilon=EPSILON)
    host, v, mean, rstd = inputs(shape, "bf16", "f32", "relu", seed=6)
    first, grads = run_forward(norm, shape, host), run_backward(norm, shape, host, mean, rstd)
    for stream in (None, ha.Stream()):
        for a, b in zip(run_forward(norm, shape, host, stream=stream), first):
            assert np.array_equal(a, b)
    for a, b in zip(run_backward(norm, shape, host, mean, rstd), grads):
        assert np.array_equal(a, b)


def test_streams_that_overlap_have_scratch_of_their_own(gpu):
    shape = (2, 20000, 48, 4)
    norm = ha.GroupNorm(*shape, "f32", epsilon=EPSILON)
    cases = [inputs(shape, "f32", "f32", "none", seed=s)[0] for s in (7, 8)]
    want = [run_forward(norm, shape, host)[0] for host in cases]
    streams = [ha.Stream(), ha.Stream()]
    bufs = [[device(h[k]) for k in ("x", "gamma", "beta")] + [empty(h["x"].shape, np.float32)] for h in cases]
    for _ in range(10):
        for b, s in zip(bufs, streams):
            norm.forward(*map(address, b), stream=s)
    for b, s, w in zip(bufs, streams, want):
        s.synchronize()
        assert np.array_equal(back(b[3], w), w)


@pytest.mark.parametrize("activation", ["none", "silu"])
@pytest.mark.parametrize("shape", [(2, 60, 24, 4), (1, 5000, 16, 4)])
def test_the_gradient_is_that_of_the_forward_pass(gpu, shape, activation):
    """Along a direction d, <dx, d> is the slope of <y, dy>, by central differences of the kernel's own forward pass."""
    norm = ha.GroupNorm(*shape, "f32", activation=activation, epsilon=EPSILON)
    host, v, _, _ = inputs(shape, "f32", "f32", activation, seed=9)
    _, mean, rstd = run_forward(norm, shape, host)
    grads = dict(zip(("x", "gamma", "beta"), run_backward(norm, shape, host, mean, rstd)))
    rng, h = np.random.default_rng(10), 2.0 ** -7
    for name, gradient in grads.items():
        d = np.sign(gradient + 1e-30).astype(np.float32)   # so that the slope is the sum of |gradient|, far above rounding
        loss = []
        for s in (h, -h):
            y = run_forward(norm, shape, dict(host, **{name: host[name] + np.float32(s) * d}))[0]
            loss.append((y.astype(np.float64) * host["dy"]).sum())
        slope, want = (loss[0] - loss[1]) / (2 * h), np.abs(gradient.astype(np.float64)).sum()
        # differences: third derivatives over 6 h^2 = 1e-5; rounding of y: 2^-24 sum |y dy| / h, 1e-5 of a slope of that size
        assert abs(slope - want) < 2e-3 * want, (name, slope, want)


def test_a_captured_call_replays(gpu):
    """Forward and backward recorded into a HIP graph (after one call that allocates the stream's scratch), replayed with other
    work in between."""
    torch = pytest.importorskip("torch")
    shape = (4, 3000, 32, 8)
    norm = ha.GroupNorm(*shape, "f32", activation="silu", epsilon=EPSILON)
    host, v, mean, rstd = inputs(shape, "f32", "f32", "silu", seed=11)
    want = run_forward(norm, shape, host)[0], run_backward(norm, shape, host, mean, rstd)
    t = {k: torch.from_numpy(a.copy()).cuda() for k, a in dict(host, mean=mean, rstd=rstd).items()}
    y, dx = torch.zeros_like(t["x"]), torch.zeros_like(t["x"])
    dgamma, dbeta = torch.zeros(32, device="cuda"), torch.zeros(32, device="cuda")

    s = ha.Stream()
    stream = torch.cuda.ExternalStream(ha._ffi.lib.he_stream_raw(s.handle))
    at = lambda *names: [t[k].data_ptr() for k in names]  # noqa: E731

    def both():
        norm.forward(*at("x", "gamma", "beta"), y.data_ptr(), stream=s)
        norm.backward(*at("dy", "x", "gamma", "beta", "mean", "rstd"), dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), stream=s)

    torch.cuda.synchronize()
    both()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        both()
    for _ in range(4):
        for v in (y, dx, dgamma, dbeta):
            v.fill_(7.0)
        run_forward(norm, shape, host)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(y.cpu().numpy(), want[0])
        for a, b in zip((dx, dgamma, dbeta), want[1]):
            assert np.array_equal(a.cpu().numpy(), b)
