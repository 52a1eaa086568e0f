"""Products in 8-bit integers through the C ABI on the GPU against the oracle, and together with what makes their operands."""
import numpy as np
import pytest

import helium_amd as ha
from device_arrays import Array, at, empty
from group_norm_cases import to_f32, to_storage
from helium_amd.int8 import pitch
from int8_cases import SMALL, check, inputs
from oracle import int8 as oracle
from oracle import rms_norm as oracle_norm
from rms_norm_cases import EPSILON

pytestmark = pytest.mark.gpu

DTYPES = ("f32", "bf16", "f16")
# tokens, inputs, channels
SIZES = SMALL + [(1, 4096, 4096), (5, 1000, 3001), (16, 11000, 200), (24, 513, 1030), (48, 4096, 1000), (64, 100, 2000), (65, 4096, 512), (130, 777, 1203),
                 (333, 1203, 777), (512, 2048, 2048), (1000, 129, 515), (2000, 512, 1024), (2050, 1000, 2060), (3, 131071, 40), (100, 70000, 130), (20000, 33, 20)]


def multiply(op, host, dtype, stream=None):
    d = {k: None if a is None else Array(a) for k, a in host.items()}
    y = empty((len(host["x"]), len(host["weights"])), np.float32 if dtype == "f32" else np.uint16)
    op.multiply(len(host["x"]), *[d[k].at for k in ("x", "x_scales", "weights", "weight_scales")], y.at, bias=at(d["bias"]), stream=stream)
    if stream is not None:
        stream.synchronize()
    return y.back()


@pytest.mark.parametrize("k", range(len(SIZES)))
def test_products_match_the_oracle(gpu, k):
    tokens, columns, channels = SIZES[k]
    dtype = DTYPES[k % 3]
    host = inputs(tokens, columns, channels, bias=k % 2, seed=k)
    check(host, dtype, to_f32(multiply(ha.Int8Matmul(columns, channels, dtype), host, dtype), dtype))


@pytest.mark.parametrize("size", [(70, 700, 130), (300, 513, 520), (257, 8192, 300), (33, 9000, 77)])
@pytest.mark.parametrize("shares", [1, 2, 4])
@pytest.mark.parametrize("shape", range(9))
def test_every_shape_and_cut(gpu, monkeypatch, shape, shares, size):
    monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", str(shape + 1))
    monkeypatch.setenv("HELIUM_HIP_INT8_SHARES", str(shares))
    tokens, columns, channels = size
    dtype = DTYPES[shape % 3]
    host = inputs(tokens, columns, channels, bias=True, seed=shape)
    check(host, dtype, to_f32(multiply(ha.Int8Matmul(columns, channels, dtype), host, dtype), dtype))


@pytest.mark.parametrize("shape", range(4))
def test_every_count_of_k_tiles(gpu, monkeypatch, shape):
    """None to several rounds of a tile's ring, and what is left behind the last; rows that end inside a k-tile."""
    monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", str(shape + 1))
    monkeypatch.setenv("HELIUM_HIP_INT8_SHARES", "1")
    for count in range(1, 18):
        columns = count * 128 - (0, 1, 127, 112, 50)[count % 5]
        host = inputs(150, columns, 270, bias=True, seed=count)
        check(host, "f32", multiply(ha.Int8Matmul(columns, 270, "f32"), host, "f32"))


@pytest.mark.parametrize("tokens", [40, 300])
def test_no_cut_changes_a_bit(gpu, monkeypatch, tokens):
    host = inputs(tokens, 8300, 130, bias=True, seed=6)
    op = ha.Int8Matmul(8300, 130, "f32")
    want = multiply(op, host, "f32")
    for shape in range(9):
        for shares in (1, 2, 4):
            monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", str(shape + 1))
            monkeypatch.setenv("HELIUM_HIP_INT8_SHARES", str(shares))
            assert np.array_equal(multiply(op, host, "f32"), want), (shape, shares)


@pytest.mark.parametrize("tokens,columns,channels", [(1, 8192, 64), (40, 6000, 64), (300, 9000, 300)])
def test_the_largest_sums_are_exact(gpu, tokens, columns, channels):
    """Every product 127 * 127, and sums far beyond the 24 bits of f32 (of which the result keeps the first)."""
    host = inputs(tokens, columns, channels, bias=False, seed=1)
    host["x"][:, :columns], host["weights"][:, :columns] = 127, 127
    host["weights"][1::2, :columns] = -127
    check(host, "f32", multiply(ha.Int8Matmul(columns, channels, "f32"), host, "f32"))


def test_scales_that_are_not_finite_stay_in_their_rows(gpu):
    host = inputs(70, 300, 50, bias=True, seed=2)
    clean = multiply(ha.Int8Matmul(300, 50, "f32"), host, "f32")
    host["x_scales"][3], host["weight_scales"][7] = np.nan, np.nan
    y = multiply(ha.Int8Matmul(300, 50, "f32"), host, "f32")
    assert np.isnan(y[3]).all() and np.isnan(y[:, 7]).all()
    rest = np.ones(y.shape, bool)
    rest[3], rest[:, 7] = False, False
    assert np.array_equal(y[rest], clean[rest])


@pytest.mark.parametrize("tokens", [1, 30, 200])
def test_a_quantized_layer(gpu, tokens):
    """A residual stream normalised into 8 bits and multiplied, and its result quantised and multiplied again: what a served layer does."""
    columns, wide = 700, 1030
    rng = np.random.default_rng(tokens)
    x, residual = (to_storage(rng.standard_normal((tokens, columns)) * s, "bf16") for s in (1.0, 2.0))
    gamma = (1 + 0.3 * rng.standard_normal(columns)).astype(np.float32)
    up, down = (rng.standard_normal(s).astype(np.float32) / 30 for s in ((wide, columns), (columns, wide)))
    quantized = []
    for w in (up, down):
        q, scales = empty((len(w), pitch(w.shape[1])), np.int8), empty((len(w),), np.float32)
        whole = Array(w)
        ha.QuantizeRows(w.shape[1], "f32").quantize(len(w), whole.at, q.at, scales.at)
        want, want_scales = oracle.quantize(w)
        assert np.array_equal(q.back()[:, :w.shape[1]], want) and np.array_equal(scales.back(), want_scales)
        quantized.append((q, scales))
    h, y1, y2 = empty((tokens, columns), np.uint16), empty((tokens, wide), np.uint16), empty((tokens, columns), np.uint16)
    q1, s1, q2, s2 = empty((tokens, pitch(columns)), np.int8), empty((tokens,), np.float32), empty((tokens, pitch(wide)), np.int8), empty((tokens,), np.float32)
    dx, dgamma, dresidual = Array(x), Array(gamma), Array(residual)
    ha.RmsNorm(columns, "bf16", residual_dtype="bf16", output="i8", epsilon=EPSILON).forward(
        tokens, dx.at, dgamma.at, q1.at, residual=dresidual.at, new_residual=h.at, scales=s1.at)
    ha.Int8Matmul(columns, wide, "bf16").multiply(tokens, q1.at, s1.at, *[a.at for a in quantized[0]], y1.at)
    ha.QuantizeRows(wide, "bf16").quantize(tokens, y1.at, q2.at, s2.at)
    ha.Int8Matmul(wide, columns, "bf16").multiply(tokens, q2.at, s2.at, *[a.at for a in quantized[1]], y2.at)
    # each step against the oracle's, from what the step before left
    hv = to_f32(x, "bf16") + to_f32(residual, "bf16")
    assert (h.back() == to_storage(hv, "bf16")).all()
    check({"x": q1.back(), "x_scales": s1.back(), "weights": quantized[0][0].back(), "weight_scales": quantized[0][1].back(), "bias": None}, "bf16", to_f32(y1.back(), "bf16"))
    want, want_scales = oracle.quantize(to_f32(y1.back(), "bf16"))
    assert np.array_equal(q2.back()[:, :wide], want) and np.array_equal(s2.back(), want_scales)
    check({"x": q2.back(), "x_scales": s2.back(), "weights": quantized[1][0].back(), "weight_scales": quantized[1][1].back(), "bias": None}, "bf16", to_f32(y2.back(), "bf16"))
    # and the whole against unquantised products: an operand is off by at most half a step, A / 254 of its row's largest
    y, _ = oracle_norm.forward(to_f32(h.back(), "bf16"), gamma, EPSILON)
    exact = y @ up.astype(np.float64).T
    most = lambda a: np.abs(a).max(axis=1, keepdims=True) / 254  # noqa: E731
    off = most(y) @ np.abs(up).sum(axis=1)[None] + np.abs(y).sum(axis=1, keepdims=True) @ most(up).T + columns * most(y) @ most(up).T
    assert (np.abs(to_f32(y1.back(), "bf16") - exact) <= 1.01 * off + 2.0 ** -8 * np.abs(exact)).all()


def test_calls_on_streams_that_overlap(gpu, monkeypatch):
    monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", "4")
    monkeypatch.setenv("HELIUM_HIP_INT8_SHARES", "4")
    op = ha.Int8Matmul(3000, 128, "f32")
    assert "shares=4" in op.describe(130)
    cases = [inputs(130, 3000, 128, False, seed=s) for s in (3, 4)]
    want = [multiply(op, h, "f32") for h in cases]
    streams = [ha.Stream(), ha.Stream()]
    operands = [[Array(h[k]) for k in ("x", "x_scales", "weights", "weight_scales")] + [empty((130, 128), np.float32)] for h in cases]
    for _ in range(10):
        for o, s in zip(operands, streams):
            op.multiply(130, *[a.at for a in o], stream=s)
    for o, s, w in zip(operands, streams, want):
        s.synchronize()
        assert np.array_equal(o[4].back(), w)


@pytest.mark.parametrize("tokens", [2, 40, 150])
def test_a_captured_call_replays(gpu, tokens):
    torch = pytest.importorskip("torch")
    op = ha.Int8Matmul(1500, 200, "f32")
    host = inputs(tokens, 1500, 200, True, seed=5)
    want = multiply(op, host, "f32")
    t = {k: torch.from_numpy(a.copy()).cuda() for k, a in host.items()}
    y = torch.zeros(tokens, 200, device="cuda")
    s = ha.Stream()
    stream = torch.cuda.ExternalStream(ha._ffi.lib.he_stream_raw(s.handle))
    call = lambda: op.multiply(tokens, *[t[k].data_ptr() for k in ("x", "x_scales", "weights", "weight_scales")], y.data_ptr(), bias=t["bias"].data_ptr(), stream=s)  # noqa: E731
    torch.cuda.synchronize()
    call()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for _ in range(4):
        y.fill_(7.0)
        multiply(op, host, "f32")
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(y.cpu().numpy(), want)


# 16-wave streams take 4096 bytes of k to a share, others 2048, tiles 512
@pytest.mark.parametrize("size", [(70, 16500, 130), (33, 16390, 77), (257, 17000, 300)])
@pytest.mark.parametrize("shares", [2, 4])
@pytest.mark.parametrize("shape", range(9))
def test_every_shape_and_cut_is_the_one_that_is_named(gpu, monkeypatch, shape, shares, size):
    tokens, columns, channels = size
    dtype = DTYPES[(shape + 1) % 3]
    host = inputs(tokens, columns, channels, bias=True, seed=shape)
    op, results = ha.Int8Matmul(columns, channels, dtype), []
    for of in (1, shares):
        monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", str(shape + 1))
        monkeypatch.setenv("HELIUM_HIP_INT8_SHARES", str(of))
        assert f" shape={shape} " in op.describe(tokens) and f" shares={of} " in op.describe(tokens)
        results.append(multiply(op, host, dtype))
    check(host, dtype, to_f32(results[0], dtype))
    assert np.array_equal(*results)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [40, 300])
def test_no_cut_of_long_sums_changes_a_bit(gpu, monkeypatch, tokens, dtype):
    host = inputs(tokens, 16600, 130, bias=True, seed=6)
    host["x_scales"] *= np.float32(2e-4)   # (results that f16 has too)
    op = ha.Int8Matmul(16600, 130, dtype)
    want = multiply(op, host, dtype)
    assert np.isfinite(to_f32(want, dtype)).all()
    for shape in range(9):
        for shares in (1, 2, 4):
            monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", str(shape + 1))
            monkeypatch.setenv("HELIUM_HIP_INT8_SHARES", str(shares))
            assert f" shape={shape} " in op.describe(tokens) and f" shares={shares} " in op.describe(tokens)
            assert np.array_equal(multiply(op, host, dtype), want), (shape, shares)
