"""Rms norm and quantised rows through the C ABI on the GPU against the 64-bit oracle."""
import numpy as np
import pytest

import helium_amd as ha
from device_arrays import Array, at, empty
from group_norm_cases import to_f32, to_storage
from helium_amd.int8 import pitch
from oracle import int8 as oracle_int8
from rms_norm_cases import BEYOND, EPSILON, LARGE, SHAPES, TYPES, beyond, check_backward, check_beyond, check_forward, check_quantized_beyond, check_quantized_norm, inputs
from test_rms_norm_cpu import borders

pytestmark = pytest.mark.gpu


def run_forward(norm, rows, host, residual, to_i8=False, in_place=False, stream=None, offset=0):
    """y, h, rstd and scales"""
    x, gamma = Array(host["x"], offset), Array(host["gamma"])
    r = Array(host["residual"]) if residual else None
    h = None if not residual else r if in_place else empty(r.like.shape, r.like.dtype)
    y = empty((rows, pitch(norm.columns)), np.int8) if to_i8 else x if in_place else empty(x.like.shape, x.like.dtype, offset)
    rstd, scales = empty((rows,), np.float32), empty((rows,), np.float32)
    norm.forward(rows, x.at, gamma.at, y.at, residual=at(r), new_residual=at(h), rstd=rstd.at, scales=scales.at if to_i8 else None, stream=stream)
    if stream is not None:
        stream.synchronize()
    return y.back(), h.back() if residual else None, rstd.back(), scales.back()


def run_backward(norm, rows, host, residual, both=True, into=None):
    """dx, dresidual, dgamma; into: the operand whose place dx takes"""
    d = {k: Array(host[k]) for k in ("dy", "h", "gamma", "rstd")}
    dh = Array(host["dh"]) if residual else None
    dx = d[into] if into else empty(host["x"].shape, host["x"].dtype)
    dresidual = empty(host["h"].shape, host["h"].dtype) if residual and both else None
    dgamma = empty((norm.columns,), np.float32)
    norm.backward(rows, d["dy"].at, d["h"].at, d["gamma"].at, d["rstd"].at, dx.at, dgamma.at, dh=at(dh), dresidual=at(dresidual))
    return dx.back(), dresidual.back() if dresidual else None, dgamma.back()


@pytest.mark.parametrize("shape,types", [(s, TYPES[(k + j) % len(TYPES)]) for k, s in enumerate(SHAPES + LARGE) for j in (0, 3, 5)])
def test_forward_and_backward_match_the_oracle(gpu, shape, types):
    (rows, columns), (dtype, residual) = shape, types
    param = dtype if rows % 2 else "f32"
    host, v = inputs(rows, columns, dtype, residual, param, seed=columns)
    norm = ha.RmsNorm(columns, dtype, residual_dtype=residual, param_dtype=param, epsilon=EPSILON)
    y, h, rstd, _ = run_forward(norm, rows, host, residual)
    check_forward(dtype, v, to_f32(y, dtype), rstd)
    assert not residual or np.array_equal(h, host["h"])
    dx, dresidual, dgamma = run_backward(norm, rows, host, residual)
    check_backward(dtype, residual, v, to_f32(dx, dtype), to_f32(dresidual, residual) if residual else None, dgamma, -(-rows // 256))


@pytest.mark.parametrize("shape,types", [(s, TYPES[k % len(TYPES)]) for k, s in enumerate(SHAPES + LARGE)])
def test_the_norm_into_8_bits_matches_the_oracle(gpu, shape, types):
    (rows, columns), (dtype, residual) = shape, types
    host, v = inputs(rows, columns, dtype, residual, "f32", seed=columns + 1)
    norm = ha.RmsNorm(columns, dtype, residual_dtype=residual, output="i8", epsilon=EPSILON)
    q, h, _, scales = run_forward(norm, rows, host, residual, to_i8=True)
    check_quantized_norm(v, q, scales)
    assert not residual or np.array_equal(h, host["h"])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1, 1), (9, 3), (8, 64), (10, 130), (7, 517), (1100, 4096), (3000, 1203), (2, 32767)])
def test_quantized_rows_are_the_oracles(gpu, shape, dtype):
    rows, columns = shape
    x = borders(rows, columns, dtype, columns)
    want, want_scales = oracle_int8.quantize(to_f32(x, dtype))
    d, q, scales = Array(x), empty((rows, pitch(columns)), np.int8), empty((rows,), np.float32)
    ha.QuantizeRows(columns, dtype).quantize(rows, d.at, q.at, scales.at)
    got = q.back()
    assert np.array_equal(got[:, :columns], want) and not got[:, columns:].any()
    assert np.array_equal(scales.back(), want_scales, equal_nan=True)


@pytest.mark.parametrize("shape", [(3, 100), (5, 2867), (2, 4096), (1500, 515)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_results_may_take_an_operands_place(gpu, shape, dtype):
    rows, columns = shape
    host, v = inputs(rows, columns, dtype, dtype, "f32", seed=3)
    norm = ha.RmsNorm(columns, dtype, residual_dtype=dtype, epsilon=EPSILON)
    for a, b in zip(run_forward(norm, rows, host, dtype, in_place=True), run_forward(norm, rows, host, dtype)):
        assert np.array_equal(a, b)
    apart = run_backward(norm, rows, host, dtype)
    for into in ("dy", "h"):
        for a, b in zip(run_backward(norm, rows, host, dtype, into=into), apart):
            assert np.array_equal(a, b)
    # the residual's gradient in dh's place, and no dx
    d = {k: Array(host[k]) for k in ("dy", "h", "gamma", "rstd", "dh")}
    dgamma = empty((columns,), np.float32)
    norm.backward(rows, d["dy"].at, d["h"].at, d["gamma"].at, d["rstd"].at, None, dgamma.at, dh=d["dh"].at, dresidual=d["dh"].at)
    assert np.array_equal(d["dh"].back(), apart[1]) and np.array_equal(dgamma.back(), apart[2])
    # nothing but this norm reads h
    norm.backward(rows, d["dy"].at, d["h"].at, d["gamma"].at, d["rstd"].at, d["dy"].at, dgamma.at)
    alone = dict(v)
    del alone["dh"]
    check_backward(dtype, dtype, alone, to_f32(d["dy"].back(), dtype), None, dgamma.back(), -(-rows // 256))


def test_operands_need_no_more_than_their_rows_alignment(gpu):
    host, v = inputs(30, 257, "bf16", None, "f32", seed=4)
    y, _, rstd, _ = run_forward(ha.RmsNorm(257, "bf16", epsilon=EPSILON), 30, host, None, offset=2)
    check_forward("bf16", v, to_f32(y, "bf16"), rstd)


def test_a_row_that_is_not_finite_stays_by_itself(gpu):
    rows, columns = 1100, 700
    host, v = inputs(rows, columns, "f32", None, "f32", seed=5)
    norm, eight = ha.RmsNorm(columns, "f32", epsilon=EPSILON), ha.RmsNorm(columns, "f32", output="i8", epsilon=EPSILON)
    clean, clean8 = run_forward(norm, rows, host, None), run_forward(eight, rows, host, None, to_i8=True)
    for bad in (np.nan, np.inf, -np.inf):
        spoilt = dict(host, x=host["x"].copy())
        spoilt["x"][1, 7] = bad
        y, _, rstd, _ = run_forward(norm, rows, spoilt, None)
        assert np.isnan(y[1, 7]) and np.array_equal(np.delete(y, 1, 0), np.delete(clean[0], 1, 0))
        q, _, _, scales = run_forward(eight, rows, spoilt, None, to_i8=True)
        assert np.isnan(scales[1]) and not q[1].any()
        assert np.array_equal(np.delete(q, 1, 0), np.delete(clean8[0], 1, 0)) and np.array_equal(np.delete(scales, 1), np.delete(clean8[3], 1))


def test_rows_of_zeros(gpu):
    host = {"x": np.zeros((3, 40), np.float32), "gamma": np.ones(40, np.float32)}
    y, _, rstd, _ = run_forward(ha.RmsNorm(40, "f32", epsilon=EPSILON), 3, host, None)
    assert not y.any() and np.allclose(rstd, EPSILON ** -0.5, rtol=1e-6)
    q, _, _, scales = run_forward(ha.RmsNorm(40, "f32", output="i8", epsilon=EPSILON), 3, host, None, to_i8=True)
    assert not q.any() and not scales.any()


def test_no_rows(gpu):
    norm = ha.RmsNorm(70, "bf16")
    norm.forward(0, None, None, None)
    dgamma = empty((70,), np.float32)
    norm.backward(0, None, None, None, None, None, dgamma.at)
    assert not dgamma.back().any()


@pytest.mark.parametrize("columns", [60, 3001])
def test_the_gradient_is_that_of_the_forward_pass(gpu, columns):
    """Along a direction d, <dh, d> is the slope of <y, dy>, by central differences of the kernel's own forward pass."""
    rows = 4
    host, v = inputs(rows, columns, "f32", None, "f32", seed=6)
    norm = ha.RmsNorm(columns, "f32", epsilon=EPSILON)
    host["rstd"] = run_forward(norm, rows, host, None)[2]
    dx, _, dgamma = run_backward(norm, rows, host, None)
    h = 2.0 ** -7
    for name, gradient in (("x", dx), ("gamma", dgamma)):
        d = np.sign(gradient + 1e-30).astype(np.float32)
        loss = [(run_forward(norm, rows, dict(host, **{name: host[name] + np.float32(s) * d}), None)[0].astype(np.float64) * host["dy"]).sum() for s in (h, -h)]
        slope, want = (loss[0] - loss[1]) / (2 * h), np.abs(gradient.astype(np.float64)).sum()
        # differences: third derivatives over 6 h^2 = 1e-5; rounding of y: 2^-24 sum |y dy| / h, 1e-5 of a slope of that size
        assert abs(slope - want) < 2e-3 * want, (name, slope, want)


def test_streams_that_overlap_have_scratch_of_their_own(gpu):
    rows, columns = 4000, 515
    norm = ha.RmsNorm(columns, "f32", epsilon=EPSILON)
    cases = [inputs(rows, columns, "f32", None, "f32", seed=s)[0] for s in (7, 8)]
    want = [run_backward(norm, rows, host, None)[2] for host in cases]
    streams = [ha.Stream(), ha.Stream()]
    operands = [[Array(h[k]) for k in ("dy", "h", "gamma", "rstd")] + [empty(h["x"].shape, np.float32), empty((columns,), np.float32)] for h in cases]
    for _ in range(10):
        for o, s in zip(operands, streams):
            norm.backward(rows, *[a.at for a in o], stream=s)
    for o, s, w in zip(operands, streams, want):
        s.synchronize()
        assert np.array_equal(o[5].back(), w)


def test_a_captured_call_replays(gpu):
    torch = pytest.importorskip("torch")
    rows, columns = 1200, 300
    norm, eight = ha.RmsNorm(columns, "f32", residual_dtype="f32", epsilon=EPSILON), ha.RmsNorm(columns, "f32", residual_dtype="f32", output="i8", epsilon=EPSILON)
    host, v = inputs(rows, columns, "f32", "f32", "f32", seed=9)
    want = run_forward(norm, rows, host, "f32")[0], run_backward(norm, rows, host, "f32")[1:], run_forward(eight, rows, host, "f32", to_i8=True)[0]
    t = {k: torch.from_numpy(a.copy()).cuda() for k, a in host.items()}
    y, h, dx, dr = (torch.zeros_like(t["x"]) for _ in range(4))
    dgamma, scales, q = torch.zeros(columns, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(rows, pitch(columns), dtype=torch.int8, device="cuda")
    s = ha.Stream()
    stream = torch.cuda.ExternalStream(ha._ffi.lib.he_stream_raw(s.handle))
    p = {k: a.data_ptr() for k, a in t.items()}

    def all_of_it():
        norm.forward(rows, p["x"], p["gamma"], y.data_ptr(), residual=p["residual"], new_residual=h.data_ptr(), stream=s)
        eight.forward(rows, p["x"], p["gamma"], q.data_ptr(), residual=p["residual"], new_residual=h.data_ptr(), scales=scales.data_ptr(), stream=s)
        norm.backward(rows, p["dy"], h.data_ptr(), p["gamma"], p["rstd"], dx.data_ptr(), dgamma.data_ptr(), dh=p["dh"], dresidual=dr.data_ptr(), stream=s)

    torch.cuda.synchronize()
    all_of_it()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        all_of_it()
    for _ in range(4):
        for a in (y, h, dx, dr, dgamma, scales, q):
            a.fill_(7)
        run_backward(norm, rows, host, "f32")
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(y.cpu().numpy(), want[0]) and np.array_equal(q.cpu().numpy(), want[2])
        for a, b in zip((dr, dgamma), want[1]):
            assert np.array_equal(a.cpu().numpy(), b)


def test_later_calls_on_a_stream_allocate_nothing_whatever_their_rows(gpu):
    """The first call is of one row, which needs no workgroup's shares; what follows is captured, of more rows than workgroups."""
    torch = pytest.importorskip("torch")
    rows, columns = 1000, 32760   # (the scratch of 256 workgroups is 33 MB)
    norm = ha.RmsNorm(columns, "bf16", epsilon=EPSILON)
    host, _ = inputs(rows, columns, "bf16", None, "f32", seed=11)
    want = run_backward(norm, rows, host, None)
    norm = ha.RmsNorm(columns, "bf16", epsilon=EPSILON)
    t = {k: torch.from_numpy(host[k].copy()).cuda() for k in ("dy", "h", "gamma", "rstd")}
    dx, dgamma = torch.zeros_like(t["dy"]), torch.zeros(columns, device="cuda")
    s = ha.Stream()
    stream = torch.cuda.ExternalStream(ha._ffi.lib.he_stream_raw(s.handle))
    call = lambda n: norm.backward(n, *[a.data_ptr() for a in (*t.values(), dx, dgamma)], stream=s)  # noqa: E731
    torch.cuda.synchronize()
    call(1)
    stream.synchronize()
    free = torch.cuda.mem_get_info()[0]
    call(300)
    stream.synchronize()
    assert torch.cuda.mem_get_info()[0] > free - (16 << 20)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call(rows)
    for _ in range(3):
        dx.fill_(7)
        dgamma.fill_(7)
        call(2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(dx.cpu().numpy(), want[0]) and np.array_equal(dgamma.cpu().numpy(), want[2])


def test_the_number_of_workgroups_is_not_the_environments(gpu, monkeypatch):
    """(A stream's scratch is sized by it.)"""
    rows, columns = 3000, 515
    norm = ha.RmsNorm(columns, "f32", epsilon=EPSILON)
    host, _ = inputs(rows, columns, "f32", None, "f32", seed=12)
    want = run_backward(norm, rows, host, None)
    for value in ("0", "4"):
        monkeypatch.setenv("HELIUM_HIP_ROWS_PER_CU", value)
        for a, b in zip(run_backward(norm, rows, host, None), want):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("rows,columns,dtype,residual,epsilon", BEYOND + [(40, 4096, "bf16", "bf16", 1e-5), (40, 12290, "f32", None, 0.0), (9, 32767, "bf16", "f32", 0.0), (700, 4096, "f32", "f32", 0.0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_whose_squares_are_beyond_f32(gpu, rows, columns, dtype, residual, epsilon, in_place):
    host, v = beyond(rows, columns, dtype, residual, epsilon, seed=columns)
    y, h, rstd, _ = run_forward(ha.RmsNorm(columns, dtype, residual_dtype=residual, epsilon=epsilon), rows, host, residual, in_place=in_place)
    check_beyond(dtype, v, epsilon, to_f32(y, dtype), rstd)
    assert not residual or np.array_equal(h, host["h"])
    if not in_place:
        q, h, _, scales = run_forward(ha.RmsNorm(columns, dtype, residual_dtype=residual, output="i8", epsilon=epsilon), rows, host, residual, to_i8=True)
        check_quantized_beyond(v, epsilon, q, scales)
        assert not residual or np.array_equal(h, host["h"])
