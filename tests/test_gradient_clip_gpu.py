"""Gradient clipping through the C ABI on the GPU against the 64-bit oracle, by itself and in a training step."""
import re

import numpy as np
import pytest

import helium_amd as ha
from device_arrays import Array, empty
from gradient_clip_cases import GROUPS, check, check_norm, inputs
from group_norm_cases import to_f32, to_storage
from oracle import gradient_clip as oracle
from oracle import muon as oracle_muon
from oracle import rms_norm as oracle_norm
from rms_norm_cases import EPSILON

pytestmark = pytest.mark.gpu

LARGE = [([3_000_001, 70_000, 5], ["f32", "bf16", "f16"]), ([20_000_003], ["bf16"]), ([1000] * 300, ["f16"] * 300), ([1 << 22, 0, (1 << 22) + 1], ["f32", "f16", "f32"])]


def clipped(clip, host, most, in_place=False, offset=0, stream=None):
    d = [Array(h, offset) for h in host]
    out = d if in_place else [empty(h.shape, h.dtype, offset) for h in host]
    norm = empty((1,), np.float32)
    clip.clip([a.at for a in d], [a.at for a in out], most, norm.at, stream=stream)
    if stream is not None:
        stream.synchronize()
    return [a.back() for a in out], norm.back()[0]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("most", [0.5, 1e6])
@pytest.mark.parametrize("k", range(len(GROUPS + LARGE)))
def test_clipping_matches_the_oracle(gpu, k, most, in_place):
    sizes, dtypes = (GROUPS + LARGE)[k]
    host, values = inputs(sizes, dtypes, 0.3, seed=k)
    clip = ha.GradientClip(sizes, dtypes)
    got, norm = clipped(clip, host, most, in_place)
    check(dtypes, values, most, got, norm)
    d, alone = [Array(h) for h in host], empty((1,), np.float32)
    clip.norm([a.at for a in d], alone.at)
    assert alone.back()[0] == norm


@pytest.mark.parametrize("offset", [2, 4, 8, 14])
def test_tensors_begin_at_any_whole_value(gpu, offset):
    sizes, dtypes = [5000, 7, 16385], ["bf16", "f16", "bf16"]
    host, values = inputs(sizes, dtypes, 0.3, seed=1)
    got, norm = clipped(ha.GradientClip(sizes, dtypes), host, 0.5, offset=offset)
    check(dtypes, values, 0.5, got, norm)


@pytest.mark.parametrize("size", [1e-38, 1e-20, 1e20, 1e36])
def test_the_norm_neither_vanishes_nor_overflows(gpu, size):
    sizes, dtypes = [1000, 999], ["f32", "bf16"]
    host, values = inputs(sizes, dtypes, size, seed=2)
    got, norm = clipped(ha.GradientClip(sizes, dtypes), host, 1.0)
    check(dtypes, values, 1.0, got, norm)


@pytest.mark.parametrize("size,most", [(1e37, 1e-3), (1e37, 1e-6), (3e36, 1e-30), (1e30, 1e-3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_factors_that_f32_holds_with_few_bits_or_none(gpu, size, most, in_place):
    sizes, dtypes = [70_000, 301, 50_001], ["f32", "bf16", "f32"]
    host, values = inputs(sizes, dtypes, size, seed=12)
    most = float(np.float32(most))   # (as the call has it)
    got, norm = clipped(ha.GradientClip(sizes, dtypes), host, most, in_place)
    check(dtypes, values, most, got)
    if oracle.norm(values) > np.finfo(np.float32).max:   # (beyond which f32 has infinity)
        assert np.isposinf(norm)
    else:
        check_norm(values, norm)


def test_no_values_and_zeros(gpu):
    norm = empty((1,), np.float32)
    for sizes in ([], [0, 0]):
        clip = ha.GradientClip(sizes, "f32")
        clip.clip([None] * len(sizes), [None] * len(sizes), 1.0, norm.at)
        assert norm.back()[0] == 0
        clip.norm([None] * len(sizes), norm.at)
        assert norm.back()[0] == 0
    got, n = clipped(ha.GradientClip([100], "f32"), [np.zeros(100, np.float32)], 1.0)
    assert n == 0 and not got[0].any()
    # nothing is left of gradients that may have no norm
    got, n = clipped(ha.GradientClip([100], "f32"), [np.ones(100, np.float32)], 0.0)
    assert n == 10 and not got[0].any()
    got, n = clipped(ha.GradientClip([100], "f32"), [np.ones(100, np.float32)], np.inf)
    assert n == 10 and (got[0] == 1).all()


def test_norms_that_are_not_finite_are_told(gpu):
    host, values = inputs([3000, 40], ["f32", "bf16"], 0.3, seed=3)
    clip = ha.GradientClip([3000, 40], ["f32", "bf16"])
    for bad in (np.nan, np.inf):
        spoilt = [host[0].copy(), host[1]]
        spoilt[0][77] = bad
        got, norm = clipped(clip, spoilt, 1.0)
        if np.isnan(bad):
            assert np.isnan(norm) and np.isnan(got[0]).all() and np.isnan(to_f32(got[1], "bf16")).all()
        else:
            assert np.isinf(norm) and np.isnan(got[0][77]) and not np.delete(got[0], 77).any() and not to_f32(got[1], "bf16").any()


def test_nothing_is_clipped_to_infinity(gpu):
    host, values = inputs([3000, 40], ["f32", "bf16"], 0.3, seed=8)
    clip = ha.GradientClip([3000, 40], ["f32", "bf16"])
    for bad in (0.5, np.nan, np.inf):
        host[0][77] = bad
        for in_place in (False, True):
            got, norm = clipped(clip, host, np.inf, in_place)
            assert all(np.array_equal(g, h, equal_nan=True) for g, h in zip(got, host))
            assert np.isfinite(norm) == np.isfinite(bad)


def test_results_are_the_same_from_call_to_call_and_overlapping_streams(gpu):
    sizes, dtypes = [300_000, 11, 5000], ["f32", "bf16", "f16"]
    clip = ha.GradientClip(sizes, dtypes)
    cases = [inputs(sizes, dtypes, 0.3, seed=s)[0] for s in (4, 5)]
    want = [clipped(clip, h, 0.5) for h in cases]
    streams = [ha.Stream(), ha.Stream()]
    d = [([Array(a) for a in h], [empty(a.shape, a.dtype) for a in h], empty((1,), np.float32)) for h in cases]
    for _ in range(10):
        for (i, o, n), s in zip(d, streams):
            clip.clip([a.at for a in i], [a.at for a in o], 0.5, n.at, stream=s)
    for (i, o, n), s, w in zip(d, streams, want):
        s.synchronize()
        assert n.back()[0] == w[1] and all(np.array_equal(a.back(), b) for a, b in zip(o, w[0]))


def test_a_captured_call_replays(gpu):
    torch = pytest.importorskip("torch")
    sizes, dtypes = [100_000, 333], ["f32", "f32"]
    clip = ha.GradientClip(sizes, dtypes)
    host, _ = inputs(sizes, dtypes, 0.3, seed=6)
    want = clipped(clip, host, 0.5)
    t = [torch.from_numpy(h.copy()).cuda() for h in host]
    out, norm = [torch.zeros_like(a) for a in t], torch.zeros(1, device="cuda")
    s = ha.Stream()
    stream = torch.cuda.ExternalStream(ha._ffi.lib.he_stream_raw(s.handle))
    call = lambda: clip.clip([a.data_ptr() for a in t], [a.data_ptr() for a in out], 0.5, norm.data_ptr(), stream=s)  # noqa: E731
    torch.cuda.synchronize()
    call()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for _ in range(4):
        for a in out + [norm]:
            a.fill_(7.0)
        clipped(clip, host, 0.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert norm.item() == want[1] and all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(out, want[0]))


def test_a_training_step_of_a_normalised_layer(gpu):
    """y = norm(x + residual) W, its gradients, clipped together, and the optimizer's step: each operator reads what the one before left."""
    rows, columns, wide = 40, 96, 64
    rng = np.random.default_rng(7)
    x, residual, dy, dh = (rng.standard_normal((rows, columns)).astype(np.float32) for _ in range(4))
    gamma, weight, momentum = (1 + 0.2 * rng.standard_normal(columns)).astype(np.float32), *(rng.standard_normal((2, wide, columns)).astype(np.float32) / 10)
    d = {k: Array(v) for k, v in dict(x=x, residual=residual, dy=dy, dh=dh, gamma=gamma, weight=weight, momentum=momentum).items()}
    y, h, rstd, dgamma, norm = empty((rows, columns), np.float32), empty((rows, columns), np.float32), empty((rows,), np.float32), empty((columns,), np.float32), empty((1,), np.float32)
    op = ha.RmsNorm(columns, "f32", residual_dtype="f32", epsilon=EPSILON)
    op.forward(rows, d["x"].at, d["gamma"].at, y.at, residual=d["residual"].at, new_residual=h.at, rstd=rstd.at)
    flow = rng.standard_normal((rows, wide)).astype(np.float32)
    dweight = Array((flow.T @ y.back()).astype(np.float32))   # (the product's own gradients are the graphs')
    op.backward(rows, d["dy"].at, h.at, d["gamma"].at, rstd.at, None, dgamma.at, dh=d["dh"].at, dresidual=d["dh"].at)
    gradients = [dweight.back(), dgamma.back()]
    ha.GradientClip([wide * columns, columns], "f32").clip([dweight.at, dgamma.at], [dweight.at, dgamma.at], 1.0, norm.at)
    ha.Muon([(wide, columns)], "f32").step([dweight.at], [d["momentum"].at], [d["weight"].at], [d["momentum"].at], [d["weight"].at], learning_rate=0.1, momentum=0.9)
    want_y, _ = oracle_norm.forward(h.back(), gamma, EPSILON)
    assert np.array_equal(h.back(), x + residual) and np.allclose(y.back(), want_y, atol=1e-5)
    want_dx, want_dgamma = oracle_norm.backward(dy, h.back(), gamma, rstd.back(), dh)
    assert np.allclose(d["dh"].back(), want_dx, atol=1e-4) and np.allclose(gradients[1], want_dgamma, atol=1e-4)
    check_norm(gradients, norm.back()[0])
    check(["f32", "f32"], gradients, 1.0, [dweight.back(), dgamma.back()])
    want, _ = oracle_muon.step(dweight.back(), momentum, weight, 0.1, 0.9, 0.0, True)
    assert np.allclose(d["weight"].back(), want, atol=1e-5)


def test_more_than_the_caches_keep_in_several_groups(gpu):
    """The first group's first chunks are read past the caches, its others and the second group's are not."""
    sizes = [830_000 + 7 * k for k in range(128)] + [900_001, 0, 33, 1_000_003, 5] + [50_009] * 60 + [70_001, 1]
    dtypes = ["bf16"] * 140 + ["f16"] * 53 + ["f32"] * 2
    clip = ha.GradientClip(sizes, dtypes)
    (chunks, passing), (_, none) = [(int(a), int(b)) for a, b in re.findall(r"chunks=(\d+) blocks=\d+ first_sum=\d+ passing=(\d+)", clip.description)]
    assert 0 < passing < chunks and none == 0
    host, values = inputs(sizes, dtypes, 0.01, seed=13)
    got, norm = clipped(clip, host, 0.5)
    check(dtypes, values, 0.5, got, norm)
    again, same = clipped(clip, host, 0.5, in_place=True)
    assert same == norm and all(np.array_equal(a, b) for a, b in zip(again, got))
