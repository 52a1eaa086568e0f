"""Group norm without a GPU: the oracle against differences, the generated kernels under emulation (host AddressSanitizer
checks every access) against the oracle, and what the entry points refuse."""
import ctypes
import re

import numpy as np
import pytest

import helium_amd as ha
from cpu_emul import run_kernel
from group_norm_cases import EPSILON, SHAPES, WIDE, WIDEST, check_backward, check_forward, inputs, to_f32
from helium_amd import _ffi
from oracle import group_norm as oracle


@pytest.mark.parametrize("activation", ["none", "silu", "relu"])
def test_the_oracles_gradients_are_those_of_its_forward_pass(activation):
    rng = np.random.default_rng(5)
    n, p, c, groups = 2, 7, 12, 3
    x, dy = rng.standard_normal((2, n, p, c))
    gamma, beta = 1 + 0.3 * rng.standard_normal(c), 0.3 * rng.standard_normal(c)
    mean, rstd = oracle.statistics(x, groups, EPSILON)
    loss = lambda x, gamma, beta: (oracle.forward(x, gamma, beta, groups, activation, EPSILON)[0] * dy).sum()  # noqa: E731
    got = oracle.backward(dy, x, gamma, beta, mean, rstd, activation)
    h = 1e-6
    for k, (v, gradient) in enumerate(zip((x, gamma, beta), got)):
        for at in rng.choice(v.size, 12, replace=False):
            step = np.zeros(v.size)
            step[at] = h
            step = step.reshape(v.shape)
            up, down = [[x, gamma, beta] for _ in range(2)]
            up[k], down[k] = v + step, v - step
            # (the difference of two sums of 168 values near one, over 2 h: 1e-14 / 2e-6; curvature adds h^2)
            assert abs((loss(*up) - loss(*down)) / (2 * h) - gradient.reshape(-1)[at]) < 1e-6


def launch(norm, backward):
    """Grid, threads, parts of a sample and text of the forward or the backward pass."""
    line = norm.description.splitlines()[backward]
    return [int(re.search(k + r"=(\d+)", line).group(1)) for k in ("grid", "threads", "chunks")] + ["#define HE_EXP2(x) exp2f(x)\n#define BATCH" + norm.source.split("#define BATCH")[1 + backward]]


def forward_emulated(norm, shape, host):
    n, p, c, groups = shape
    grid, threads, chunks, text = launch(norm, False)
    y, stat = np.empty((n, p, c), host["x"].dtype), np.empty((n, groups), np.float32)
    if norm.description.startswith("group_norm forward: whole"):
        return run_kernel(text, "group_norm_forward", grid, threads, [(host[k], 0) for k in ("x", "gamma", "beta")] + [(y, 1), (stat, 1), (stat, 1)])
    parts, = run_kernel(text, "group_norm_stats", grid, threads, [(host["x"], 0), (np.empty((n, groups, chunks, 2), np.float32), 1)])
    mean, rstd = stat, stat
    if chunks > 32:
        parts, mean, rstd = run_kernel(text, "group_norm_merge", n * groups, int(re.search(r"#define MERGERS (\d+)", text).group(1)), [(parts, 0), (np.empty((n, groups, 2), np.float32), 1), (stat, 1), (stat, 1)])
    return run_kernel(text, "group_norm_apply", grid, threads, [(host["x"], 0), (host["gamma"], 0), (host["beta"], 0), (parts, 0), (y, 1), (mean, 2), (rstd, 2)])


def backward_emulated(norm, shape, host, mean, rstd):
    n, p, c, groups = shape
    grid, threads, chunks, text = launch(norm, True)
    given = [(host[k], 0) for k in ("dy", "x", "gamma", "beta")] + [(mean, 0), (rstd, 0)]
    dx, dparam, sums = np.empty((n, p, c), host["x"].dtype), np.empty(c, np.float32), np.empty((n, 2, c), np.float32)
    if norm.description.splitlines()[1].startswith("group_norm backward: whole"):
        samples, dx = run_kernel(text, "group_norm_backward", grid, threads, given + [(sums, 1), (dx, 1)])
        return [dx] + run_kernel(text, "group_norm_parameters", (c + 63) // 64, 256, [(samples, 0), (dparam, 1), (dparam, 1)])
    parts, = run_kernel(text, "group_norm_sums", grid, threads, given + [(np.empty((n * chunks, 2, c), np.float32), 1)])
    samples, = run_kernel(text, "group_norm_fold", n * ((2 * c + 31) // 32), 1024, [(parts, 0), (sums, 1)])
    return run_kernel(text, "group_norm_gradient", grid + (c + 63) // 64, threads, given + [(samples, 0), (dx, 1), (dparam, 1), (dparam, 1)])


CASES = [(shape, ("f32", "bf16", "f16")[k % 3], ("none", "relu", "silu")[(k // 2) % 3]) for k, shape in enumerate(SHAPES)]


@pytest.mark.parametrize("parts", ["0", "1"])
@pytest.mark.parametrize("shape,dtype,activation", CASES)
def test_the_kernels_match_the_oracle(monkeypatch, shape, dtype, activation, parts):
    monkeypatch.setenv("HELIUM_HIP_NORM_PARTS", parts)   # 1: through memory also where a workgroup could hold its groups
    param_dtype = dtype if shape[1] % 2 else "f32"
    norm = ha.GroupNorm(*shape, dtype, param_dtype=param_dtype, activation=activation, epsilon=EPSILON)
    host, v, mean, rstd = inputs(shape, dtype, param_dtype, activation, seed=shape[1])
    y, got_mean, got_rstd = forward_emulated(norm, shape, host)
    check_forward(shape, dtype, activation, v, to_f32(y, dtype), got_mean, got_rstd)
    dx, dgamma, dbeta = backward_emulated(norm, shape, host, mean, rstd)
    check_backward(shape, dtype, activation, v, mean, rstd, to_f32(dx, dtype), dgamma, dbeta)


@pytest.mark.parametrize("shape,dtype", WIDE)
def test_groups_of_more_channels_than_a_workgroup_has_threads(shape, dtype):
    """Up to the widest slice there is, also of single elements: sums of every channel, in the 160 KB of a workgroup's LDS."""
    norm = ha.GroupNorm(*shape, dtype, activation="silu", epsilon=EPSILON)
    host, v, mean, rstd = inputs(shape, dtype, "f32", "silu", seed=13)
    y, got_mean, got_rstd = forward_emulated(norm, shape, host)
    check_forward(shape, dtype, "silu", v, to_f32(y, dtype), got_mean, got_rstd)
    dx, dgamma, dbeta = backward_emulated(norm, shape, host, mean, rstd)
    check_backward(shape, dtype, "silu", v, mean, rstd, to_f32(dx, dtype), dgamma, dbeta)


@pytest.mark.parametrize("shape,dtype", WIDEST)
def test_a_thread_has_at_least_one_pixel(shape, dtype):
    norm = ha.GroupNorm(*shape, dtype, epsilon=EPSILON)
    assert all(int(n) >= 1 for n in re.findall(r"rows_per_thread=(\d+)", norm.description)), norm.description
    if shape[1] > 10:
        return  # (its 256 blocks take minutes under emulation)
    host, v, mean, rstd = inputs(shape, dtype, "f32", "none", seed=14)
    y, got_mean, got_rstd = forward_emulated(norm, shape, host)
    check_forward(shape, dtype, "none", v, to_f32(y, dtype), got_mean, got_rstd)


def test_forward_parts_hold_48_registers_or_all_64():
    """Three quarters of the rows where they divide, never a half."""
    rows = lambda *shape: int(re.search(r"rows_per_thread=(\d+)", ha.GroupNorm(*shape, "bf16").description).group(1))  # noqa: E731
    assert rows(2, 262144, 128, 32) == 12       # 16 vectors of 4 registers
    assert rows(64, 1000, 16384, 8) == 12       # one column of 2048 channels
    assert rows(64, 1000, 16384, 1) == 2        # eight columns: two rows, 64 registers


LEVEL = """
extern "C" void emu_level(const float* from, float* to, const u64* count) { group_norm_level(from, to, *count); }
"""


@pytest.mark.parametrize("batch,channels,levels", [(1024, 5, [1024]), (1025, 40, [1025, 5]), (300000, 3, [300000, 1172, 5])])
def test_sums_over_many_samples_are_no_long_chains(batch, channels, levels):
    """Every sum a tenth: added up one after the other in f32 each rounding leans to the same side, and 75000 of them lose four digits."""
    norm = ha.GroupNorm(batch, 1, channels, 1, "f32")
    text = launch(norm, True)[3]
    assert [int(n) for n in norm.description.split("samples=")[1].split(",")] == levels
    sums = np.full((batch, 2, channels), 0.1, np.float32) * np.array([[1], [-2]], np.float32)
    rows = [sums]
    for count in levels[1:]:
        rows += run_kernel(text + LEVEL, "emu_level", count * ((2 * channels + 63) // 64), 256,
                           [(rows[-1], 0), (np.empty((count, 2, channels), np.float32), 1), (np.array([len(rows[-1])], np.uint64), 0)])
    together = np.concatenate([r.reshape(-1) for r in rows])
    text += """
extern "C" void emu_parameters(const float* samples, float* dgamma, float* dbeta) { parameter_gradients<4>(blockIdx.x, samples, dgamma, dbeta); }
"""
    dgamma, dbeta = run_kernel(text, "emu_parameters", (channels + 63) // 64, 256, [(together, 0)] + [(np.empty(channels, np.float32), 1)] * 2)
    # chains of at most 256 + 64 + 64 additions and the few that join them, each off by 2^-24 of the sum
    for got, each in ((dbeta, np.float32(0.1)), (dgamma, np.float32(-0.2))):
        assert np.abs(got / (batch * np.float64(each)) - 1).max() < 400 * 2.0 ** -24, got


@pytest.mark.parametrize("parts", ["0", "1"])
@pytest.mark.parametrize("epsilon", [0.0, 1.0, 2.0 ** -149])
def test_every_accepted_epsilon_compiles(monkeypatch, epsilon, parts):
    """Whole numbers among them, and the smallest value there is."""
    monkeypatch.setenv("HELIUM_HIP_NORM_PARTS", parts)
    shape = (2, 37, 32, 4)
    norm = ha.GroupNorm(*shape, "f32", epsilon=epsilon)
    host, v, _, _ = inputs(shape, "f32", "f32", "none", seed=12)
    y, mean, rstd = forward_emulated(norm, shape, host)
    want, wmean, wrstd = oracle.forward(v["x"], v["gamma"], v["beta"], 4, "none", epsilon)
    # (sums of 296 values of about 2.5: 1024 roundings of 2^-24 each are more than their error, relative to |mean| + std and to the variance)
    assert np.abs(mean - wmean).max() < 1024 * 2.0 ** -24 * 10 and np.abs(rstd / wrstd - 1).max() < 2 * 1024 * 2.0 ** -24
    assert np.abs(y - want).max() < 4 * 1024 * 2.0 ** -24 * np.abs(want).max() * 10
    dx, dgamma, dbeta = backward_emulated(norm, shape, host, wmean.astype(np.float32), wrstd.astype(np.float32))
    assert np.isfinite(dx).all() and np.isfinite(dgamma).all() and np.isfinite(dbeta).all()


def launches(norm):
    """Workgroups and threads of every launch but the levels'."""
    forward, backward = ({k: int(v) for k, v in re.findall(r"#define (MERGE_BLOCKS|MERGERS|FOLD_BLOCKS|BLOCKS|T) (\d+)", "#define BATCH" + t)}
                         for t in norm.source.split("#define BATCH")[1:])
    return [(forward["BLOCKS"], forward["T"]), (backward["BLOCKS"] + (norm.channels + 63) // 64, backward["T"]),
            (forward["MERGE_BLOCKS"], forward["MERGERS"]), (backward["FOLD_BLOCKS"], 1024)]


@pytest.mark.parametrize("shape,dtype", [((1 << 20, 1, 64, 1), "bf16"), ((1 << 22, 1, 2, 1), "f32"), ((1 << 14, 6400, 256, 256), "f32"), ((1 << 10, 1 << 10, 16384, 1), "f32")])
def test_every_launch_has_fewer_threads_than_two_to_the_32(shape, dtype):
    """Where the small launches between the tensor's own would have 2^32 and more: a thread block of 1024 to 32 sums, or to a group."""
    norm = ha.GroupNorm(*shape, dtype)
    for blocks, threads in launches(norm):
        assert blocks * threads < 1 << 32, norm.description


def test_tensors_of_more_blocks_than_a_launch_has_are_refused_at_creation():
    assert launches(ha.GroupNorm((1 << 24) - 2, 1, 64, 1, "bf16"))[1] == ((1 << 24) - 1, 256)   # (with the workgroup of the parameters)
    for batch in ((1 << 24) - 1, 1 << 24):
        with pytest.raises(ha.HeliumError, match="too large for one launch"):
            ha.GroupNorm(batch, 1, 64, 1, "bf16")
    for extents in ((1 << 62, 1 << 2), (1 << 31, 1 << 40), (1, 1 << 62)):   # (whose products wrap)
        with pytest.raises(ha.HeliumError, match="extents too large"):
            ha.GroupNorm(*extents, 64, 1, "bf16")


def test_few_workgroups_merge_and_fold_as_many_do(monkeypatch):
    """The launches whose workgroups may have to take several groups or sums in turn, made to."""
    shape = (3, 9000, 40, 4)
    norm = ha.GroupNorm(*shape, "f32")
    host, v, mean, rstd = inputs(shape, "f32", "f32", "none", seed=16)
    n, p, c, groups = shape
    grid, threads, chunks, text = launch(norm, False)
    assert chunks > 32
    mergers = int(re.search(r"#define MERGERS (\d+)", text).group(1))
    parts, = run_kernel(text, "group_norm_stats", grid, threads, [(host["x"], 0), (np.empty((n, groups, chunks, 2), np.float32), 1)])
    stat = np.empty((n, groups), np.float32)
    merged = [run_kernel(re.sub(r"#define MERGE_BLOCKS \d+", f"#define MERGE_BLOCKS {blocks}", text), "group_norm_merge", blocks, mergers,
                         [(parts, 0), (np.empty((n, groups, 2), np.float32), 1), (stat, 1), (stat, 1)]) for blocks in (n * groups, 5)]
    assert all(np.array_equal(a, b) for a, b in zip(*merged)) and np.allclose(merged[0][1], mean, atol=1e-4)
    chunks, text = launch(norm, True)[2:]
    sums = np.random.default_rng(17).standard_normal((n, chunks, 2, c)).astype(np.float32)
    folded = [run_kernel(re.sub(r"#define FOLD_BLOCKS \d+", f"#define FOLD_BLOCKS {blocks}", text), "group_norm_fold", blocks, 1024,
                         [(sums, 0), (np.empty((n, 2, c), np.float32), 1)])[0] for blocks in (n * 3, 2)]
    # (chains of chunks / 32 and five more additions)
    assert np.array_equal(*folded) and (np.abs(folded[0] - sums.astype(np.float64).sum(axis=1)) <= (chunks / 32 + 6) * 2.0 ** -24 * np.abs(sums).sum(axis=1)).all()


def test_more_blocks_than_a_launch_has_are_refused():
    """2^32 workgroups of the second launch, though the tensor's own launch would have fewer than 2^31."""
    with pytest.raises(ha.HeliumError, match="too large for one launch"):
        ha.GroupNorm(1 << 30, 1, 64, 1, "bf16")


@pytest.mark.parametrize("kwargs,says", [
    (dict(channels=30, groups=4), "do not divide"),
    (dict(groups=0), "groups 0"),
    (dict(pixels=0), "pixels 0"),
    (dict(batch=-1), "batch -1"),
    (dict(epsilon=-1.0), "epsilon"),
    (dict(epsilon=float("nan")), "epsilon"),
    (dict(dtype="u32"), "dtype u32"),
    (dict(dtype="bf16", param_dtype="f16"), "parameters are f32 or of the tensor's type"),
    (dict(channels=32768, groups=1), "at most 16384"),
])
def test_what_cannot_be_normalised_is_refused(kwargs, says):
    given = dict(batch=2, pixels=9, channels=32, groups=4, dtype="f32", epsilon=1e-5)
    with pytest.raises(ha.HeliumError, match=says):
        ha.GroupNorm(**{**given, **kwargs})


def test_unknown_activations_and_null_handles_are_refused():
    with pytest.raises(ValueError):
        ha.GroupNorm(1, 1, 8, 1, "f32", activation="tanh")
    h = ctypes.c_void_p()
    assert _ffi.lib.he_group_norm_create(ctypes.byref(h), 1, 1, 8, 1, _ffi.F32, _ffi.F32, 7, 1e-5) == _ffi.ERR_INVALID
    assert _ffi.lib.he_group_norm_create(None, 1, 1, 8, 1, _ffi.F32, _ffi.F32, 0, 1e-5) == _ffi.ERR_INVALID
    assert _ffi.lib.he_group_norm_forward(None, *[None] * 7) == _ffi.ERR_INVALID
    assert _ffi.lib.he_group_norm_backward(None, *[None] * 10) == _ffi.ERR_INVALID
    assert _ffi.lib.he_group_norm_destroy(None) == _ffi.OK


def test_null_and_misaligned_operands_are_refused_before_any_launch():
    norm = ha.GroupNorm(1, 4, 16, 2, "bf16")
    good = 4096  # (an address that nothing follows: every call below is refused)
    for bad in (None, good + 8):
        with pytest.raises(ha.HeliumError, match="aligned"):
            norm.forward(bad, good, good, good)
        with pytest.raises(ha.HeliumError, match="aligned"):
            norm.backward(good, good, good, good, good, good, bad, good, good)
    with pytest.raises(ha.HeliumError, match="gamma or beta"):
        norm.forward(good, None, good, good)
    with pytest.raises(ha.HeliumError, match="needs the statistics"):
        norm.backward(good, good, good, good, None, good, good, good, good)
    with pytest.raises(ha.HeliumError, match="gradients are null"):
        norm.backward(good, good, good, good, good, good, good, None, good)


def test_an_empty_batch_needs_no_operands():
    ha.GroupNorm(0, 4, 16, 2, "bf16").forward(None, None, None, None)
