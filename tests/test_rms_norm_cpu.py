"""Rms norm and quantised rows without a GPU: the oracle, the generated kernels under the CPU emulation, and what is refused."""
import ctypes
import re

import numpy as np
import pytest

import helium_amd as ha
from cpu_emul import run_kernel
from group_norm_cases import to_f32, to_storage
from helium_amd import _ffi
from helium_amd.int8 import pitch
from oracle import int8 as oracle_int8
from oracle import rms_norm as oracle
from rms_norm_cases import BEYOND, EPSILON, SHAPES, TYPES, beyond, check_backward, check_beyond, check_forward, check_quantized_beyond, check_quantized_norm, inputs


def test_the_oracles_gradients_are_those_of_its_forward_pass():
    rng = np.random.default_rng(1)
    h, dy = rng.standard_normal((2, 3, 7))
    gamma = 1 + 0.3 * rng.standard_normal(7)
    dh, dgamma = oracle.backward(dy, h, gamma, oracle.rstd(h, EPSILON))
    loss = lambda h, gamma: (oracle.forward(h, gamma, EPSILON)[0] * dy).sum()  # noqa: E731
    step = 1e-6
    for at in np.ndindex(3, 7):
        d = np.zeros((3, 7))
        d[at] = step
        assert abs((loss(h + d, gamma) - loss(h - d, gamma)) / (2 * step) - dh[at]) < 1e-7
    for c in range(7):
        d = np.zeros(7)
        d[c] = step
        assert abs((loss(h, gamma + d) - loss(h, gamma - d)) / (2 * step) - dgamma[c]) < 1e-7


def test_the_oracles_whole_numbers_are_the_nearest_ones():
    from fractions import Fraction

    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, 40)).astype(np.float32)
    x[1] = to_f32(to_storage(x[1], "bf16"), "bf16")
    x[2, :3] = [4.0, 2.0, -2.0]   # half of the largest: 63.5
    x[3, 0] = 127 * 0.25
    x[3, 1:5] = [0.125, -0.125, 0.375, 31.625]
    q, scales = oracle_int8.quantize(x)
    for r, row in enumerate(x):
        a = max(Fraction(float(abs(v))) for v in row)
        for c, v in enumerate(row):
            assert q[r, c] == round(127 * Fraction(float(v)) / a)   # (ties to even)


def parts(op):
    """How rows are cut, and the texts of forward (or quantisation) and backward."""
    return {k: int(n) for k, n in re.findall(r"(\w+)=(\d+)", op.description)}, ["#define C " + s for s in op.source.split("#define C ")[1:]]


def pointers(names, types, given):
    """Parameters and arguments of a wrapper; what is not given is null."""
    params = ", ".join(f"{types[n]} {n}" for n in names if n in given)
    return params, ", ".join(n if n in given else f"({types[n]})nullptr" for n in names)


FORWARD = ("x", "gamma", "residual", "new_residual", "y", "rstd", "scales")
FORWARD_TYPES = dict(zip(FORWARD, ("const elem_t*", "const param_t*", "const stream_t*", "stream_t*", "void*", "float*", "float*")))
BACKWARD = ("dy", "h", "gamma", "rstd", "dh", "dx", "dresidual", "parts")
BACKWARD_TYPES = dict(zip(BACKWARD, ("const elem_t*", "const stream_t*", "const param_t*", "const float*", "const stream_t*", "elem_t*", "stream_t*", "float*")))


def emulated_forward(tiling, text, rows, buffers):
    """buffers: by name (array, mode)"""
    params, args = pointers(FORWARD, FORWARD_TYPES, buffers)
    call = f"rows_forward_few(*rows, {args})" if "gamma" in buffers else "rows_quantize(*rows, x, (u8*)y, scales)"
    text += f"\nextern \"C\" void emu_forward(const u64* rows, {params}) {{ {call}; }}\n"
    given = [buffers[n] for n in FORWARD if n in buffers]
    side = tiling["threads"] // tiling["lanes"]
    got = run_kernel(text, "emu_forward", -(-rows // side), tiling["threads"], [(np.array([rows], np.uint64), 0)] + given)
    return dict(zip([n for n in FORWARD if n in buffers and buffers[n][1]], got))


def emulated_backward(tiling, text, rows, columns, blocks, buffers):
    buffers = dict(buffers, parts=(np.zeros((blocks, columns), np.float32), 1))
    params, args = pointers(BACKWARD, BACKWARD_TYPES, buffers)
    text += f"""
extern "C" void emu_backward(const u64* rows, const u32* blocks, {params}) {{ rows_backward{"_more" if "dh" in buffers else ""}(*rows, *blocks, {args}); }}
extern "C" void emu_fold(const float* parts, const u32* count, float* dgamma) {{ rows_fold(parts, *count, dgamma); }}
"""
    count = (np.array([blocks], np.uint32), 0)
    given = [buffers[n] for n in BACKWARD if n in buffers]
    got = run_kernel(text, "emu_backward", blocks, tiling["threads"], [(np.array([rows], np.uint64), 0), count] + given)
    got = dict(zip([n for n in BACKWARD if n in buffers and buffers[n][1]], got))
    got["dgamma"], = run_kernel(text, "emu_fold", (columns + 15) // 16, 1024, [(got["parts"], 0), count, (np.zeros(columns, np.float32), 1)])
    return got


CASES = [(shape, *TYPES[k % len(TYPES)], k % 2) for k, shape in enumerate(SHAPES)]


@pytest.mark.parametrize("shape,dtype,residual,same", CASES)
def test_the_kernels_match_the_oracle(shape, dtype, residual, same):
    rows, columns = shape
    param = dtype if same else "f32"
    host, v = inputs(rows, columns, dtype, residual, param, seed=columns)
    norm = ha.RmsNorm(columns, dtype, residual_dtype=residual, param_dtype=param, epsilon=EPSILON)
    tiling, (forward, back) = parts(norm)
    buffers = {"x": (host["x"], 0), "gamma": (host["gamma"], 0), "y": (np.empty_like(host["x"]), 1), "rstd": (np.empty(rows, np.float32), 1)}
    if residual:
        buffers.update(residual=(host["residual"], 0), new_residual=(np.empty_like(host["h"]), 1))
    got = emulated_forward(tiling, forward, rows, buffers)
    check_forward(dtype, v, to_f32(got["y"], dtype), got["rstd"])
    assert not residual or np.array_equal(got["new_residual"], host["h"])
    buffers = {k: (host[k], 0) for k in ("dy", "h", "gamma", "rstd")}
    buffers["dx"] = (np.empty_like(host["x"]), 1)
    if residual:
        buffers.update(dh=(host["dh"], 0), dresidual=(np.empty_like(host["h"]), 1))
    got = emulated_backward(tiling, back, rows, columns, 3, buffers)   # (of fewer rows, workgroups without any leave zeros)
    check_backward(dtype, residual, v, to_f32(got["dx"], dtype), to_f32(got["dresidual"], residual) if residual else None, got["dgamma"], rows)


@pytest.mark.parametrize("shape,dtype,residual,same", [c for c in CASES if c[0][1] < 2000][2::2])
def test_the_norm_into_8_bits_matches_the_oracle(shape, dtype, residual, same):
    rows, columns = shape
    host, v = inputs(rows, columns, dtype, residual, "f32", seed=columns + 1)
    tiling, (text,) = parts(ha.RmsNorm(columns, dtype, residual_dtype=residual, output="i8", epsilon=EPSILON))
    buffers = {"x": (host["x"], 0), "gamma": (host["gamma"], 0), "y": (np.empty((rows, pitch(columns)), np.int8), 1), "scales": (np.empty(rows, np.float32), 1)}
    if residual:
        buffers.update(residual=(host["residual"], 0), new_residual=(np.empty_like(host["h"]), 1))
    got = emulated_forward(tiling, text, rows, buffers)
    check_quantized_norm(v, got["y"], got["scales"])
    assert not residual or np.array_equal(got["new_residual"], host["h"])


def borders(rows, columns, dtype, seed):
    """Values on and next to the middle of two whole numbers, of ordinary, tiny and huge rows, rows of zeros and rows that are not finite."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, columns)).astype(np.float32)
    for r in range(rows):
        if r % 3 == 1:   # halves of whole steps, of rows whose largest value is 127 and 381 quarters
            most = 127 * (0.25 if r % 2 else 0.75)
            x[r] = np.rint(x[r] * 80).clip(-253, 253) * most / 254
            x[r, 0] = most
        if r % 3 == 2 and columns > 2:
            x[r, 1] = np.abs(x[r]).max() / 2
    if dtype != "f16":
        x *= np.array([1.0, 1e-38, 1e36, 1.0, 1e-30], np.float32)[np.arange(rows) % 5, None]
    if rows > 6:
        x[3], x[5, columns // 2], x[6, columns - 1] = 0, np.nan, np.inf
    return to_storage(x, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1, 1), (9, 3), (8, 64), (10, 130), (7, 517)])
def test_quantized_rows_are_the_oracles(shape, dtype):
    rows, columns = shape
    x = borders(rows, columns, dtype, columns)
    want, scales = oracle_int8.quantize(to_f32(x, dtype))
    tiling, (text,) = parts(ha.QuantizeRows(columns, dtype))
    got = emulated_forward(tiling, text, rows, {"x": (x, 0), "y": (np.empty((rows, pitch(columns)), np.int8), 1), "scales": (np.empty(rows, np.float32), 1)})
    assert np.array_equal(got["y"][:, :columns], want) and not got["y"][:, columns:].any()
    assert np.array_equal(got["scales"], scales, equal_nan=True)


@pytest.mark.parametrize("epsilon", [0.0, 1.0, 2.0 ** -149])
def test_every_accepted_epsilon_compiles(epsilon):
    ha.RmsNorm(16, "f32", epsilon=epsilon)


def test_the_pitch_is_whole_vectors():
    assert [pitch(n) for n in (1, 16, 17, 4096, 1203)] == [16, 16, 32, 4096, 1216] and pitch(0) == 0


@pytest.mark.parametrize("kwargs,says", [
    (dict(columns=0), "0 columns"),
    (dict(columns=32769), "at most 32768"),
    (dict(epsilon=-1.0), "epsilon"),
    (dict(epsilon=float("inf")), "epsilon"),
    (dict(dtype="u32"), "dtype u32"),
    (dict(dtype="bf16", residual_dtype="f16"), "residual is f32 or of the operand's type"),
    (dict(dtype="f16", param_dtype="bf16"), "gamma is f32 or of the operand's type"),
])
def test_what_cannot_be_normalised_is_refused(kwargs, says):
    with pytest.raises(ha.HeliumError, match=says):
        ha.RmsNorm(**{**dict(columns=64, dtype="f32"), **kwargs})


def test_quantizing_refuses_what_it_does_not_take():
    with pytest.raises(ha.HeliumError, match="at most 32768"):
        ha.QuantizeRows(40000, "bf16")
    with pytest.raises(ha.HeliumError, match="dtype bool"):
        ha.QuantizeRows(64, "bool")
    q, good = ha.QuantizeRows(64, "bf16"), 4096
    for args, says in (((None, good, good), "x is null"), ((good + 8, good, good), "x is null or not aligned to 16"), ((good, good + 8, good), "y is null or not aligned to 16"),
                       ((good, good, None), "scales is null")):
        with pytest.raises(ha.HeliumError, match=says):
            q.quantize(2, *args)
    with pytest.raises(ha.HeliumError, match="-1 rows"):
        q.quantize(-1, good, good, good)
    q.quantize(0, None, None, None)


def test_operands_are_checked_before_any_launch():
    """(Addresses that nothing follows: every call here is refused.)"""
    good = 4096
    norm = ha.RmsNorm(64, "bf16", residual_dtype="f32")
    for given, says in ((dict(x=None), "x is null"), (dict(y=good + 2), "y is null or not aligned to 16"), (dict(gamma=good + 2), "gamma is null or not aligned to 4"),
                        (dict(residual=None), "the residual is null"), (dict(new_residual=None), "the new residual is null"), (dict(rows=-2), "-2 rows"),
                        (dict(rstd=good + 1), "rstd is not aligned"), (dict(rows=1 << 40), "too many for one launch")):
        with pytest.raises(ha.HeliumError, match=says):
            norm.forward(**{**dict(rows=2, x=good, gamma=good, y=good, residual=good, new_residual=good), **given})
    for given, says in ((dict(dy=None), "dy is null"), (dict(h=good + 4), "h is null or not aligned to 16"), (dict(rstd=None), "rstd is null"),
                        (dict(dx=None, dresidual=None), "both null"), (dict(dgamma=None), "dgamma is null"), (dict(dh=good + 4), "dh is null"), (dict(rows=-2), "-2 rows")):
        with pytest.raises(ha.HeliumError, match=says):
            norm.backward(**{**dict(rows=2, dy=good, h=good, gamma=good, rstd=good, dx=good, dgamma=good), **given})
    plain = ha.RmsNorm(64, "bf16")
    with pytest.raises(ha.HeliumError, match="without a residual"):
        plain.forward(2, good, good, good, residual=good)
    with pytest.raises(ha.HeliumError, match="without a residual"):
        plain.backward(2, good, good, good, good, good, good, dh=good)
    eight = ha.RmsNorm(64, "bf16", output="i8")
    with pytest.raises(ha.HeliumError, match="no gradient"):
        eight.backward(2, good, good, good, good, good, good)
    with pytest.raises(ha.HeliumError, match="scales is null"):
        eight.forward(2, good, good, good)
    with pytest.raises(ValueError):
        ha.RmsNorm(64, "bf16", output="i4")
    plain.forward(0, None, None, None)
    h = ctypes.c_void_p()
    assert _ffi.lib.he_rms_norm_create(ctypes.byref(h), 64, _ffi.F32, -2, _ffi.F32, 0, 1e-5) == _ffi.ERR_INVALID
    assert _ffi.lib.he_rms_norm_create(None, 64, _ffi.F32, -1, _ffi.F32, 0, 1e-5) == _ffi.ERR_INVALID
    assert _ffi.lib.he_rms_norm_forward(None, 1, *[None] * 8) == _ffi.ERR_INVALID
    assert _ffi.lib.he_rms_norm_backward(None, 1, *[None] * 9) == _ffi.ERR_INVALID
    assert _ffi.lib.he_rms_norm_destroy(None) == _ffi.OK
    assert _ffi.lib.he_quantize_rows_create(None, 64, _ffi.F32) == _ffi.ERR_INVALID
    assert _ffi.lib.he_quantize_rows(None, 1, *[None] * 4) == _ffi.ERR_INVALID
    assert _ffi.lib.he_quantize_rows_destroy(None) == _ffi.OK


@pytest.mark.parametrize("rows,columns,dtype,residual,epsilon", BEYOND)
@pytest.mark.parametrize("output", ["same", "i8"])
def test_rows_whose_squares_are_beyond_f32(rows, columns, dtype, residual, epsilon, output):
    host, v = beyond(rows, columns, dtype, residual, epsilon, seed=columns)
    tiling, (text, *_) = parts(ha.RmsNorm(columns, dtype, residual_dtype=residual, output=output, epsilon=epsilon))
    buffers = {"x": (host["x"], 0), "gamma": (host["gamma"], 0), "rstd": (np.empty(rows, np.float32), 1)}
    buffers["y"] = (np.empty_like(host["x"]) if output == "same" else np.empty((rows, pitch(columns)), np.int8), 1)
    if output == "i8":
        buffers["scales"] = (np.empty(rows, np.float32), 1)
    if residual:
        buffers.update(residual=(host["residual"], 0), new_residual=(np.empty_like(host["h"]), 1))
    got = emulated_forward(tiling, text, rows, buffers)
    assert not residual or np.array_equal(got["new_residual"], host["h"])
    if output == "same":
        check_beyond(dtype, v, epsilon, to_f32(got["y"], dtype), got["rstd"])
    else:
        check_quantized_beyond(v, epsilon, got["y"], got["scales"])
