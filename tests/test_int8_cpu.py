"""Products in 8-bit integers without a GPU: the generated kernels under the CPU emulation, how calls are cut, and what is refused."""
import ctypes
import re

import numpy as np
import pytest

import helium_amd as ha
from cpu_emul import run_kernel
from group_norm_cases import to_f32
from helium_amd import _ffi
from int8_cases import SMALL, check, inputs
from oracle import int8 as oracle

# the matrix instructions: lane l holds 16 neighbouring k of row l % 32 (or 16); c[i] is row (i / 4) * 8 + (l / 32) * 4 + i % 4 of
# column l % 32, or row (l / 16) * 4 + i of column l % 16
SHIM = r"""
typedef int emu_i32x4 __attribute__((ext_vector_type(4)));
typedef int emu_i32x16 __attribute__((ext_vector_type(16)));
static signed char g_i8a[1024][16], g_i8b[1024][16];
template <int SIDE, class C> static inline C emu_i8(emu_i32x4 a, emu_i32x4 b, C c) {
    unsigned tid = threadIdx.x, base = tid & ~63u, lane = tid & 63u;
    memcpy(g_i8a[tid], &a, 16);
    memcpy(g_i8b[tid], &b, 16);
    WAVE_BAR();
    for (int i = 0; i < SIDE * SIDE / 64; i++) {
        unsigned row = SIDE == 32 ? (i / 4) * 8 + (lane / 32) * 4 + i % 4 : (lane / 16) * 4 + i, col = lane % SIDE;
        for (int g = 0; g < 64 / SIDE; g++)
            for (int k = 0; k < 16; k++) c[i] += g_i8a[base + row + SIDE * g][k] * g_i8b[base + col + SIDE * g][k];
    }
    WAVE_BAR();
    return c;
}
#define MFMA_32(a, b, c) emu_i8<32>(a, b, c)
#define MFMA_16(a, b, c) emu_i8<16>(a, b, c)
"""

FIELDS = ("x", "x_scales", "weights", "weight_scales")


def emulated(op, host, dtype, shape, shares):
    """What the kernels of one of the shapes make of a call."""
    tokens, channels, columns = len(host["x"]), len(host["weights"]), host["x"].shape[1]
    said = dict(re.findall(r"(\w+)=(\w+)", op.describe(tokens)))
    assert int(said["shape"]) == shape and int(said["shares"]) == shares
    threads, grid, wide = int(said["threads"]), int(said["grid"]), -(-channels // 4) * 4
    texts = op.source.split("//// shape\n")[1:]
    bias = "bias" if host["bias"] is not None else "nullptr"
    wrapper = f"""
extern "C" void emu(const u8* x, const float* xs, const u8* w, const float* ws, const float* bias, out_t* y, int* parked) {{
    Call c{{x, w, xs, ws, {bias}, y, {tokens}, {channels}, {columns}, {grid}, {shares}, {wide}, parked}};
    ENTRY_OF(c);
}}
"""
    given = [(host[k], 0) for k in FIELDS] + [(host["bias"] if host["bias"] is not None else np.zeros(1, np.float32), 0)]
    y, parked = np.empty((tokens, channels), np.float32 if dtype == "f32" else np.uint16), np.zeros((shares if shares > 1 else 0, tokens, wide), np.int32)
    entry = "int8_stream" if "blocks_n" in said else "int8_product"
    y, parked = run_kernel(SHIM + texts[shape] + wrapper.replace("ENTRY_OF", entry), "emu", grid, threads, given + [(y, 1), (parked, 2)], grid_y=shares)
    if shares > 1:
        y, = run_kernel(SHIM + texts[-1] + wrapper.replace("ENTRY_OF", "int8_join"), "emu", -(-tokens * wide // 4 // 256), 256, given + [(y, 1), (parked, 0)])
    return y


SHAPES, TILES = 9, 4


# (size, shape): every shape at two or three sizes
PAIRS = [(k, shape) for shape in range(SHAPES) for k in range(len(SMALL)) if (shape + k) % 3 == 0]


@pytest.mark.parametrize("k,shape", PAIRS)
def test_the_kernels_match_the_oracle(monkeypatch, k, shape):
    tokens, columns, channels = SMALL[k]
    dtype = ("f32", "bf16", "f16")[k % 3]
    monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", str(shape + 1))
    monkeypatch.setenv("HELIUM_HIP_INT8_SHARES", "1")
    host = inputs(tokens, columns, channels, bias=k % 2, seed=k)
    y = emulated(ha.Int8Matmul(columns, channels, dtype), host, dtype, shape, 1)
    check(host, dtype, to_f32(y, dtype))


@pytest.mark.parametrize("shape,tokens,columns,channels,shares", [
    (0, 20, 1100, 300, 1), (1, 130, 400, 130, 1), (1, 9, 2100, 70, 4), (2, 140, 1300, 70, 1), (2, 30, 1300, 70, 2), (3, 70, 700, 130, 1), (3, 70, 2100, 70, 4),
    (4, 5, 9000, 18, 4), (7, 70, 8192, 17, 2), (6, 40, 5000, 33, 2), (8, 70, 2500, 66, 1),
])
def test_several_tiles_shares_and_rounds_of_the_ring(monkeypatch, shape, tokens, columns, channels, shares):
    monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", str(shape + 1))
    monkeypatch.setenv("HELIUM_HIP_INT8_SHARES", str(shares))
    host = inputs(tokens, columns, channels, bias=True, seed=9)
    y = emulated(ha.Int8Matmul(columns, channels, "f16"), host, "f16", shape, shares)
    check(host, "f16", to_f32(y, "f16"))


def test_the_oracles_product_is_exact():
    host = inputs(2, 40, 3, True, 1)
    want = [[sum(int(a) * int(b) for a, b in zip(x, w)) for w in host["weights"]] for x in host["x"]]
    want = np.array(want) * host["x_scales"].astype(np.float64)[:, None] * host["weight_scales"].astype(np.float64) + host["bias"]
    assert np.allclose(oracle.product(*[host[k] for k in FIELDS], host["bias"]), want, rtol=1e-14)


def test_every_call_is_cut():
    op = ha.Int8Matmul(16, 16, "f32")
    assert op.source.count("//// shape\n") == SHAPES + 1 and op.source.count("int8_product(Call") == TILES
    used = set()
    for columns in (1, 100, 1000, 4096, 16384, 131071):
        for channels in (1, 17, 300, 1024, 4096, 16384, 1 << 20):
            op = ha.Int8Matmul(columns, channels, "bf16")
            for tokens in (1, 15, 16, 17, 33, 48, 49, 64, 65, 100, 128, 200, 333, 512, 1000, 5000):
                said = dict(re.findall(r"(\w+)=([\w.]+)", op.describe(tokens)))
                used.add(int(said["shape"]))
                shares = int(said["shares"])
                assert int(said["grid"]) >= 1 and shares >= 1
                assert shares == 1 or (shares * tokens * (channels + 3) <= 1 << 23 and shares <= -(-columns // 512) and float(said["estimate"]) > 0)
    assert used == set(range(SHAPES))   # (nothing is built that no call takes)


def test_shapes_that_there_are_none_of_are_not_forced(monkeypatch):
    op = ha.Int8Matmul(700, 130, "f32")
    want = op.describe(70)
    for shape in ("-1", "-20", "0", "none"):
        monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", shape)
        assert op.describe(70) == want
    monkeypatch.setenv("HELIUM_HIP_INT8_SHAPE", "1000")
    assert f"shape={SHAPES - 1} " in op.describe(70)


@pytest.mark.parametrize("kwargs,says", [
    (dict(inputs=0), "0 inputs"),
    (dict(channels=-1), "-1 channels"),
    (dict(inputs=1 << 17), "131071 are taken"),
    (dict(channels=(1 << 24) + 1), "2.24 are taken"),
    (dict(dtype="u32"), "dtype u32"),
])
def test_what_cannot_be_multiplied_is_refused(kwargs, says):
    with pytest.raises(ha.HeliumError, match=says):
        ha.Int8Matmul(**{**dict(inputs=64, channels=64, dtype="f32"), **kwargs})


def test_operands_are_checked_before_any_launch():
    op, good = ha.Int8Matmul(64, 32, "bf16"), 4096
    fine = dict(tokens=2, x=good, x_scales=good, weights=good, weight_scales=good, y=good)
    for given, says in ((dict(x=None), "tokens are null"), (dict(x=good + 8), "tokens are null or not aligned to 16"), (dict(weights=good + 4), "weights are null or not aligned to 16"),
                        (dict(x_scales=None), "tokens' scales"), (dict(weight_scales=good + 2), "weights' scales"), (dict(y=good + 1), "result is null or not aligned to 2"),
                        (dict(bias=good + 2), "bias is not aligned"), (dict(tokens=-1), "-1 tokens"), (dict(tokens=1 << 25), "at most 2.24")):
        with pytest.raises(ha.HeliumError, match=says):
            op.multiply(**{**fine, **given})
    with pytest.raises(ha.HeliumError, match="too many for one launch"):
        ha.Int8Matmul(64, 1 << 24, "bf16").multiply(**dict(fine, tokens=1 << 24))
    op.multiply(0, None, None, None, None, None)
    h = ctypes.c_void_p()
    assert _ffi.lib.he_int8_matmul_create(None, 64, 64, _ffi.F32) == _ffi.ERR_INVALID
    assert _ffi.lib.he_int8_matmul(None, 1, *[None] * 7) == _ffi.ERR_INVALID
    assert _ffi.lib.he_int8_matmul_describe(h, 1, None, 0) == _ffi.ERR_INVALID
    with pytest.raises(ha.HeliumError):
        op.describe(0)
    assert _ffi.lib.he_int8_matmul_destroy(None) == _ffi.OK


def test_shared_sums_fit_their_scratch():
    """(2^22 sums of 32 bits: rows of channels in fours, of every share.)"""
    most = 0
    for columns in (512, 1000, 4096, 9000, 16384, 131071):
        for channels in (1, 3, 64, 130, 1001, 1024, 4097, 20000, 1 << 20):
            op = ha.Int8Matmul(columns, channels, "bf16")
            for tokens in (1, 2, 7, 16, 33, 64, 65, 100, 127, 200, 255, 333, 511, 777, 1024, 3000, 5000, 20000, 1 << 20):
                shares = int(re.search(r" shares=(\d+)", op.describe(tokens))[1])
                if shares > 1:
                    most = max(most, shares * tokens * -(-channels // 4) * 4)
    assert 1 << 20 < most <= 1 << 22
