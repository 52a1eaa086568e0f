"""Gradient clipping without a GPU: the generated kernels under the CPU emulation, how tensors are cut, and what is refused."""
import ctypes
import re

import numpy as np
import pytest

import helium_amd as ha
from cpu_emul import run_kernel
from gradient_clip_cases import GROUPS, check, check_norm, inputs
from helium_amd import _ffi

SHIM = r"""
static double g_shfl64[1024];
static inline double emu_shfl64(double v, int mask) {
    unsigned tid = threadIdx.x;
    g_shfl64[tid] = v;
    WAVE_BAR();
    double r = g_shfl64[(tid & ~63u) | ((tid & 63u) ^ (unsigned)mask)];
    WAVE_BAR();
    return r;
}
#define SHFL_XOR_F64(v, m) emu_shfl64(v, m)
static int g_votes[1024];
static inline int emu_count(bool p) {
    unsigned tid = threadIdx.x;
    g_votes[tid] = p;
    WAVE_BAR();
    int n = 0;
    for (unsigned l = 0; l < 64; l++) n += g_votes[(tid & ~63u) + l];
    WAVE_BAR();
    return n;
}
#define COUNT_LANES(p) emu_count(p)
"""
TABLE = np.dtype([("first", np.uint32), ("dtype", np.uint32), ("bytes", np.uint64)])


def groups_of(clip):
    return [{k: int(v) for k, v in re.findall(r"(\w+)=(\d+)", line)} for line in clip.description.splitlines()[1:]]


def emulated(clip, host, most, in_place=False, passing=0):
    """out and norm of a call, by its launches one after the other."""
    table, groups = np.frombuffer(clip.table(), TABLE), groups_of(clip)
    sums = np.concatenate([run_group(clip, table, g, host, passing) for g in groups]) if groups else np.zeros(0)
    norm = np.zeros(1, np.float32)
    got = [None] * len(host)
    for g in reversed(groups):
        if not g["blocks"]:
            for k in range(g["count"]):
                got[g["first"] + k] = host[g["first"] + k]
            continue
        names = [f"i{k}" for k in range(g["count"])]
        params = "".join(f"const u8* {n}, " for n in names) + "".join(f"u8* o{k}, " for k in range(g["count"]))
        fill = "".join(f"o.in[{k}] = {'o' if in_place else 'i'}{k}; o.out[{k}] = o{k}; " for k in range(g["count"]))
        text = SHIM + clip.source + f"""
extern "C" void emu({params}const Tensor* t, const double* sums, float* norm) {{
    Both o{{}}; {fill} clip_scale(o, t, {g["count"]}, {g["chunks"]}, {passing}, sums, {len(sums)}, {most!r}f, norm);
}}
"""
        of = host[g["first"]:g["first"] + g["count"]]
        outs = [(h, 2) if in_place else (np.empty_like(h), 1) for h in of]
        *out, norm = run_kernel(text, "emu", g["blocks"], 256, [(h, 0) for h in of] + outs + [(table[g["first"]:g["first"] + g["count"]], 0), (sums, 0), (norm, 2)])
        got[g["first"]:g["first"] + g["count"]] = out
    return got, norm[0], sums


def run_group(clip, table, g, host, passing=0):
    if not g["blocks"]:
        return np.zeros(0)
    params = "".join(f"const u8* i{k}, " for k in range(g["count"]))
    fill = "".join(f"o.in[{k}] = i{k}; " for k in range(g["count"]))
    text = SHIM + clip.source + f"""
extern "C" void emu({params}const Tensor* t, double* sums) {{ Inputs o{{}}; {fill} clip_squares(o, t, {g["count"]}, {g["chunks"]}, {passing}, sums); }}
"""
    of = host[g["first"]:g["first"] + g["count"]]
    return run_kernel(text, "emu", g["blocks"], 256, [(h, 0) for h in of] + [(table[g["first"]:g["first"] + g["count"]], 0), (np.zeros(g["blocks"]), 1)])[0]


@pytest.mark.parametrize("k,most", [(k, most) for k in range(len(GROUPS)) for most in (0.5, 1e6) if len(GROUPS[k][0]) < 100 or most == 0.5])
def test_the_kernels_match_the_oracle(k, most):
    sizes, dtypes = GROUPS[k]
    host, values = inputs(sizes, dtypes, 0.3, seed=k)
    clip = ha.GradientClip(sizes, dtypes)
    got, norm, sums = emulated(clip, host, most, passing=k % 2)
    check(dtypes, values, most, got, norm)
    text = SHIM + clip.source + f"\nextern \"C\" void emu(const double* sums, float* norm) {{ clip_norm(sums, {len(sums)}, norm); }}\n"
    check_norm(values, run_kernel(text, "emu", 1, 256, [(sums, 0), (np.zeros(1, np.float32), 1)])[0][0])


@pytest.mark.parametrize("size,most", [(1e37, 1e-3), (1e37, 1e-6), (3e36, 1e-30), (1e30, 1e-3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_factors_that_f32_holds_with_few_bits_or_none(size, most, in_place):
    """(most / norm is below 2^-126, where f32 has fewer than 24 bits, in all but the last.)"""
    sizes, dtypes = [700, 300, 5000], ["f32", "bf16", "f32"]
    host, values = inputs(sizes, dtypes, size, seed=12)
    most = float(np.float32(most))   # (as the call has it)
    got, _, _ = emulated(ha.GradientClip(sizes, dtypes), host, most, in_place=in_place)
    check(dtypes, values, most, got)


def test_results_may_take_the_gradients_places():
    sizes, dtypes = GROUPS[1]
    host, values = inputs(sizes, dtypes, 0.3, seed=9)
    for most in (0.5, 1e6):
        got, _, _ = emulated(ha.GradientClip(sizes, dtypes), host, most, in_place=True)
        check(dtypes, values, most, got)


def test_a_workgroup_goes_through_several_chunks():
    """Fewer workgroups than chunks, as large models have: the tensors of 40 chunks by 7 workgroups."""
    sizes, dtypes = [70000, 0, 50001, 90000], ["f32", "f32", "bf16", "f16"]
    host, values = inputs(sizes, dtypes, 0.3, seed=10)
    clip = ha.GradientClip(sizes, dtypes)
    table = np.frombuffer(clip.table(), TABLE)
    g = dict(groups_of(clip)[0], blocks=7)
    sums = run_group(clip, table, g, host)
    assert abs(np.sqrt(sums.sum()) / np.sqrt(sum((v.astype(np.float64) ** 2).sum() for v in values)) - 1) < 1e-12


def test_workgroups_are_dealt_by_the_work():
    clip = ha.GradientClip([1 << 28] * 130 + [16], "bf16")
    groups = groups_of(clip)
    assert len(groups) == 2 and groups[0]["first_sum"] == 0 and groups[1]["first_sum"] == groups[0]["blocks"]
    assert sum(g["blocks"] for g in groups) <= 1025 and groups[0]["blocks"] > 60 * groups[1]["blocks"] > 0
    # (192 MB stay in the caches: 12288 chunks from the end)
    chunks = [128 << 15, (2 << 15) + 1]
    assert [g["passing"] for g in groups] == [chunks[0], chunks[1] - 12288]
    groups = groups_of(ha.GradientClip([1 << 20] * 128 + [1 << 20], "f32"))
    assert [g["passing"] for g in groups] == [129 * 256 - 12288, 0]
    assert groups_of(ha.GradientClip([3, 4], "f32"))[0]["blocks"] == 2
    table = np.frombuffer(clip.table(), TABLE)
    assert np.array_equal(table["first"][:3], [0, 1 << 15, 2 << 15]) and table["bytes"][130] == 32


def test_no_tensors_compile():
    ha.GradientClip([], "f32")
    ha.GradientClip([0, 0], "f32")


@pytest.mark.parametrize("sizes,dtypes,says", [
    ([-1], "f32", "-1 values"),
    ([4], "u32", "dtype u32"),
    ([1 << 40], "f32", "tensor 0 has"),
    ([1 << 39] * 64, "f32", "too large for one launch"),
    ([1] * 65537, "f32", "at most 65536"),
])
def test_what_cannot_be_clipped_is_refused(sizes, dtypes, says):
    with pytest.raises(ha.HeliumError, match=says):
        ha.GradientClip(sizes, dtypes)


def test_operands_are_checked_before_any_launch():
    clip, good = ha.GradientClip([4, 0, 8], ["f32", "f32", "bf16"]), 4096
    for gradients, out, says in (([good, None], [good, None, good], "lists|2 gradients"), ([good, None, None], [good, None, good], "gradients, tensor 2 is null"),
                                 ([good + 2, None, good], [good, None, good], "gradients, tensor 0"), ([good, None, good], [good, None, good + 1], "results, tensor 2")):
        with pytest.raises((ha.HeliumError, ValueError), match=says):
            clip.clip(gradients, out, 1.0)
    fine = [good, None, good]
    for most in (-1.0, float("nan")):
        with pytest.raises(ha.HeliumError, match="largest norm"):
            clip.clip(fine, fine, most)
    with pytest.raises(ha.HeliumError, match="norm is not aligned"):
        clip.clip(fine, fine, 1.0, good + 2)
    with pytest.raises(ha.HeliumError, match="norm is null"):
        clip.norm(fine, None)
    with pytest.raises(ha.HeliumError, match="takes 3 tensors, got 2"):
        clip.norm(fine[:2], good)
    with pytest.raises(ValueError):
        ha.GradientClip([1, 2], ["f32"])
    assert _ffi.lib.he_gradient_clip_create(None, None, None, 0) == _ffi.ERR_INVALID
    h = ctypes.c_void_p()
    assert _ffi.lib.he_gradient_clip_create(ctypes.byref(h), None, None, 2) == _ffi.ERR_INVALID
    assert _ffi.lib.he_gradient_norm(None, None, 0, None, None) == _ffi.ERR_INVALID
    assert _ffi.lib.he_gradient_clip(None, None, None, 0, 1.0, None, None) == _ffi.ERR_INVALID
    assert _ffi.lib.he_gradient_clip_table(None, None, 0, None) == _ffi.ERR_INVALID
    assert _ffi.lib.he_gradient_clip_destroy(None) == _ffi.OK
