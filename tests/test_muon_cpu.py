"""Orthogonalised updates without a GPU: the oracle's properties, the kernels under emulation (host AddressSanitizer checks every
access) against the oracle, and what the entry points refuse."""
import ctypes
import heapq
import time

import numpy as np
import pytest

import helium_amd as ha
from cpu_emul import run_kernel
from helium_amd import _ffi, backend
from muon_cases import SHAPES, check, check_rounded_once, matrix, runs_of, to_f32, to_storage
from oracle import muon as oracle

MATRIX = np.dtype([("rows", "u4"), ("cols", "u4"), ("mp", "u4"), ("np", "u4"), ("tall", "u4"), ("first_part", "u4"), ("parts", "u4"),
                   ("shape_scale", "f4"), ("at", "u8", 9)])
PRODUCT = np.dtype([(k, "u4") for k in ("mp", "np")] + [(k, "f4") for k in ("c1", "c2", "cs", "ci")]
                   + [(k, "u8") for k in ("p", "q", "e1", "e2", "out", "turned", "low", "parked_at")])
TASK = np.dtype([(k, "u4") for k in ("matrix", "i", "j", "k_begin", "k_end", "slot", "share", "shares")])
BLOCK = np.dtype([("matrix", "u4"), ("i", "u4"), ("j", "u4")])


def test_singular_values_go_where_the_polynomial_takes_them():
    rng = np.random.default_rng(1)
    for shape in ((20, 33), (33, 20), (12, 12)):
        u, s, vt = np.linalg.svd(rng.standard_normal(shape), full_matrices=False)
        got = oracle.orthogonalize((u * s) @ vt)
        want = (u * oracle.singular_values_after(s / (np.linalg.norm(s) + oracle.NORM_FLOOR))) @ vt
        assert np.abs(got - want).max() < 1e-10


def test_the_iteration_never_leaves_the_range_that_the_kernels_operands_are_scaled_for():
    s = np.linspace(0, 1, 200001)
    for _ in range(40):
        s = oracle.singular_values_after(s, 1)
        assert s.min() >= 0 and s.max() < 1.21
    a, b, c = oracle.COEFFICIENTS
    t = np.linspace(0, 1.21, 10001) ** 2
    assert np.abs(b * t + c * t * t).max() < 2.82 and 2.82 * 8192 < 65504 and 1.21 * 4096 < 65504 and 1.4642 * 8192 < 65504


def test_five_steps_bring_the_documented_range_near_one():
    s = oracle.singular_values_after(np.linspace(0.01, 1, 100001))
    assert s.min() > 0.65 and s.max() < 1.21


@pytest.mark.parametrize("kind", ["normal", "low_rank", "one_entry", "zero"])
@pytest.mark.parametrize("split,runs", [(True, None), (False, None), (True, [3, 2])])
def test_the_documented_arithmetic_is_within_the_tests_own_tolerance(kind, split, runs):
    for k, shape in enumerate(SHAPES):
        u = matrix(shape, kind, 1 + k).astype(np.float32)
        check(oracle.modelled(u, split, 5, runs), u, "f32", split, 5, runs)


def test_several_steps_at_once_cost_few_digits():
    """Singular values over three decades, where an error of X X^T weighs most: in 64 bits the two forms are one."""
    rng = np.random.default_rng(2)
    u, _, vt = np.linalg.svd(rng.standard_normal((96, 400)), full_matrices=False)
    u = (u * np.logspace(0, -3, 96)) @ vt
    want = oracle.orthogonalize(u)
    far = {str(r): np.linalg.norm(oracle.modelled(u, True, 5, r) - want) / np.linalg.norm(want) for r in (None, [3, 2])}
    assert far["None"] < 1e-5 and far["[3, 2]"] < 1e-5, far


def test_how_steps_are_taken_goes_by_shape_and_precision():
    runs = lambda *a, **k: runs_of(ha.Muon(*a, **k))  # noqa: E731
    assert runs([(512, 512)], "f32") == [1] * 5
    assert runs([(512, 4608)], "f32") == [3, 2] and runs([(4608, 512)], "f32", steps=4) == [2, 2] and runs([(512, 4608)], "f32", steps=7) == [3, 2, 2]
    assert runs([(512, 4608)], "bf16", precision="f16_f32") == [1] * 5


def test_a_caller_can_have_steps_one_by_one():
    try:
        backend.set_option(backend.OPT_MUON_SEVERAL_STEPS, 0)
        assert runs_of(ha.Muon([(512, 4608)], "f32")) == [1] * 5
    finally:
        backend.set_option(backend.OPT_MUON_SEVERAL_STEPS, 1)
    assert runs_of(ha.Muon([(512, 4608)], "f32")) == [3, 2]


SHFL = r"""
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
static inline int emu_frexp_exp(double x) { int e; (void)frexp(x, &e); return e; }
#define FREXP_EXP(x) emu_frexp_exp(x)
#define LDEXP_F64(x, n) ldexp(x, n)
#define LDEXP_F32(x, n) ldexpf(x, n)
"""


def emulated(shapes, dtype, split, steps, in_storage, step=None):
    """The launches of a call, one after the other. `step`: (momenta, weights, learning rate, mu, decay, nesterov)."""
    muon = ha.Muon(shapes, dtype, precision="f32_f32" if split else "f16_f32", steps=steps)
    mats, tasks, joins = np.frombuffer(muon.table(0), MATRIX), [np.frombuffer(muon.table(t), TASK) for t in (1, 2, 3)], [np.frombuffer(muon.table(t), TASK) for t in (4, 5, 6)]
    parts, blocks = (np.frombuffer(muon.table(t), BLOCK) for t in (7, 8))
    said = [dict(s.split("=") for s in line.split()[1:]) for line in muon.description.splitlines() if line.startswith("muon")]
    workspace = int(said[0]["workspace"])
    elements, *products = muon.source.split("\n//// product ")
    names = [f"in{k}" for k in range(len(shapes))]
    fill = "".join(f"o.in[{k}] = in{k}; " for k in range(len(shapes)))
    params = ", ".join(f"const elem_t* in{k}" for k in range(len(shapes)))
    if step:
        fill += "".join(f"o.momentum[{k}] = m{k}; o.new_momentum[{k}] = nm{k}; o.weight[{k}] = w{k}; " for k in range(len(shapes)))
        fill += "o.learning_rate = %.9gf; o.mu = %.9gf; o.weight_decay = %.9gf; o.nesterov = %d; " % step[2:]
        params += "".join(f", const float* m{k}, float* nm{k}, const float* w{k}" for k in range(len(shapes)))
    out_type = "float" if step else "elem_t"
    outs = ", ".join(f"{out_type}* out{k}" for k in range(len(shapes)))
    fill_out = "".join(f"o.out[{k}] = out{k}; " for k in range(len(shapes)))
    which = "true" if step else "false"
    wrappers = f"""
extern "C" void emu_norm(const Matrix* m, const Block* t, double* s, {params}) {{ Operands o{{}}; {fill} norm_part<{which}>(m, t, s, o); }}
extern "C" void emu_convert(const Matrix* m, const Block* t, const double* s, char* ws, {params}) {{ Operands o{{}}; {fill} convert_block<{which}>(m, t, s, ws, o); }}
extern "C" void emu_finish(const Matrix* m, const Block* t, const char* ws, {params}, {outs}) {{ Operands o{{}}; {fill} {fill_out} finish_block<{which}>(m, t, ws, o); }}
"""
    text = SHFL + elements + wrappers
    given = [(a, 0) for a in in_storage]
    sums = np.zeros(len(parts))
    if step:
        momenta, weights = step[0], step[1]
        for m, w in zip(momenta, weights):
            given += [(m, 0), (np.empty_like(m), 1), (w, 0)]
    got = run_kernel(text, "emu_norm", len(parts), 256, [(mats, 0), (parts, 0), (sums, 1)] + given)
    sums, new_momenta = got[0], got[1:]
    if step:  # from here on the new momenta are inputs
        given = [(a, 0) for a in in_storage] + [b for m, n, w in zip(momenta, new_momenta, weights) for b in ((m, 0), (n, 0), (w, 0))]
    ws, = run_kernel(text, "emu_convert", len(blocks), 256, [(mats, 0), (blocks, 0), (sums, 0), (np.empty(workspace, np.uint8), 1)] + given)
    kinds = {}
    for p, product in enumerate(products):
        name, body = product.split("\n", 1)
        kinds[name] = {key: int(v) for key, v in said[1 + p].items() if key != "estimate"}, tasks[p], joins[p], SHFL + body + f"""
extern "C" void emu_product(const Product* what, const u32* matrices, const Task* t, char* ws, float* parked) {{ product<{name.upper()}>(what, *matrices, t, ws, parked); }}
extern "C" void emu_join(const Product* what, const u32* matrices, const Task* t, char* ws, const float* parked) {{ join<{name.upper()}>(what, *matrices, t, ws, parked); }}
"""
    what, matrices = np.frombuffer(muon.table(9), PRODUCT).reshape(-1, len(shapes)), np.array([len(shapes)], np.uint32)
    lines = [line.split()[:2] for line in muon.description.split("\nlaunch ")[1:]]
    for k, (name, of) in enumerate(lines):
        if of != "of=0":
            continue
        count = 2 if k + 1 < len(lines) and lines[k + 1][1] == "of=1" else 1
        cut, tasks_of, joins_of, body = kinds[name]
        parked = np.full(max(cut["parked"], 1) * 2, np.nan, np.float32)
        ws, parked = run_kernel(body, "emu_product", cut["grid"], cut["threads"], [(what[k:k + count], 0), (matrices, 0), (tasks_of, 0), (ws, 2), (parked, 2)], grid_y=count)
        if cut["join_grid"]:
            ws, = run_kernel(body, "emu_join", cut["join_grid"], 256, [(what[k:k + count], 0), (matrices, 0), (joins_of, 0), (ws, 2), (parked, 0)], grid_y=count)
    outs = [np.empty(s, np.float32 if step else in_storage[0].dtype) for s in shapes]
    return run_kernel(text, "emu_finish", len(blocks), 256, [(mats, 0), (blocks, 0), (ws, 0)] + given + [(o, 1) for o in outs]), new_momenta


@pytest.mark.parametrize("dtype,split,steps,runs", [("f32", True, 1, "0"), ("f32", True, 3, "1"), ("f32", True, 5, "1"), ("f32", True, 2, "0"), ("bf16", False, 2, "0"), ("f16", False, 1, "0")])
def test_the_kernels_match_the_oracle(monkeypatch, dtype, split, steps, runs):
    monkeypatch.setenv("HELIUM_HIP_MUON_RUNS", runs)          # several steps at once, whatever they are estimated to take
    monkeypatch.setenv("HELIUM_HIP_MUON_ONE_BY_ONE", "1" if runs == "0" else "0")
    shapes = [(70, 90), (1, 1)] if steps > 2 else [(5, 9), (70, 33), (1, 1), (40, 150)]
    stored = [to_storage(matrix(s, "normal", 3), dtype) for s in shapes]
    got, _ = emulated(shapes, dtype, split, steps, stored)
    for g, s in zip(got, stored):
        check(to_f32(g, dtype), to_f32(s, dtype), dtype, split, steps, {"0": None, "1": {3: [3], 5: [3, 2]}.get(steps)}[runs])


def test_f16_results_have_the_digits_of_their_type(monkeypatch):
    """Also at f16_f32: five steps with operands of 11 bits would leave a result of 11 bits with eight of them."""
    monkeypatch.setenv("HELIUM_HIP_MUON_ONE_BY_ONE", "1")
    shapes = [(40, 70)]
    stored = [to_storage(matrix(s, "normal", 21), "f16") for s in shapes]
    got, _ = emulated(shapes, "f16", False, 5, stored)
    for g, s in zip(got, stored):
        check_rounded_once(to_f32(g, "f16"), to_f32(s, "f16"), "f16")


@pytest.mark.parametrize("nesterov", [0, 1])
def test_the_kernels_step_matches_the_oracles(nesterov):
    shapes = [(6, 10), (20, 3)]
    rng = np.random.default_rng(8)
    grads = [to_storage(rng.standard_normal(s), "bf16") for s in shapes]
    momenta, weights = ([rng.standard_normal(s).astype(np.float32) for s in shapes] for _ in range(2))
    new_weights, new_momenta = emulated(shapes, "bf16", True, 2, grads, (momenta, weights, 0.1, 0.9, 0.02, nesterov))
    for g, m, w, nw, nm in zip(grads, momenta, weights, new_weights, new_momenta):
        want_w, want_m = oracle.step(to_f32(g, "bf16"), m, w, np.float32(0.1), np.float32(0.9), np.float32(0.02), nesterov, 2)
        assert np.abs(nm - want_m).max() < 4 * 2.0 ** -24 * np.abs(want_m).max()
        # the orthogonalised part is good to some 1e-6 of values up to 1.2, times 0.1 sqrt(rows / columns)
        assert np.abs(nw - want_w).max() < 1e-5


@pytest.mark.parametrize("precision", ["f32_f32", "f16_f32"])
@pytest.mark.parametrize("shapes", [[(4096, 4096)] * 128 + [(4096, 11008)] * 96, [(32768, 262144)], [(8, 8)] * 65536, [(1 << 20, 32768)]])
def test_large_groups_are_cut_in_seconds(shapes, precision):
    """What the choice of tiles goes by is counted, not made: candidates of these groups have up to a thousand million tasks."""
    began = time.monotonic()
    muon = ha.Muon(shapes, "bf16", precision=precision)
    assert time.monotonic() - began < 20   # (most of a second or two is the compiler's; made and dealt, the first group took 50 seconds)
    for line in muon.description.splitlines()[1:4]:
        said = dict(s.split("=") for s in line.split()[1:])
        assert int(said["grid"]) * int(said["threads"]) < 1 << 32 and int(said["join_grid"]) * 256 < 1 << 32


@pytest.mark.parametrize("shapes,precision,steps,values", [
    ([(4096, 4096)], "f32_f32", 5, 5 * 4096 ** 2),                  # one step at a time: X, X^T twice, A and B
    ([(4096, 4096)], "f32_f32", 1, 4 * 4096 ** 2),
    ([(512, 4608)], "f32_f32", 5, 3 * 512 * 4608 + 5 * 512 ** 2),   # runs of three and two: C and two Q's too
    ([(4600, 500)], "f32_f32", 3, 2 * 512 * 4608 + 5 * 512 ** 2),   # one run of three
    ([(512, 4608)], "f16_f32", 5, 4 * 512 * 4608 + 2 * 512 ** 2),   # X's low part
])
def test_the_workspace_holds_what_the_launches_use(shapes, precision, steps, values):
    muon = ha.Muon(shapes, "bf16", precision=precision, steps=steps)
    lines = [dict(s.split("=") for s in line.split()[1:]) for line in muon.description.splitlines()[:4]]
    parked = max(int(line["parked"]) * (2 if p == 1 else 1) for p, line in enumerate(lines[1:]))
    matrices = values * (4 if precision == "f32_f32" else 2)
    assert 0 <= int(lines[0]["workspace"]) - matrices - 4 * parked - 8 * int(lines[0]["shares"]) < 16 * 256   # (each buffer begins at 256 bytes)


def test_groups_of_more_blocks_than_a_launch_has_are_refused_before_anything_is_made():
    began = time.monotonic()
    for shapes in ([(1 << 20, 32768)] * 2, [(4096, 4096)] * 65536):
        with pytest.raises(ha.HeliumError, match="too many elements"):
            ha.Muon(shapes, "f32")
    assert time.monotonic() - began < 10


def lengths_by_simulation(lengths, slots, base, each):
    """When the last of these tasks ends, each given to the place that is free first, the longest ones first."""
    free = [0.0] * slots
    for n in sorted(lengths, reverse=True):
        heapq.heappush(free, heapq.heappop(free) + base + each * n)
    return max(free)


@pytest.mark.parametrize("shapes", [[(64, 576)], [(1000, 512), (777, 1203)], [(4096, 1024), (1024, 4096)], [(700, 3000)] * 9, [(128, 128)] * 2000])
def test_a_cuts_estimate_is_that_of_its_own_tasks(monkeypatch, shapes):
    """The estimate comes from counts of tasks of each length; here the tasks that were made are dealt out one by one."""
    tiles = {64: (2, 2.5, 0.28, 0.50), 128: (2, 3.5, 0.85, 1.65), 192: (1, 5.0, 0.85, 2.00), 256: (1, 6.0, 2.00, 2.85)}
    for tile, (per_cu, base, alone, full) in tiles.items():
        monkeypatch.setenv("HELIUM_HIP_MUON_TILE", str(tile))
        muon = ha.Muon(shapes, "f32")
        for p, line in enumerate(muon.description.splitlines()[1:4]):
            said = dict(s.split("=") for s in line.split()[1:])
            tasks = np.frombuffer(muon.table(1 + p), TASK)
            assert len(tasks) == int(said["grid"])
            slots = 256 * per_cu
            f = min(1.0, len(tasks) / slots)
            want = lengths_by_simulation([int(t["k_end"]) - int(t["k_begin"]) for t in tasks], slots, base, alone + (full - alone) * f * f)
            if int(said["parked"]):
                want += 2.5 + 4.0 * int(said["parked"]) / 5e6
            assert abs(float(said["estimate"]) - want) < 0.051 + 1e-9 * want, (tile, line, want)   # (printed with one digit)


@pytest.mark.parametrize("shapes,dtype,precision,steps,says", [
    ([(4, 0)], "f32", "f32_f32", 5, "matrix 0 is 4 x 0"),
    ([(4, 4), (-1, 3)], "f32", "f32_f32", 5, "matrix 1 is -1 x 3"),
    ([(40000, 40000)], "f32", "f32_f32", 5, "extents up to"),
    ([(2 << 20, 4)], "f32", "f32_f32", 5, "extents up to"),
    ([(4, 4)], "u32", "f32_f32", 5, "dtype u32"),
    ([(4, 4)], "f32", "f32_f32", 0, "0 steps"),
    ([(4, 4)], "f32", "f32_f32", 33, "33 steps"),
    ([], "f32", "f32_f32", 5, "bad argument"),
])
def test_what_cannot_be_orthogonalised_is_refused(shapes, dtype, precision, steps, says):
    with pytest.raises(ha.HeliumError, match=says):
        ha.Muon(shapes, dtype, precision=precision, steps=steps)


def test_operands_are_checked_before_any_launch():
    muon = ha.Muon([(4, 4), (3, 5)], "f32")
    good = 4096  # (an address that nothing follows: every call below is refused)
    with pytest.raises(ha.HeliumError, match="takes 2 matrices, got 1"):
        muon.orthogonalize([good], [good])
    with pytest.raises(ValueError):
        muon.orthogonalize([good, good], [good])
    for bad in (None, good + 4):
        with pytest.raises(ha.HeliumError, match="matrix 1 is null or not 16-byte aligned"):
            muon.orthogonalize([good, bad], [good, good])
        with pytest.raises(ha.HeliumError, match="matrix 0 is null or not 16-byte aligned"):
            muon.step([good] * 2, [good] * 2, [good] * 2, [good] * 2, [bad, good], learning_rate=0.1)
    with pytest.raises(ha.HeliumError, match="not finite"):
        muon.step([good] * 2, [good] * 2, [good] * 2, [good] * 2, [good] * 2, learning_rate=float("nan"))
    with pytest.raises(ValueError):
        ha.Muon([(4, 4)], "f32", precision="bf16_f32")
    h, shape = ctypes.c_void_p(), (ctypes.c_int64 * 2)(4, 4)
    assert _ffi.lib.he_muon_create(ctypes.byref(h), shape, 1, _ffi.F32, 2, 5) == _ffi.ERR_INVALID   # bf16_f32
    assert _ffi.lib.he_muon_orthogonalize(None, None, None, 0, None) == _ffi.ERR_INVALID
    assert _ffi.lib.he_muon_destroy(None) == _ffi.OK
