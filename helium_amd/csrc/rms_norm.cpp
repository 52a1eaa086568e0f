#include "rms_norm.h"

#include <algorithm>
#include <cmath>
#include <future>
#include <sstream>

namespace he {

namespace {

// ---- device text ---------------------------------------------------------------------------------------------------
// One text for all kernels; the definitions ahead of it hold the problem and the tiling:
//   C (columns), V, NV, L (lanes of a row), T (threads), BF16 / F16, STREAM_SAME (h has x's type, otherwise f32), PARAM_SAME, RESIDUAL,
//   TO_I8, NORM, PITCH, EPS, X_ALIGN, H_ALIGN, Y_ALIGN (what rows are aligned to, in bytes), STREAM_OUT
//
// A row of C values is cut into vectors of V; where V does not divide C the last of them begins at C - V and shares values with the one
// before it (both make the same results of those; sums leave them out once).
const char* kCommon = R"HIP(
typedef unsigned char u8;
typedef unsigned short u16;
typedef unsigned int u32;
typedef unsigned long long u64;
#if BF16
typedef __bf16 elem_t;
#elif F16
typedef _Float16 elem_t;
#else
typedef float elem_t;
#endif
#if STREAM_SAME
typedef elem_t stream_t;
#else
typedef float stream_t;
#endif
#if PARAM_SAME
typedef elem_t param_t;
#else
typedef float param_t;
#endif
#define ROWS (T / L)
#define WAVES (T / 64)
#define WAVES_OF_ROW (L > 64 ? L / 64 : 1)
#define RAGGED (C % V != 0)
#if V == 1
typedef elem_t elem_v;
typedef stream_t stream_v;
typedef u8 byte_v;
#define AT(v, i) (v)
#else
typedef elem_t elem_v __attribute__((ext_vector_type(V), aligned(X_ALIGN)));
typedef stream_t stream_v __attribute__((ext_vector_type(V), aligned(H_ALIGN)));
typedef u8 byte_v __attribute__((ext_vector_type(V), aligned(RAGGED ? 1 : V)));
#define AT(v, i) (v)[i]
#endif

struct Lane {
    u32 l;       // of the row
    u32 slot;    // the row of the workgroup
};
__device__ __forceinline__ Lane lane() { return {threadIdx.x % L, threadIdx.x / L}; }
#define HAS(p, k) ((C + V - 1) / V % L == 0 && (k) < (C + V - 1) / V / L ? true : (p).l + (k) * L < (C + V - 1) / V)
__device__ __forceinline__ u32 start(const Lane& p, int k) {
    const u32 s = (p.l + k * L) * V;
    return RAGGED && s + V > C ? C - V : s;
}
// Whether the i-th value of a vector is this vector's to count.
__device__ __forceinline__ bool counts(const Lane& p, int k, int i) { return !RAGGED || start(p, k) + i >= (p.l + k * L) * V; }

__device__ __forceinline__ float of_bits(u32 b) { return __builtin_bit_cast(float, b); }
__device__ __forceinline__ u32 bits_of(float f) { return __builtin_bit_cast(u32, f); }

// The sum and the largest magnitude (as bits: of a NaN they are larger than of anything else) over the lanes of a row, the same in every
// lane. `red`: of LDS, not used again before the next barrier but one.
template <bool SUM, bool MOST> __device__ __forceinline__ void over_row(float& sum, u32& most, float (*red)[2]) {
#pragma unroll
    for (int m = (L < 64 ? L : 64) / 2; m > 0; m /= 2) {
        if (SUM) sum += __shfl_xor(sum, m, 64);
        if (MOST) {
            const u32 other = bits_of(__shfl_xor(of_bits(most), m, 64));
            most = other > most ? other : most;
        }
    }
#if L > 64
    if ((threadIdx.x & 63u) == 0) {
        if (SUM) red[threadIdx.x >> 6][0] = sum;
        if (MOST) red[threadIdx.x >> 6][1] = of_bits(most);
    }
    __syncthreads();
    const u32 first = (threadIdx.x / L) * WAVES_OF_ROW;
    sum = 0.0f;
    most = 0;
#pragma unroll
    for (u32 w = 0; w < WAVES_OF_ROW; w++) {
        if (SUM) sum += red[first + w][0];
        if (MOST) most = bits_of(red[first + w][1]) > most ? bits_of(red[first + w][1]) : most;
    }
#endif
}
#if STREAM_OUT
#define STORE(p, v) __builtin_nontemporal_store(v, p)
#else
#define STORE(p, v) (*(p) = (v))
#endif
)HIP";

// A row is read once and held in registers; its sum of squares (and the largest |h gamma|) are joined over its lanes, and the results
// are written. In 8 bits: with p = h gamma and P = max |p|, q = rint(127 p / P) needs no 1 / rms, which goes into the scale,
// rstd P / 127, alone.
//
// Rows that are only quantised: q = rint(127 x / A), exactly, ties to even (x = A / 2 is one). The f32 quotient is a whole number off at
// most next to a border, and there the remainder decides: 254 x - 2 q A has no rounding in f32 where x has 11 bits, in f64 where it has 24.
const char* kForward = R"HIP(
__device__ __forceinline__ u32 whole(float x, float most, float inverse) {
    float r = rintf(x * inverse);
#if !NORM
#if BF16 || F16
    const float off = __builtin_fmaf(-2.0f * r, most, 254.0f * x), half = most;
#else
    const double off = __builtin_fma(-2.0 * (double)r, (double)most, 254.0 * (double)x), half = most;
#endif
    const bool odd = (int)r & 1;
    if (off > half || (off == half && odd)) r += 1.0f;
    else if (off < -half || (off == -half && odd)) r -= 1.0f;
#endif
    return (u32)(int)r & 255u;
}
extern "C" __global__ __launch_bounds__(T) void rows_forward(u64 rows, const elem_t* x, const param_t* __restrict__ gamma, const stream_t* residual,
                                                             stream_t* new_residual, void* y, float* __restrict__ rstd_out, float* __restrict__ scales) {
    __shared__ float red[WAVES][2];
    const Lane p = lane();
    const u64 row = (u64)blockIdx.x * ROWS + p.slot;
    const bool there = row < rows;
    float h[NV][V], sum = 0.0f;
    u32 most = 0;
    elem_v hx[NV];
#if RESIDUAL
    stream_v hr[NV];
#endif
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (there && HAS(p, k)) {
            hx[k] = *(const elem_v*)(x + row * C + start(p, k));
#if RESIDUAL
            hr[k] = *(const stream_v*)(residual + row * C + start(p, k));
#endif
        }
#pragma unroll
    for (int k = 0; k < NV; k++) {
#pragma unroll
        for (int i = 0; i < V; i++) h[k][i] = 0.0f;
        if (there && HAS(p, k)) {
#pragma unroll
            for (int i = 0; i < V; i++) h[k][i] = (float)AT(hx[k], i);
#if RESIDUAL
            // (rounded to the stream's type: what is normalised is what its other readers see)
            stream_v out;
#pragma unroll
            for (int i = 0; i < V; i++) {
                AT(out, i) = (stream_t)(h[k][i] + (float)AT(hr[k], i));
                h[k][i] = (float)AT(out, i);
            }
            hr[k] = out;
#endif
#pragma unroll
            for (int i = 0; i < V; i++) {
                if (NORM && counts(p, k, i)) sum += h[k][i] * h[k][i];
#if TO_I8
                if (NORM) h[k][i] *= (float)gamma[start(p, k) + i];
                const u32 size = bits_of(h[k][i]) & 0x7fffffffu;
                most = size > most ? size : most;
#endif
            }
        }
    }
    over_row<NORM, TO_I8>(sum, most, red);
    float rstd = 1.0f;
#if NORM
    rstd = 1.0f / sqrtf(sum / (float)C + EPS);
    if (rstd_out && there && p.l == 0) rstd_out[row] = rstd;
#endif
#if TO_I8
    // A row that is not finite throughout has no scale: NaN, and zeros.
    const bool finite = most < 0x7f800000u && rstd < __builtin_inff();
    // (a power of two keeps 127 / size and 254 x in range)
    const float size = of_bits(most), up = size < 0x1p-64f ? 0x1p64f : size > 0x1p64f ? 0x1p-64f : 1.0f;
    const float inverse = finite && size > 0.0f ? 127.0f / (size * up) : 0.0f;
    if (there && p.l == 0) scales[row] = finite ? rstd * size / 127.0f : __builtin_nanf("");
#endif
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (there && HAS(p, k)) {
            const u32 c = start(p, k);
#if RESIDUAL
            STORE((stream_v*)(new_residual + row * C + c), hr[k]);
#endif
#if TO_I8
            byte_v out;
#pragma unroll
            for (int i = 0; i < V; i++) AT(out, i) = finite ? (u8)whole(h[k][i] * up, size * up, inverse) : (u8)0;
            *(byte_v*)((u8*)y + row * PITCH + c) = out;
#else
            elem_v out;
#pragma unroll
            for (int i = 0; i < V; i++) AT(out, i) = (elem_t)(h[k][i] * rstd * (float)gamma[c + i]);
            STORE((elem_v*)((elem_t*)y + row * C + c), out);
#endif
        }
#if TO_I8
    for (u32 c = C + p.l; c < PITCH; c += L)
        if (there) ((u8*)y)[row * PITCH + c] = 0;
#endif
}
)HIP";

// With xh = h rstd and flow = dy gamma: dh' = dh + rstd (flow - xh mean(flow xh)), dgamma = sum over the rows of dy xh. A workgroup goes through rows
// `gridDim.x` apart and keeps its share of dgamma in registers; `rows_fold` adds up the workgroups' shares. The order is fixed.
const char* kBackward = R"HIP(
extern "C" __global__ __launch_bounds__(T) void rows_backward(u64 rows, u32 blocks, const elem_t* dy, const stream_t* h, const param_t* __restrict__ gamma,
                                                              const float* __restrict__ rstd_of, const stream_t* dh, elem_t* dx, stream_t* dresidual,
                                                              float* __restrict__ parts) {
    __shared__ float red[2][WAVES][2];
    __shared__ float joined[ROWS > 1 ? C : 1];
    const Lane p = lane();
    float share[NV][V];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < V; i++) share[k][i] = 0.0f;
    u32 turn = 0;
    for (u64 first = (u64)blockIdx.x * ROWS; first < rows; first += (u64)blocks * ROWS, turn ^= 1) {
        const u64 row = first + p.slot;
        const bool there = row < rows;
        const float rstd = there ? rstd_of[row] : 0.0f;
        elem_v hd[NV];
        stream_v hh[NV], hr[NV];
#pragma unroll
        for (int k = 0; k < NV; k++)
            if (there && HAS(p, k)) {
                const u64 at = row * C + start(p, k);
                hd[k] = *(const elem_v*)(dy + at);
                hh[k] = *(const stream_v*)(h + at);
                if (dh) hr[k] = *(const stream_v*)(dh + at);
            }
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; k++)
            if (there && HAS(p, k))
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (counts(p, k, i)) {
                        const float t = (float)AT(hd[k], i) * ((float)AT(hh[k], i) * rstd);
                        sum += t * (float)gamma[start(p, k) + i];
                        share[k][i] += t;
                    }
        u32 none = 0;
        over_row<true, false>(sum, none, red[turn]);
        const float mean = sum / (float)C;
#pragma unroll
        for (int k = 0; k < NV; k++)
            if (there && HAS(p, k)) {
                const u64 at = row * C + start(p, k);
                elem_v out;
                stream_v more;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float xh = (float)AT(hh[k], i) * rstd;
                    float d = ((float)AT(hd[k], i) * (float)gamma[start(p, k) + i] - xh * mean) * rstd;
                    if (dh) d += (float)AT(hr[k], i);
                    AT(out, i) = (elem_t)d;
                    AT(more, i) = (stream_t)d;
                }
                if (dx) STORE((elem_v*)(dx + at), out);
                if (dresidual) STORE((stream_v*)(dresidual + at), more);
            }
    }
    // rows side by side: first those of a wave, then the waves' one after the other
#if L < 64
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < V; i++)
            for (int m = L; m < 64; m *= 2) share[k][i] += __shfl_xor(share[k][i], m, 64);
#endif
    const u32 group = threadIdx.x / (L < 64 ? 64 : L), groups = T / (L < 64 ? 64 : L);
    const bool mine = L >= 64 || (threadIdx.x & 63u) < L;
    float* to = parts + (u64)blockIdx.x * C;
    for (u32 g = 0; g < groups; g++) {
        if (g == group && mine)
#pragma unroll
            for (int k = 0; k < NV; k++)
                if (HAS(p, k))
#pragma unroll
                    for (int i = 0; i < V; i++)
                        if (counts(p, k, i)) {
                            const u32 c = start(p, k) + i;
                            const float s = (g ? joined[c] : 0.0f) + share[k][i];
                            if (g + 1 == groups) to[c] = s;
                            else joined[c] = s;
                        }
        if (groups > 1) __syncthreads();
    }
}

// dgamma[c] = the sum of `count` shares: 64 columns to a workgroup, the shares dealt to its 16 waves.
extern "C" __global__ __launch_bounds__(1024) void rows_fold(const float* __restrict__ parts, u32 count, float* __restrict__ dgamma) {
    __shared__ float part[16][64];
    const u32 column = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + column;
    float s = 0.0f;
    if (c < C)
#pragma unroll 8
        for (u32 n = wave; n < count; n += 16) s += parts[(u64)n * C + c];
    part[wave][column] = s;
    __syncthreads();
    if (wave == 0 && c < C) {
        for (u32 w = 1; w < 16; w++) s += part[w][column];
        dgamma[c] = s;
    }
}
)HIP";

constexpr uint64_t kThreads = 1ull << 32;  // a launch has fewer
constexpr int64_t kMostColumns = 32768;

int pow2_ceil(int64_t x) {
    int p = 1;
    while (p < x) p *= 2;
    return p;
}
// What a row of so many bytes is aligned to, if the first one is.
int row_alignment(int64_t bytes) { return (int)std::min<int64_t>(16, bytes & -bytes); }
int value_bytes(int dtype) { return (int)dtype_bits(dtype) / 8; }

std::string definitions(const RowProblem& pr, const RowTiling& t, bool stream_out) {
    std::ostringstream s;
    s << "#define C " << pr.columns << "\n#define V " << t.vec << "\n#define NV " << t.vectors << "\n#define L " << t.lanes << "\n#define T " << t.threads
      << "\n#define BF16 " << (pr.dtype == HE_BF16) << "\n#define F16 " << (pr.dtype == HE_F16) << "\n#define STREAM_SAME "
      << (pr.stream_dtype() == pr.dtype) << "\n#define PARAM_SAME " << (pr.param_dtype == pr.dtype) << "\n#define RESIDUAL " << pr.residual()
      << "\n#define TO_I8 " << pr.to_i8 << "\n#define NORM " << pr.norm << "\n#define PITCH " << quantized_pitch(pr.columns) << "ull\n#define EPS "
      << strfmt("%.9ef", (double)pr.epsilon) << "\n#define X_ALIGN " << row_alignment(pr.columns * value_bytes(pr.dtype)) << "\n#define H_ALIGN "
      << row_alignment(pr.columns * value_bytes(pr.stream_dtype())) << "\n#define STREAM_OUT " << stream_out << "\n";
    return s.str();
}

}  // namespace

std::string RowTiling::describe() const { return strfmt("vec=%d vectors=%d lanes=%d threads=%d", vec, vectors, lanes, threads); }

RowTiling plan_rows(const RowProblem& pr, int values) {
    RowTiling t;
    t.vec = 16 / value_bytes(pr.dtype);
    while (t.vec > pr.columns) t.vec /= 2;
    const int64_t vectors = (pr.columns + t.vec - 1) / t.vec;
    t.lanes = std::min(1024, pow2_ceil((vectors * t.vec + values - 1) / values));
    t.vectors = (int)((vectors + t.lanes - 1) / t.lanes);
    t.threads = std::max(256, t.lanes);
    return t;
}

RmsNorm::RmsNorm(const RowProblem& pr) : pr_(pr) {
    const char* what = pr.norm ? "rms norm" : "quantize rows";
    HE_REQUIRE(pr.columns >= 1, HE_ERR_INVALID, "%s: %lld columns", what, (long long)pr.columns);
    HE_REQUIRE(pr.columns <= kMostColumns, HE_ERR_UNSUPPORTED, "%s: %lld columns, at most %lld are taken", what, (long long)pr.columns, (long long)kMostColumns);
    HE_REQUIRE(pr.dtype == HE_F16 || pr.dtype == HE_BF16 || pr.dtype == HE_F32, HE_ERR_INVALID, "%s does not take dtype %s", what, dtype_name(pr.dtype));
    HE_REQUIRE(!pr.residual() || pr.residual_dtype == HE_F32 || pr.residual_dtype == pr.dtype, HE_ERR_INVALID,
               "rms norm: the residual is f32 or of the operand's type, not %s", dtype_name(pr.residual_dtype));
    HE_REQUIRE(pr.param_dtype == HE_F32 || pr.param_dtype == pr.dtype, HE_ERR_INVALID, "rms norm: gamma is f32 or of the operand's type, not %s",
               dtype_name(pr.param_dtype));
    HE_REQUIRE(std::isfinite(pr.epsilon) && pr.epsilon >= 0, HE_ERR_INVALID, "rms norm: epsilon %g", (double)pr.epsilon);
    few_ = plan_rows(pr, 8);
    many_ = plan_rows(pr, tuning::get_int("HELIUM_HIP_ROWS_VALUES", 16));
    back_ = plan_rows(pr, tuning::get_int("HELIUM_HIP_ROWS_BACK_VALUES", 16));
    const std::string few = definitions(pr, few_, false) + kCommon + kForward;
    const std::string many = definitions(pr, many_, true) + kCommon + kForward;
    const std::string back = definitions(pr, back_, true) + kCommon + kBackward;
    const bool has_back = pr.norm && !pr.to_i8;
    auto compiled = std::async(std::launch::async, [&] { (void)rtc_compile(many, "rows_forward", {}); });
    auto back_compiled = std::async(std::launch::async, [&] { if (has_back) (void)rtc_compile(back, "rows_backward", {}); });
    few_kernel_ = std::make_unique<JitKernel>(few, "rows_forward");
    compiled.get();
    many_kernel_ = std::make_unique<JitKernel>(many, "rows_forward");
    back_compiled.get();
    source_ = few + "\n" + many;
    describe_ = std::string(pr.norm ? "rms_norm" : "quantize_rows") + " few rows: " + few_.describe() + "\nmany rows: " + many_.describe();
    if (has_back) {
        back_kernel_ = std::make_unique<JitKernel>(back, "rows_backward");
        fold_kernel_ = std::make_unique<JitKernel>(back, "rows_fold");
        source_ += "\n" + back;
        describe_ += "\nbackward: " + back_.describe();
    }
}

RmsNorm::~RmsNorm() { scratch_.release(); }

namespace {
constexpr int kCUs = 256;
void check_tensor(const char* what, const void* p, int64_t alignment) {
    HE_REQUIRE(p && ((uintptr_t)p & (alignment - 1)) == 0, HE_ERR_INVALID, "%s is null or not aligned to %lld bytes", what, (long long)alignment);
}
}  // namespace

const RowTiling& RmsNorm::forward_tiling(int64_t rows) const { return rows <= 4 * kCUs ? few_ : many_; }

void RmsNorm::forward(int64_t rows, const void* x, const void* gamma, const void* residual, void* new_residual, void* y, float* rstd, float* scales,
                      hipStream_t stream) {
    HE_REQUIRE(rows >= 0, HE_ERR_INVALID, "%lld rows", (long long)rows);
    const int64_t align = row_alignment(pr_.columns * value_bytes(pr_.dtype)), stream_align = row_alignment(pr_.columns * value_bytes(pr_.stream_dtype()));
    HE_REQUIRE(pr_.residual() || (!residual && !new_residual), HE_ERR_INVALID, "rms norm: made without a residual");
    if (rows == 0) return;
    check_tensor("x", x, align);
    if (pr_.norm) check_tensor("gamma", gamma, value_bytes(pr_.param_dtype));
    if (pr_.residual()) {
        check_tensor("the residual", residual, stream_align);
        check_tensor("the new residual", new_residual, stream_align);
    }
    check_tensor("y", y, pr_.to_i8 ? 16 : align);
    HE_REQUIRE(((uintptr_t)rstd & 3) == 0, HE_ERR_INVALID, "rstd is not aligned to 4 bytes");
    if (pr_.to_i8) check_tensor("the list of scales", scales, 4);
    const RowTiling& t = forward_tiling(rows);
    const uint64_t blocks = ((uint64_t)rows + t.rows() - 1) / t.rows();
    HE_REQUIRE(blocks < kThreads / t.threads, HE_ERR_UNSUPPORTED, "%lld rows are too many for one launch", (long long)rows);
    uint64_t count = (uint64_t)rows;
    const uint32_t grid[3] = {(uint32_t)blocks, 1, 1}, block[3] = {(uint32_t)t.threads, 1, 1};
    void* args[] = {&count, &x, &gamma, &residual, &new_residual, &y, &rstd, &scales};
    (&t == &few_ ? few_kernel_ : many_kernel_)->launch(grid, block, 0, stream, args, true);
}

void RmsNorm::backward(int64_t rows, const void* dy, const void* h, const void* gamma, const float* rstd, const void* dh, void* dx, void* dresidual,
                       float* dgamma, hipStream_t stream) {
    HE_REQUIRE(back_kernel_, HE_ERR_UNSUPPORTED, "rms norm: an output in 8 bits has no gradient");
    HE_REQUIRE(rows >= 0, HE_ERR_INVALID, "%lld rows", (long long)rows);
    HE_REQUIRE(pr_.residual() || (!dh && !dresidual), HE_ERR_INVALID, "rms norm: made without a residual");
    check_tensor("dgamma", dgamma, 4);
    const int64_t align = row_alignment(pr_.columns * value_bytes(pr_.dtype)), stream_align = row_alignment(pr_.columns * value_bytes(pr_.stream_dtype()));
    if (rows) {
        check_tensor("dy", dy, align);
        check_tensor("h", h, stream_align);
        check_tensor("gamma", gamma, value_bytes(pr_.param_dtype));
        check_tensor("rstd", rstd, 4);
        HE_REQUIRE(dx || dresidual, HE_ERR_INVALID, "rms norm: dx and the residual's gradient are both null");
        if (dh) check_tensor("dh", dh, stream_align);
        if (dx) check_tensor("dx", dx, align);
        if (dresidual) check_tensor("the residual's gradient", dresidual, stream_align);
    }
    const uint64_t most = (uint64_t)kCUs * tuning::get_int("HELIUM_HIP_ROWS_BACK_PER_CU", 2);
    uint32_t blocks = (uint32_t)std::min<uint64_t>(most, ((uint64_t)rows + back_.rows() - 1) / back_.rows());
    uint64_t count = (uint64_t)rows;
    const uint32_t grid[3] = {blocks, 1, 1}, block[3] = {(uint32_t)back_.threads, 1, 1};
    const uint32_t fold_grid[3] = {(uint32_t)((pr_.columns + 63) / 64), 1, 1}, fold_block[3] = {1024, 1, 1};
    std::lock_guard<std::mutex> lk(mu_);
    // (one workgroup's share is the sum already)
    float* parts = blocks == 1 ? dgamma : scratch_.get(most * pr_.columns, 0, stream).floats;
    void* args[] = {&count, &blocks, &dy, &h, &gamma, &rstd, &dh, &dx, &dresidual, &parts};
    if (blocks) back_kernel_->launch(grid, block, 0, stream, args, blocks == 1);
    if (blocks == 1) return;
    void* fold_args[] = {&parts, &blocks, &dgamma};
    fold_kernel_->launch(fold_grid, fold_block, 0, stream, fold_args, true);
}

}  // namespace he

// ---- C ABI ------------------------------------------------------------------------------------------------
struct he_rms_norm_s {
    he::RmsNorm impl;
    explicit he_rms_norm_s(const he::RowProblem& pr) : impl(pr) {}
};
struct he_quantize_rows_s {
    he::RmsNorm impl;
    explicit he_quantize_rows_s(const he::RowProblem& pr) : impl(pr) {}
};

extern "C" {

int he_rms_norm_create(he_rms_norm_t* norm, int64_t columns, int dtype, int residual_dtype, int param_dtype, int to_i8, float epsilon) {
    return he::guard([&] {
        HE_REQUIRE(norm && residual_dtype >= -1, HE_ERR_INVALID, "bad argument");
        he::RowProblem pr;
        pr.columns = columns, pr.dtype = dtype, pr.residual_dtype = residual_dtype, pr.param_dtype = param_dtype, pr.to_i8 = to_i8 != 0, pr.epsilon = epsilon;
        *norm = new he_rms_norm_s(pr);
    });
}

int he_rms_norm_destroy(he_rms_norm_t norm) {
    return he::guard([&] { delete norm; });
}

int he_rms_norm_forward(he_rms_norm_t norm, int64_t rows, const void* x, const void* gamma, const void* residual, void* new_residual, void* y, float* rstd,
                        float* scales, he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(norm, HE_ERR_INVALID, "null rms norm");
        norm->impl.forward(rows, x, gamma, residual, new_residual, y, rstd, scales, stream ? stream->s : nullptr);
    });
}

int he_rms_norm_backward(he_rms_norm_t norm, int64_t rows, const void* dy, const void* h, const void* gamma, const float* rstd, const void* dh, void* dx,
                         void* dresidual, float* dgamma, he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(norm, HE_ERR_INVALID, "null rms norm");
        norm->impl.backward(rows, dy, h, gamma, rstd, dh, dx, dresidual, dgamma, stream ? stream->s : nullptr);
    });
}

const char* he_rms_norm_source(he_rms_norm_t norm) { return norm ? norm->impl.source().c_str() : ""; }
const char* he_rms_norm_describe(he_rms_norm_t norm) { return norm ? norm->impl.describe().c_str() : ""; }

int64_t he_quantized_pitch(int64_t columns) { return columns > 0 && columns <= INT64_MAX - 15 ? he::quantized_pitch(columns) : 0; }

int he_quantize_rows_create(he_quantize_rows_t* quantize, int64_t columns, int dtype) {
    return he::guard([&] {
        HE_REQUIRE(quantize, HE_ERR_INVALID, "bad argument");
        he::RowProblem pr;
        pr.columns = columns, pr.dtype = dtype, pr.to_i8 = true, pr.norm = false;
        *quantize = new he_quantize_rows_s(pr);
    });
}

int he_quantize_rows_destroy(he_quantize_rows_t quantize) {
    return he::guard([&] { delete quantize; });
}

int he_quantize_rows(he_quantize_rows_t quantize, int64_t rows, const void* x, void* q, float* scales, he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(quantize, HE_ERR_INVALID, "null quantize rows");
        quantize->impl.forward(rows, x, nullptr, nullptr, nullptr, q, nullptr, scales, stream ? stream->s : nullptr);
    });
}

const char* he_quantize_rows_source(he_quantize_rows_t quantize) { return quantize ? quantize->impl.source().c_str() : ""; }
const char* he_quantize_rows_describe(he_quantize_rows_t quantize) { return quantize ? quantize->impl.describe().c_str() : ""; }

}  // extern "C"
