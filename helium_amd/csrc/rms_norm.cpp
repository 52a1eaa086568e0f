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
//   TO_I8, PITCH, EPS, X_ALIGN, H_ALIGN (what vectors are aligned to, in bytes)
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
// (a macro: a template's parameter would lose the vectors' alignment)
#define STORE(past, p, v) do { if (past) __builtin_nontemporal_store(v, p); else *(p) = (v); } while (0)
)HIP";

// 8 bits. Adding 1.5 * 2^23 to a value within +-2^22 rounds it to a whole number, which the sum's last bits are (1.5 * 2^52 in 64 bits).
// A row that is not finite throughout has no scale: NaN, and zeros.
const char* kBytes = R"HIP(
#define WHOLE_BITS(t) bits_of((t) + 12582912.0f)
struct Steps { float up, size; bool finite; };   // values times `up`, a power of two, have `size` for their largest: 127 / size and its remainder are in range
__device__ __forceinline__ Steps steps_of(u32 most) {
    const float size = of_bits(most), up = size < 0x1p-64f ? 0x1p64f : size > 0x1p64f ? 0x1p-64f : 1.0f;
    return {up, size * up, most < 0x7f800000u};
}
__device__ __forceinline__ void store_bytes(u8* row, u32 c, const u32 (&whole)[V], bool finite) {
    byte_v out;
#pragma unroll
    for (int i = 0; i < V; i++) AT(out, i) = (u8)(finite ? whole[i] : 0u);
    *(byte_v*)(row + c) = out;
}
__device__ __forceinline__ void store_padding(u8* row, const Lane& p) {
    for (u32 c = C + p.l; c < PITCH; c += L) row[c] = 0;
}
)HIP";

// A row is read once and held in registers; its sum of squares (and the largest |h gamma|) are joined over its lanes, and the results
// are written. In 8 bits: with p = h gamma and P = max |p|, q = rint(127 p / P) needs no 1 / rms, which goes into the scale,
// rstd P / 127, alone.
//
// Bound by memory: 8192 x 4096 bf16 with a residual 47.1 us (5.7 TB/s, the rate of a copy), into 8 bits 2048 x 4096 10.6 us (5.5 TB/s); f32 residuals beside
// 16-bit operands, 2000 x 16384, 71 us (5.5 TB/s; 90 with accesses of 16 bytes of the narrower type). One row of 4096: a launch, 2.5 us. Rows beyond 16384 with an f32 operand do not
// fit a thread's 128 registers and keep some 400 bytes of theirs in scratch memory: 1000 x 32768 f32 354 us, with a residual 441 (46 and 92 at the rate of a copy).
//
// A sum of squares that f32 cannot hold (from values of some 1e17 on in long rows, of 1.8e19 in any; without an epsilon to speak of, of values below 1e-15) is taken
// again of the values times a power of two; other rows' results are as they would be without it.
const char* kForward = R"HIP(
__device__ __forceinline__ bool beyond(float sum) { return !(sum < __builtin_inff()) || (EPS < 0x1p-80f && sum < 0x1p-90f); }
// PAST: results bypass the caches
template <bool PAST> __device__ __forceinline__ void forward(u64 rows, const elem_t* x, const param_t* __restrict__ gamma, const stream_t* residual,
                                                            stream_t* new_residual, void* y, float* __restrict__ rstd_out, float* __restrict__ scales) {
    __shared__ float red[2][WAVES][2];
    const Lane p = lane();
    const u64 row = (u64)blockIdx.x * ROWS + p.slot;
    const bool there = row < rows;
    float h[NV][V], weight[NV][V], sum = 0.0f;
    u32 most = 0;
    elem_v hx[NV];
#if RESIDUAL
    stream_v hr[NV];
#endif
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (there && HAS(p, k)) {
#pragma unroll
            for (int i = 0; i < V; i++) weight[k][i] = (float)gamma[start(p, k) + i];
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
                if (counts(p, k, i)) sum += h[k][i] * h[k][i];
#if TO_I8
                h[k][i] *= weight[k][i];
                const u32 size = bits_of(h[k][i]) & 0x7fffffffu;
                most = size > most ? size : most;
#endif
            }
        }
    }
    over_row<true, TO_I8>(sum, most, red[0]);
#if RESIDUAL
    // (not before all lanes have what they read: a ragged row's last two vectors overlap, and the new residual may lie in the old one's place)
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (there && HAS(p, k)) STORE(PAST, (stream_v*)(new_residual + row * C + start(p, k)), hr[k]);
#endif
    float rstd = 1.0f / sqrtf(sum / (float)C + EPS);
    // (the same answer in all threads that meet in over_row: those of a wave, or of a workgroup)
#if L > 64
    bool again = false;
#pragma unroll
    for (u32 r = 0; r < ROWS; r++) {
        float s = 0.0f;
#pragma unroll
        for (u32 w = 0; w < WAVES_OF_ROW; w++) s += red[0][r * WAVES_OF_ROW + w][0];
        again = again || beyond(s);
    }
#else
    const bool again = __any(there && beyond(sum));
#endif
    if (again) {
        const float by = sum < 1.0f ? 0x1p100f : 0x1p-80f;
        float squares = 0.0f;
        u32 none = 0;
#pragma unroll
        for (int k = 0; k < NV; k++)
            if (there && HAS(p, k))
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (counts(p, k, i)) {
#if RESIDUAL
                        const float v = (float)AT(hr[k], i) * by;
#else
                        const float v = (float)AT(hx[k], i) * by;
#endif
                        squares += v * v;
                    }
        over_row<true, false>(squares, none, red[1]);
        if (beyond(sum)) rstd = by / sqrtf(squares / (float)C + EPS * by * by);
    }
    if (rstd_out && there && p.l == 0) rstd_out[row] = rstd;
#if TO_I8
    const Steps s = steps_of(most);
    const bool finite = s.finite && rstd < __builtin_inff();
    const float inverse = s.size > 0.0f ? 127.0f / s.size : 0.0f;
    if (there && p.l == 0) scales[row] = finite ? rstd * of_bits(most) / 127.0f : __builtin_nanf("");
    if (s.up != 1.0f)
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < V; i++) h[k][i] *= s.up;
    u8* to = (u8*)y + row * PITCH;
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (there && HAS(p, k)) {
            u32 whole[V];
#pragma unroll
            for (int i = 0; i < V; i++) whole[i] = bits_of(__builtin_fmaf(h[k][i], inverse, 12582912.0f));
            store_bytes(to, start(p, k), whole, finite);
        }
    if (there) store_padding(to, p);
#else
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (there && HAS(p, k)) {
            const u32 c = start(p, k);
            elem_v out;
#pragma unroll
            for (int i = 0; i < V; i++) AT(out, i) = (elem_t)(h[k][i] * rstd * weight[k][i]);
            STORE(PAST, (elem_v*)((elem_t*)y + row * C + c), out);
        }
#endif
}
#define FORWARD(name, past) \
    extern "C" __global__ __launch_bounds__(T) void name(u64 rows, const elem_t* x, const param_t* gamma, const stream_t* residual, stream_t* new_residual, void* y, float* rstd, float* scales) { forward<past>(rows, x, gamma, residual, new_residual, y, rstd, scales); }
FORWARD(rows_forward, true)
FORWARD(rows_forward_few, false)   // results that stay in the caches for whoever reads them next
)HIP";

// q = rint(127 x / A), exactly, ties to even. 127 / A is taken in two parts, and x times both is added up with one rounding: a quotient in the
// middle of two whole numbers (x = A / 2 has one) is a value of the type, and so comes out as itself. Any other one is further from the middle
// than it is off: x = a 2^i and A = b 2^j with whole a and b give a distance of at least 1 / (2 a) of x / A, where the error is 2^-16 of that
// in f32 (a has 8 or 11 bits) and 2^-45 in f64 (24 bits).
//
// 4096 x 4096 bf16 10.9 us (4.6 TB/s), f32 14.9 (5.6 TB/s). Deciding by the remainder instead was bound by its arithmetic: 17.7 us.
const char* kQuantize = R"HIP(
#if BF16 || F16
typedef float wide_t;
#define ROUNDED(t) WHOLE_BITS(t)
#else
typedef double wide_t;
#define ROUNDED(t) (u32)__builtin_bit_cast(u64, (t) + 6755399441055744.0)
#endif
__device__ __forceinline__ float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }
#if (BF16 || F16) && V > 1
typedef u16 u16_v __attribute__((ext_vector_type(V)));
#endif
extern "C" __global__ __launch_bounds__(T) void rows_quantize(u64 rows, const elem_t* __restrict__ x, u8* __restrict__ y, float* __restrict__ scales) {
    __shared__ float red[WAVES][2];
    const Lane p = lane();
    const u64 row = (u64)blockIdx.x * ROWS + p.slot;
    const bool there = row < rows;
    elem_v hx[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        hx[k] = elem_v((elem_t)0.0f);
        if (there && HAS(p, k)) hx[k] = *(const elem_v*)(x + row * C + start(p, k));
    }
    u32 most = 0;
#if (BF16 || F16) && V > 1
    // (magnitudes in their own bits, two at a time)
    u16_v largest = u16_v((u16)0);
#pragma unroll
    for (int k = 0; k < NV; k++) largest = __builtin_elementwise_max(largest, __builtin_bit_cast(u16_v, hx[k]) & u16_v((u16)0x7fff));
#pragma unroll
    for (int i = 0; i < V; i++) most = largest[i] > most ? largest[i] : most;
    most = bits_of((float)__builtin_bit_cast(elem_t, (u16)most)) & 0x7fffffffu;
#else
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            const u32 size = bits_of((float)AT(hx[k], i)) & 0x7fffffffu;
            most = size > most ? size : most;
        }
#endif
    float none = 0.0f;
    over_row<false, true>(none, most, red);
    const Steps s = steps_of(most);
    const wide_t size = s.size, inverse = size > 0 ? (wide_t)127 / size : (wide_t)0, rest = size > 0 ? fused(-size, inverse, (wide_t)127) / size : (wide_t)0;
    if (there && p.l == 0) scales[row] = s.finite ? of_bits(most) / 127.0f : __builtin_nanf("");
    u8* to = y + row * PITCH;
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (there && HAS(p, k)) {
            u32 whole[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                const wide_t v = (float)AT(hx[k], i) * s.up;
                whole[i] = ROUNDED(fused(v, inverse, v * rest));
            }
            store_bytes(to, start(p, k), whole, s.finite);
        }
    if (there) store_padding(to, p);
}
)HIP";

// With xh = h rstd and flow = dy gamma: dh' = dh + rstd (flow - xh mean(flow xh)), dgamma = sum over the rows of dy xh. A workgroup goes through rows
// `blocks` apart and keeps its share of dgamma in registers; `rows_fold` adds up the workgroups' shares. The order is fixed.
//
// Bound by memory: 8192 x 4096 bf16 with the residual's gradient 50.8 us with the fold (5.3 TB/s); with the next row's loads under conditions, or with
// gamma's loads in between, 57 to 60: the counter of loads then runs to zero before each row. Rows of 1024 threads, which are not asked for ahead: 4096 x 5120 bf16 beside an f32
// stream 69.6 us (59 at the rate of a copy), 4096 x 8192 102 (94), 1500 x 16384 bf16 52.5 (34.5); 1000 x 32768 f32, whose values do not fit the registers either, 236 (92).
const char* kBackward = R"HIP(
template <bool MORE> __device__ __forceinline__ void backward(u64 rows, u32 blocks, const elem_t* dy, const stream_t* h, const param_t* __restrict__ gamma,
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
    // A row's operands are asked for while the row before is worked on, but for rows of 1024 threads: those have 128 registers each, which is too few for the widest rows (with
    // the prefetch, 16384 bf16 with dh and 16384 f32 spill; 8192 beside an f32 stream would fit in 100, and are not told apart). The loads are
    // the same for every thread and row, from the last one's place where there is none: loads under a condition would be waited for at once.
    struct Row { elem_v dy[NV]; stream_v h[NV], dh[NV]; float rstd; } next;
    auto load = [&](Row& r, u64 row) {
        row = row < rows ? row : rows - 1;
        r.rstd = rstd_of[row];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const u32 c = (p.l + k * L) * V;
            const u64 at = row * C + (c + V > C ? C - V : c);
            r.dy[k] = *(const elem_v*)(dy + at);
            r.h[k] = *(const stream_v*)(h + at);
            if (MORE) r.dh[k] = *(const stream_v*)(dh + at);
        }
    };
    // (gamma stays as well: a load between a row's and the next row's would be waited for with both)
#if T < 1024
    float held[NV][V];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < V; i++) held[k][i] = HAS(p, k) ? (float)gamma[start(p, k) + i] : 0.0f;
#define GAMMA(k, i) held[k][i]
#else
#define GAMMA(k, i) (float)gamma[start(p, k) + (i)]
#endif
    const u64 step = (u64)blocks * ROWS;
    u32 turn = 0;
    load(next, (u64)blockIdx.x * ROWS + p.slot);
    for (u64 first = (u64)blockIdx.x * ROWS; first < rows; first += step, turn ^= 1) {
        const u64 row = first + p.slot;
        const bool there = row < rows;
        const Row r = next;
        if (T < 1024) load(next, row + step);
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; k++)
            if (there && HAS(p, k))
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (counts(p, k, i)) {
                        const float t = (float)AT(r.dy[k], i) * ((float)AT(r.h[k], i) * r.rstd);
                        sum += t * GAMMA(k, i);
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
                    const float xh = (float)AT(r.h[k], i) * r.rstd;
                    float d = ((float)AT(r.dy[k], i) * GAMMA(k, i) - xh * mean) * r.rstd;
                    if (MORE) d += (float)AT(r.dh[k], i);
                    AT(out, i) = (elem_t)d;
                    AT(more, i) = (stream_t)d;
                }
                if (dx) STORE(true, (elem_v*)(dx + at), out);
                if (dresidual) STORE(true, (stream_v*)(dresidual + at), more);
            }
        if (T == 1024) load(next, row + step);
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
#define BACKWARD(name, more) \
    extern "C" __global__ __launch_bounds__(T) void name(u64 rows, u32 blocks, const elem_t* dy, const stream_t* h, const param_t* gamma, const float* rstd, const stream_t* dh, elem_t* dx, stream_t* dresidual, float* parts) { backward<more>(rows, blocks, dy, h, gamma, rstd, dh, dx, dresidual, parts); }
BACKWARD(rows_backward, false)
#if RESIDUAL
BACKWARD(rows_backward_more, true)   // with what reaches h from elsewhere
#endif

// dgamma[c] = the sum of `count` shares: 16 columns to a workgroup, the shares dealt to its 64 rows of threads. 256 shares of 4096 columns 4.7 us; 16 columns are half a line of 128
// bytes, and the workgroups that have its halves run on different XCDs: 8.4 MB are fetched of 4.2.
extern "C" __global__ __launch_bounds__(1024) void rows_fold(const float* __restrict__ parts, u32 count, float* __restrict__ dgamma) {
    __shared__ float part[16][16];
    const u32 column = threadIdx.x & 15u, row = threadIdx.x >> 4, c = blockIdx.x * 16 + column;
    float s = 0.0f;
    if (c < C)
#pragma unroll 8
        for (u32 n = row; n < count; n += 64) s += parts[(u64)n * C + c];
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    if ((threadIdx.x & 63u) < 16) part[threadIdx.x >> 6][column] = s;
    __syncthreads();
    if (threadIdx.x < 16 && c < C) {
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

std::string definitions(const RowProblem& pr, const RowTiling& t) {
    std::ostringstream s;
    s << "#define C " << pr.columns << "\n#define V " << t.vec << "\n#define NV " << t.vectors << "\n#define L " << t.lanes << "\n#define T " << t.threads
      << "\n#define BF16 " << (pr.dtype == HE_BF16) << "\n#define F16 " << (pr.dtype == HE_F16) << "\n#define STREAM_SAME "
      << (pr.stream_dtype() == pr.dtype) << "\n#define PARAM_SAME " << (pr.param_dtype == pr.dtype) << "\n#define RESIDUAL " << pr.residual()
      << "\n#define TO_I8 " << pr.to_i8 << "\n#define PITCH " << quantized_pitch(pr.columns) << "ull\n#define EPS "
      << strfmt("%.9ef", (double)pr.epsilon) << "\n#define X_ALIGN " << std::min(t.vec * value_bytes(pr.dtype), row_alignment(pr.columns * value_bytes(pr.dtype))) << "\n#define H_ALIGN "
      << std::min(t.vec * value_bytes(pr.stream_dtype()), row_alignment(pr.columns * value_bytes(pr.stream_dtype()))) << "\n";
    return s.str();
}

}  // namespace

std::string RowTiling::describe() const { return strfmt("vec=%d vectors=%d lanes=%d threads=%d", vec, vectors, lanes, threads); }

RowTiling plan_rows(const RowProblem& pr) {
    // 16 bytes of the wider type in an access, and two accesses of each operand to a thread (one to four are within 5% of each other on 8192 x 4096 and 2000 x
    // 1024, in bf16 and f32; eight, a row to a wave, take 51.5 instead of 47.4 us).
    RowTiling t;
    t.vec = 16 / std::max(value_bytes(pr.dtype), value_bytes(pr.stream_dtype()));
    while (t.vec > pr.columns) t.vec /= 2;
    const int64_t vectors = (pr.columns + t.vec - 1) / t.vec;
    t.lanes = std::min(1024, pow2_ceil((vectors + 1) / 2));
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
    tiling_ = plan_rows(pr);
    const std::string text = definitions(pr, tiling_) + kCommon, back = text + kBackward;
    const bool has_back = pr.norm && !pr.to_i8;
    auto compiled = std::async(std::launch::async, [&] { if (has_back) (void)rtc_compile(back, "rows_backward", {}); });
    source_ = text + kBytes + (pr.norm ? kForward : kQuantize);
    forward_ = std::make_unique<JitKernel>(source_, pr.norm ? "rows_forward" : "rows_quantize");
    if (pr.norm) forward_few_ = std::make_unique<JitKernel>(source_, "rows_forward_few");
    compiled.get();
    if (has_back) {
        backward_ = std::make_unique<JitKernel>(back, "rows_backward");
        if (pr.residual()) backward_more_ = std::make_unique<JitKernel>(back, "rows_backward_more");
        fold_ = std::make_unique<JitKernel>(back, "rows_fold");
        source_ += "\n" + back;
    }
    describe_ = std::string(pr.norm ? "rms_norm " : "quantize_rows ") + tiling_.describe();
}

RmsNorm::~RmsNorm() { scratch_.release(); }

namespace {
constexpr int kCUs = 256;
void check_tensor(const char* what, const void* p, int64_t alignment) {
    HE_REQUIRE(p && ((uintptr_t)p & (alignment - 1)) == 0, HE_ERR_INVALID, "%s is null or not aligned to %lld bytes", what, (long long)alignment);
}
}  // namespace

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
    const RowTiling& t = tiling_;
    const uint64_t blocks = ((uint64_t)rows + t.rows() - 1) / t.rows();
    HE_REQUIRE(blocks < kThreads / t.threads, HE_ERR_UNSUPPORTED, "%lld rows are too many for one launch", (long long)rows);
    uint64_t count = (uint64_t)rows;
    const uint32_t grid[3] = {(uint32_t)blocks, 1, 1}, block[3] = {(uint32_t)t.threads, 1, 1};
    void* args[] = {&count, &x, &gamma, &residual, &new_residual, &y, &rstd, &scales};
    void* quantize_args[] = {&count, &x, &y, &scales};
    // (results of 4 MB and more in 16 bits bypass the caches: 8192 x 4096 48.6 -> 47.1 us; asking in the kernel cost as much again)
    const bool few = pr_.norm && rows * pr_.columns < (1 << 21);
    (few ? forward_few_ : forward_)->launch(grid, block, 0, stream, pr_.norm ? args : quantize_args, true);
}

void RmsNorm::backward(int64_t rows, const void* dy, const void* h, const void* gamma, const float* rstd, const void* dh, void* dx, void* dresidual,
                       float* dgamma, hipStream_t stream) {
    HE_REQUIRE(backward_, HE_ERR_UNSUPPORTED, "rms norm: an output in 8 bits has no gradient");
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
    // (one workgroup to a CU where it has one row at a time, otherwise two: 8192 x 4096 bf16 50.6 and 52.5 us, 1517 x 2867 16.4 and 17.5; 8192 x 1024 f32 20.0 and
    // 19.0, 30000 x 256 bf16 15.3 and 14.6. Four: 57.0, 21.2, 20.4, 15.4)
    const uint64_t most = (uint64_t)kCUs * (tiling_.rows() == 1 ? 1 : 2);
    uint32_t blocks = (uint32_t)std::min<uint64_t>(most, ((uint64_t)rows + tiling_.rows() - 1) / tiling_.rows());
    uint64_t count = (uint64_t)rows;
    const uint32_t grid[3] = {blocks, 1, 1}, block[3] = {(uint32_t)tiling_.threads, 1, 1};
    const uint32_t fold_grid[3] = {(uint32_t)((pr_.columns + 15) / 16), 1, 1}, fold_block[3] = {1024, 1, 1};
    std::lock_guard<std::mutex> lk(mu_);
    // (asked for whatever the rows are, so that a stream's first call is the one that allocates; one workgroup's share is the sum already)
    float* const scratch = scratch_.get(most * pr_.columns, 0, stream).floats;
    float* parts = blocks == 1 ? dgamma : scratch;
    void* args[] = {&count, &blocks, &dy, &h, &gamma, &rstd, &dh, &dx, &dresidual, &parts};
    if (blocks) (dh ? backward_more_ : backward_)->launch(grid, block, 0, stream, args, blocks == 1);
    if (blocks == 1) return;
    void* fold_args[] = {&parts, &blocks, &dgamma};
    fold_->launch(fold_grid, fold_block, 0, stream, fold_args, true);
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
