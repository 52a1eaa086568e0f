#include "muon.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <sstream>

namespace he {

namespace {

constexpr int kGroup = 32;       // matrices whose operands one launch takes by value
constexpr uint32_t kPart = 8192; // elements of one share of a sum of squares
constexpr uint32_t kBlock = 64;  // rows and columns of one block of the conversions

// Newton-Schulz iteration on f16 matrix cores. With X scaled to a Frobenius norm of at most 1, no singular value ever leaves
// [0, 1.21]: the step's polynomial a s + b s^3 + c s^5 maps [0, 1] there and [1, 1.21] into [0.68, 0.96]. So every entry has a known
// bound, and fixed powers of two keep f16 operands in range: X 2^12 (at most 4956 of 65504), A 2^13 (1.47 2^13), B 2^13 (|b s + c s^2|
// stays below 2.81). A value's f16 rounding has 11 bits; its remainder in a second f16 gives 22, and three of the four products of
// such pairs (the fourth is 2^-22 of the result) run at three times f16's cost, where f32 matrix instructions take sixteen times.
// Measured against 64 bits: errors as of f32 products, 1e-6 to 1e-5.
const char* kCommon = R"HIP(
typedef unsigned short u16;
typedef unsigned int u32;
typedef unsigned long long u64;
typedef _Float16 f16_t;
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef u32 u32x4 __attribute__((ext_vector_type(4)));
#if BF16
typedef __bf16 elem_t;
#elif F16
typedef _Float16 elem_t;
#else
typedef float elem_t;
#endif
#ifndef LDS_AS
#define LDS_AS __attribute__((address_space(3)))
#define GLOBAL_AS __attribute__((address_space(1)))
#endif
#ifndef WAIT_LOADS
#define WAIT_LOADS(n) (0x0070 | ((n) & 15) | (((n) >> 4) << 14))   /* vmcnt(n), and lgkmcnt(0): this wave's reads of LDS are done */
#endif
#ifndef KERNEL_ATTRS
#define KERNEL_ATTRS __attribute__((amdgpu_waves_per_eu(2, 2)))
#endif
#ifndef HE_WS_STORE
// Partial results on their way to another workgroup: device-scope accesses go past the L2 of the XCD they come from, so what is
// written this way and waited for before a ticket is taken is there for whoever sees the ticket.
#define HE_WS_STORE(p, v) __hip_atomic_store((p), (v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
#define HE_WS_LOAD(p) __hip_atomic_load((p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
#define HE_WS_TICKET(p) __hip_atomic_fetch_add((p), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
#endif
struct Matrix {
    u32 rows, cols, mp, np;
    u32 tall, first_part, parts;
    float shape_scale;
    u64 x, xt[2], a, b, x_low;
};
struct Block { u32 matrix, i, j; };
struct Task { u32 matrix, i, j, k_begin, k_end, slot, share, shares; };
struct Operands {
    const elem_t* in[GROUP];
    const float* momentum[GROUP];
    float* new_momentum[GROUP];
    const float* weight[GROUP];
    void* out[GROUP];
    u32 first;   // the group's first matrix
    float learning_rate, mu, weight_decay;
    int nesterov;
};
#define X_SCALE 4096.0f
#define A_SCALE 8192.0f
#define B_SCALE 8192.0f
#define NS_A 3.4445f
#define NS_B -4.7750f
#define NS_C 2.0315f

// Matrices of the workspace are rows of chunks of 8 values: with PARTS == 2 the chunk's high parts, then its low ones, so that a row's
// 128 bytes are 32 values in two parts or 64 in one and are moved alike.
#define PARTS (SPLIT ? 2 : 1)
__device__ __forceinline__ u64 chunk_at(u64 row, u32 col, u32 pitch) { return (row * pitch + col) * PARTS; }   // col: a multiple of 8

__device__ __forceinline__ f16x8 high_of(const float (&v)[8]) {
    f16x8 h;
#pragma unroll
    for (int e = 0; e < 8; e++) h[e] = (f16_t)v[e];
    return h;
}
__device__ __forceinline__ f16x8 low_of(const float (&v)[8], f16x8 h) {
    f16x8 l;
#pragma unroll
    for (int e = 0; e < 8; e++) l[e] = (f16_t)(v[e] - (float)h[e]);
    return l;
}
// Eight values of a row. `low`: where the low parts go if the format has none (may be null).
__device__ __forceinline__ void put(f16_t* __restrict__ to, u64 row, u32 col, u32 pitch, const float (&v)[8], f16_t* __restrict__ low) {
    const f16x8 h = high_of(v);
    f16_t* at = to + chunk_at(row, col, pitch);
    *(f16x8*)at = h;
    if (SPLIT) *(f16x8*)(at + 8) = low_of(v, h);
    else if (low) *(f16x8*)(low + row * pitch + col) = low_of(v, h);
}
__device__ __forceinline__ void get(const f16_t* __restrict__ from, u64 row, u32 col, u32 pitch, float (&v)[8], const f16_t* __restrict__ low) {
    const f16_t* at = from + chunk_at(row, col, pitch);
    const f16x8 h = *(const f16x8*)at;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)h[e];
    if (SPLIT || low) {
        const f16x8 l = *(const f16x8*)(SPLIT ? at + 8 : low + row * pitch + col);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += (float)l[e];
    }
}

// Up to eight neighbouring values of a caller's row; `whole`: all eight are there, at an address that a vector access may have.
template <class E> __device__ __forceinline__ void row_of(const E* __restrict__ from, u32 left, bool whole, float (&v)[8]) {
    typedef E vec_t __attribute__((ext_vector_type(16 / sizeof(E))));
    if (whole) {
#pragma unroll
        for (u32 b = 0; b < 8 * sizeof(E) / 16; b++) {
            const vec_t x = ((const vec_t*)from)[b];
#pragma unroll
            for (u32 e = 0; e < 16 / sizeof(E); e++) v[b * (16 / sizeof(E)) + e] = (float)x[e];
        }
    } else {
#pragma unroll
        for (u32 e = 0; e < 8; e++) v[e] = e < left ? (float)from[e] : 0.0f;
    }
}
template <class E> __device__ __forceinline__ void row_to(E* __restrict__ to, u32 left, bool whole, const float (&v)[8]) {
    typedef E vec_t __attribute__((ext_vector_type(16 / sizeof(E))));
    if (whole) {
#pragma unroll
        for (u32 b = 0; b < 8 * sizeof(E) / 16; b++) {
            vec_t x;
#pragma unroll
            for (u32 e = 0; e < 16 / sizeof(E); e++) x[e] = (E)v[b * (16 / sizeof(E)) + e];
            ((vec_t*)to)[b] = x;
        }
    } else {
#pragma unroll
        for (u32 e = 0; e < 8; e++)
            if (e < left) to[e] = (E)v[e];
    }
}

// Eight neighbouring values of the matrix that is orthogonalised (zeros beyond it): of the operand itself, or of the step's update,
// from the gradient and the new momentum.
template <bool STEP> __device__ __forceinline__ void updates_of(const Operands& o, u32 k, u32 r, u32 c, u32 rows, u32 cols, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.0f;
    if (r >= rows || c >= cols) return;
    const u64 at = (u64)r * cols + c;
    const bool whole = cols % 8 == 0;
    if (!STEP || o.nesterov) row_of<elem_t>(o.in[k] + at, cols - c, whole, v);
    if (STEP) {
        float m[8];
        row_of<float>(o.new_momentum[k] + at, cols - c, whole, m);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = o.nesterov ? v[e] + o.mu * m[e] : m[e];
    }
}
)HIP";

const char* kElements = R"HIP(
// Shares of |U|^2, in 64 bits: squares of f32 neither overflow nor vanish there. The step's first pass also writes the new momenta.
template <bool STEP> __device__ __forceinline__ void norm_part(const Matrix* __restrict__ mats, const Block* __restrict__ parts, double* __restrict__ sums, const Operands& o) {
    __shared__ double wave_sums[4];
    const Block t = parts[blockIdx.x];
    const u32 k = t.matrix - o.first;
    const u64 size = (u64)mats[t.matrix].rows * mats[t.matrix].cols, begin = (u64)t.i * PART, end = begin + PART < size ? begin + PART : size;
    double s = 0.0;
    for (u64 e = begin + threadIdx.x * 8; e < end; e += 2048) {
        const u32 left = end - e < 8 ? (u32)(end - e) : 8u;
        float u[8];
        row_of<elem_t>(o.in[k] + e, left, left == 8, u);
        if (STEP) {
            float m[8];
            row_of<float>(o.momentum[k] + e, left, left == 8, m);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                m[i] = o.mu * m[i] + u[i];
                u[i] = o.nesterov ? u[i] + o.mu * m[i] : m[i];
            }
            row_to<float>(o.new_momentum[k] + e, left, left == 8, m);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) s += (double)u[i] * (double)u[i];
    }
    for (int m = 32; m > 0; m /= 2) s += SHFL_XOR_F64(s, m);
    if ((threadIdx.x & 63u) == 0) wave_sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) sums[blockIdx.x + t.j] = wave_sums[0] + wave_sums[1] + wave_sums[2] + wave_sums[3];
}

// U / (|U| + floor) in f16 parts, in both orientations, zeros beyond the matrix. A block of 64 x 64: 8 lanes take the 64 columns of a
// row, 8 values each.
template <bool STEP> __device__ __forceinline__ void convert_block(const Matrix* __restrict__ mats, const Block* __restrict__ blocks, const double* __restrict__ sums, char* __restrict__ ws, const Operands& o) {
    __shared__ float tile[64][65];
    __shared__ double total;
    const Block t = blocks[blockIdx.x];
    const Matrix& m = mats[t.matrix];
    const u32 k = t.matrix - o.first, rows_p = m.tall ? m.np : m.mp, cols_p = m.tall ? m.mp : m.np, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    if (wave == 0) {
        double s = 0.0;
        for (u32 p = lane; p < m.parts; p += 64) s += sums[m.first_part + p];
        for (int d = 32; d > 0; d /= 2) s += SHFL_XOR_F64(s, d);
        if (lane == 0) total = s;
    }
    __syncthreads();
    const double scale = (double)X_SCALE / (sqrt(total) + (double)NORM_FLOOR);
    f16_t *natural = (f16_t*)(ws + (m.tall ? m.xt[0] : m.x)), *turned = (f16_t*)(ws + (m.tall ? m.x : m.xt[0])), *low = (f16_t*)(ws + m.x_low);
    const u32 c = t.j * 64 + (lane & 7u) * 8;
#pragma unroll
    for (u32 pass = 0; pass < 2; pass++) {
        const u32 i = pass * 32 + wave * 8 + (lane >> 3), r = t.i * 64 + i;
        float v[8];
        updates_of<STEP>(o, k, r, c, m.rows, m.cols, v);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = (float)((double)v[e] * scale);
            tile[i][(lane & 7u) * 8 + e] = v[e];
        }
        put(natural, r, c, cols_p, v, SPLIT || m.tall ? nullptr : low);
    }
    __syncthreads();
#pragma unroll
    for (u32 pass = 0; pass < 2; pass++) {
        const u32 i = pass * 32 + wave * 8 + (lane >> 3);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = tile[(lane & 7u) * 8 + e][i];
        put(turned, t.j * 64 + i, t.i * 64 + (lane & 7u) * 8, rows_p, v, SPLIT || !m.tall ? nullptr : low);
    }
}

// The last X to where it goes, by way of LDS where the matrix was iterated as its transpose.
template <bool STEP> __device__ __forceinline__ void finish_block(const Matrix* __restrict__ mats, const Block* __restrict__ blocks, const char* __restrict__ ws, const Operands& o) {
    __shared__ float tile[64][65];
    const Block t = blocks[blockIdx.x];
    const Matrix& m = mats[t.matrix];
    const u32 k = t.matrix - o.first, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = t.j * 64 + (lane & 7u) * 8;
    const f16_t *from = (const f16_t*)(ws + m.x), *low = SPLIT ? nullptr : (const f16_t*)(ws + m.x_low);
    if (m.tall) {
#pragma unroll
        for (u32 pass = 0; pass < 2; pass++) {
            const u32 i = pass * 32 + wave * 8 + (lane >> 3);
            float v[8];
            get(from, t.j * 64 + i, t.i * 64 + (lane & 7u) * 8, m.np, v, low);
#pragma unroll
            for (int e = 0; e < 8; e++) tile[(lane & 7u) * 8 + e][i] = v[e];
        }
        __syncthreads();
    }
#pragma unroll
    for (u32 pass = 0; pass < 2; pass++) {
        const u32 i = pass * 32 + wave * 8 + (lane >> 3), r = t.i * 64 + i;
        if (r >= m.rows || c >= m.cols) continue;
        float v[8];
        if (m.tall)
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = tile[i][(lane & 7u) * 8 + e];
        else get(from, r, c, m.np, v, low);
        const u64 e0 = (u64)r * m.cols + c;
        const bool whole = c + 8 <= m.cols && m.cols % 8 == 0;
        if (STEP) {
            float w[8];
            row_of<float>(o.weight[k] + e0, m.cols - c, whole, w);
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = (w[e] - o.learning_rate * o.weight_decay * w[e]) - o.learning_rate * m.shape_scale * (v[e] * (1.0f / X_SCALE));
            row_to<float>((float*)o.out[k] + e0, m.cols - c, whole, w);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] *= 1.0f / X_SCALE;
            row_to<elem_t>((elem_t*)o.out[k] + e0, m.cols - c, whole, v);
        }
    }
}

extern "C" __global__ __launch_bounds__(256) void muon_norm(const Matrix* __restrict__ mats, const Block* __restrict__ parts, double* __restrict__ sums, Operands o) { norm_part<false>(mats, parts, sums, o); }
extern "C" __global__ __launch_bounds__(256) void muon_norm_step(const Matrix* __restrict__ mats, const Block* __restrict__ parts, double* __restrict__ sums, Operands o) { norm_part<true>(mats, parts, sums, o); }
extern "C" __global__ __launch_bounds__(256) void muon_convert(const Matrix* __restrict__ mats, const Block* __restrict__ blocks, const double* __restrict__ sums, char* __restrict__ ws, Operands o) { convert_block<false>(mats, blocks, sums, ws, o); }
extern "C" __global__ __launch_bounds__(256) void muon_convert_step(const Matrix* __restrict__ mats, const Block* __restrict__ blocks, const double* __restrict__ sums, char* __restrict__ ws, Operands o) { convert_block<true>(mats, blocks, sums, ws, o); }
extern "C" __global__ __launch_bounds__(256) void muon_finish(const Matrix* __restrict__ mats, const Block* __restrict__ blocks, const char* __restrict__ ws, Operands o) { finish_block<false>(mats, blocks, ws, o); }
extern "C" __global__ __launch_bounds__(256) void muon_finish_step(const Matrix* __restrict__ mats, const Block* __restrict__ blocks, const char* __restrict__ ws, Operands o) { finish_block<true>(mats, blocks, ws, o); }
)HIP";

// One kernel for the three products of a step, each of the form R = alpha P Q^T + beta E with P, Q row-major and contiguous along the
// sum (X and its transpose are both kept for that; A and B are symmetric):
//   gram    A = X X^T           P = Q = X            lower tiles, stored twice
//   square  B = b A + c A A     P = Q = A, E = A     lower tiles, stored twice
//   apply   X = a X + B X       P = B, Q = XT, E = X  whole, stored as X and as XT
const char* kProduct = R"HIP(
#define BM TILE
#define BN TILE
#define WAVES (WAVES_M * WAVES_N)
#define WTM (BM / WAVES_M)
#define WTN (BN / WAVES_N)
#define MB (WTM / 32)
#define NB (WTN / 32)
#define BK (64 / PARTS)                 /* values of a row in a k-tile: 128 bytes */
#define KS (BK / 16)                    /* matrix instructions along a k-tile */
#define STAGE_HALVES ((BM + BN) * 64)
#define LOADS ((BM + BN) / 8 / WAVES)   /* direct loads of a wave per k-tile: 8 rows of 128 bytes each */
#define SROWS (WTM < 64 ? WTM : 64)     /* a wave's strip: rows and columns of results that go through LDS at a time */
#define SCOLS (WTN < 64 ? WTN : 64)
#define STRIP_PITCH (SCOLS + 1)         /* odd: rows and columns are both read without bank conflicts */
#define STRIP_FLOATS (WAVES * SROWS * STRIP_PITCH)
#define LDS_HALVES (STAGES * STAGE_HALVES > 2 * STRIP_FLOATS ? STAGES * STAGE_HALVES : 2 * STRIP_FLOATS)
enum { GRAM, SQUARE, APPLY };

__device__ __forceinline__ void strip_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int STAGE> __device__ __forceinline__ void product(const Matrix* __restrict__ mats, const Task* __restrict__ tasks, char* __restrict__ ws, float* __restrict__ shared_tiles, u32* __restrict__ tickets, u32 turn, u32 last_step) {
    __shared__ __attribute__((aligned(16))) f16_t lds[LDS_HALVES];
    __shared__ u32 last;
    const Task t = tasks[blockIdx.x];
    const Matrix& m = mats[t.matrix];
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave_m = wave / WAVES_N, wave_n = wave % WAVES_N;
    const u32 k_len = (STAGE == GRAM ? m.np : m.mp) * PARTS;   // halves of a row
    const f16_t* p_rows = (const f16_t*)(ws + (STAGE == GRAM ? m.x : STAGE == SQUARE ? m.a : m.b)) + (u64)t.i * BM * k_len;
    const f16_t* q_rows = (const f16_t*)(ws + (STAGE == GRAM ? m.x : STAGE == SQUARE ? m.a : m.xt[turn])) + (u64)t.j * BN * k_len;
    // Direct loads: lane l of the load of rows 8 r .. 8 r + 7 takes row l / 8 and, so that fragment reads of 8 neighbouring rows
    // meet 8 different bank groups, the chunk (l % 8) ^ (l / 8) of its 128 bytes.
    const u32 lane_off = (lane >> 3) * k_len + (((lane & 7u) ^ (lane >> 3)) << 3);
    auto fetch = [&](u32 kt, u32 slot) {
        f16_t* base = lds + slot * STAGE_HALVES;
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const u32 row = (wave * LOADS + l) * 8;   // of P's rows, then Q's
            const f16_t* src = (row < BM ? p_rows + (u64)row * k_len : q_rows + (u64)(row - BM) * k_len) + (u64)kt * 64 + lane_off;
            __builtin_amdgcn_global_load_lds((const GLOBAL_AS u32*)src, (LDS_AS u32*)(base + row * 64), 16, 0, 0);
        }
    };
    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
    const u32 frag_row = lane & 31u, half = lane >> 5, swz = lane & 7u;
    u32 slot = 0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++)
        if (t.k_begin + s < t.k_end) fetch(t.k_begin + s, s);
    for (u32 kt = t.k_begin; kt < t.k_end; kt++) {
        // this wave's loads of the k-tile have landed (those of the STAGES - 2 behind it may be on their way), then the other waves'
        if (kt + STAGES - 2 < t.k_end) __builtin_amdgcn_s_waitcnt(WAIT_LOADS((STAGES - 2) * LOADS));
        else __builtin_amdgcn_s_waitcnt(WAIT_LOADS(0));
        // (the bare barrier: __syncthreads() would wait for all loads; no wave still reads the stage that is filled next)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (kt + STAGES - 1 < t.k_end) fetch(kt + STAGES - 1, slot + STAGES - 1 < STAGES ? slot + STAGES - 1 : slot - 1);
        const f16_t *p = lds + slot * STAGE_HALVES + (wave_m * WTM + frag_row) * 64, *q = lds + slot * STAGE_HALVES + (BM + wave_n * WTN + frag_row) * 64;
#pragma unroll
        for (int kk = 0; kk < KS; kk++) {
            f16x8 a[PARTS][MB], b[PARTS][NB];
#pragma unroll
            for (int part = 0; part < PARTS; part++) {
                const u32 chunk = (((kk * 2 + half) * PARTS + part) ^ swz) * 8;
#pragma unroll
                for (int i = 0; i < MB; i++) a[part][i] = *(const f16x8*)(p + i * 32 * 64 + chunk);
#pragma unroll
                for (int j = 0; j < NB; j++) b[part][j] = *(const f16x8*)(q + j * 32 * 64 + chunk);
            }
            // high x high, high x low, low x high
#pragma unroll
            for (int c = 0; c < (SPLIT ? 3 : 1); c++)
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int j = 0; j < NB; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[c == 2][i], b[c == 1][j], acc[i][j], 0, 0, 0);
        }
        slot = slot + 1 < STAGES ? slot + 1 : 0;
    }

    // A tile whose sum several workgroups share: each parks its part, the last to arrive adds them up in their order and goes on.
    if (t.shares > 1) {
        u64* mine = (u64*)(shared_tiles + (u64)(t.slot + t.share) * (BM * BN)) + wave * (WTM * WTN / 2) + lane;
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float two[2] = {acc[i][j][2 * e], acc[i][j][2 * e + 1]};
                    HE_WS_STORE(mine + ((i * NB + j) * 8 + e) * 64, __builtin_bit_cast(u64, two));
                }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (threadIdx.x == 0) last = HE_WS_TICKET(tickets + t.slot) + 1 == t.shares;
        __syncthreads();
        if (!last) return;
        if (threadIdx.x == 0) HE_WS_STORE(tickets + t.slot, 0u);   // as the next launch wants it
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
        for (u32 s = 0; s < t.shares; s++) {
            const u64* from = (const u64*)(shared_tiles + (u64)(t.slot + s) * (BM * BN)) + wave * (WTM * WTN / 2) + lane;
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int j = 0; j < NB; j++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        struct Two { float v[2]; } two = __builtin_bit_cast(Two, HE_WS_LOAD(from + ((i * NB + j) * 8 + e) * 64));
                        acc[i][j][2 * e] += two.v[0];
                        acc[i][j][2 * e + 1] += two.v[1];
                    }
        }
    }
    __syncthreads();   // the operand stages become the waves' strips

    // Results: a lane holds rows (e / 4) * 8 + half * 4 + e % 4 of column lane % 32 of each 32 x 32 block. Through a strip in LDS a lane gets
    // 8 neighbours of a row, adds E, stores them, and puts them back for the transposed copy.
    const u32 pitch = STAGE == APPLY ? m.np : m.mp;
    const f16_t* e_rows = (const f16_t*)(ws + (STAGE == SQUARE ? m.a : m.x));
    f16_t *plain = (f16_t*)(ws + (STAGE == GRAM ? m.a : STAGE == SQUARE ? m.b : m.x)), *turned = (f16_t*)(ws + (STAGE == GRAM ? m.a : STAGE == SQUARE ? m.b : m.xt[turn ^ 1u]));
    // (of X the low part counts in either precision: what f16 drops of a X in each step would stay dropped, and the small
    // singular values with it)
    f16_t* low = STAGE == APPLY && !SPLIT ? (f16_t*)(ws + m.x_low) : nullptr;
    float* strip = (float*)lds + wave * (SROWS * STRIP_PITCH);
    const bool mirrored = STAGE == APPLY ? !last_step : t.i != t.j;
    constexpr u32 row_lanes = SCOLS / 8, col_lanes = SROWS / 8;   // lanes along a row of the strip, and along a column
#pragma unroll
    for (int i = 0; i < WTM / SROWS; i++)
#pragma unroll
        for (int j = 0; j < WTN / SCOLS; j++) {
            const u32 row0 = t.i * BM + wave_m * WTM + i * SROWS, col0 = t.j * BN + wave_n * WTN + j * SCOLS;
#pragma unroll
            for (int di = 0; di < SROWS / 32; di++)
#pragma unroll
                for (int dj = 0; dj < SCOLS / 32; dj++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        strip[(di * 32 + (e / 4) * 8 + half * 4 + e % 4) * STRIP_PITCH + dj * 32 + frag_row] = acc[i * (SROWS / 32) + di][j * (SCOLS / 32) + dj][e];
            strip_sync();
#pragma unroll
            for (u32 s = 0; s < SROWS * row_lanes / 64; s++) {
                const u32 r = s * (64 / row_lanes) + lane / row_lanes, c = lane % row_lanes * 8;
                float v[8], other[8];
                if (STAGE != GRAM) get(e_rows, row0 + r, col0 + c, pitch, other, low);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float sum = strip[r * STRIP_PITCH + c + e];
                    v[e] = STAGE == GRAM ? sum * (A_SCALE / (X_SCALE * X_SCALE))
                         : STAGE == SQUARE ? NS_B * other[e] + (NS_C * B_SCALE / (A_SCALE * A_SCALE)) * sum
                                           : NS_A * other[e] + (1.0f / B_SCALE) * sum;
                    strip[r * STRIP_PITCH + c + e] = v[e];
                }
                put(plain, row0 + r, col0 + c, pitch, v, low);
            }
            strip_sync();
            if (mirrored)
#pragma unroll
                for (u32 s = 0; s < SCOLS * col_lanes / 64; s++) {
                    const u32 c = s * (64 / col_lanes) + lane / col_lanes, r = lane % col_lanes * 8;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = strip[(r + e) * STRIP_PITCH + c];
                    put(turned, col0 + c, row0 + r, m.mp, v, nullptr);
                }
            strip_sync();
        }
}

#define KERNEL(name, stage) extern "C" __global__ __launch_bounds__(WAVES * 64) KERNEL_ATTRS void name(const Matrix* __restrict__ mats, const Task* __restrict__ tasks, char* __restrict__ ws, float* __restrict__ shared_tiles, u32* __restrict__ tickets, u32 turn, u32 last_step) { product<stage>(mats, tasks, ws, shared_tiles, tickets, turn, last_step); }
KERNEL(muon_gram, GRAM)
KERNEL(muon_square, SQUARE)
KERNEL(muon_apply, APPLY)
)HIP";

struct OperandsArg {
    const void* in[kGroup];
    const float* momentum[kGroup];
    float* new_momentum[kGroup];
    const float* weight[kGroup];
    void* out[kGroup];
    uint32_t first;
    float learning_rate, mu, weight_decay;
    int32_t nesterov;
};

// Tasks in the order of their blocks: blocks are dealt round-robin to the 8 XCDs, each with an L2 of its own, so XCD x gets the
// x-th eighth of a sequence in which neighbours share rows and columns.
void deal(std::vector<MuonTask>& tasks) {
    const size_t n = tasks.size(), whole = n / 8, over = n % 8;
    std::vector<MuonTask> out(n);
    for (size_t b = 0; b < n; b++) {
        const size_t x = b % 8;
        out[b] = tasks[x * whole + std::min(x, over) + b / 8];
    }
    tasks.swap(out);
}

// The tasks of one product of every matrix: bands of four tile rows, column by column; a tile's sum is dealt to several workgroups
// where there are too few tiles to fill the chip. `slots`: workgroups that it runs at once; `least`: k-tiles a share has at least.
std::vector<MuonTask> tasks_of(const std::vector<MuonMatrix>& mats, uint32_t tile, bool lower, bool along_n, uint32_t bk, uint32_t slots, uint32_t least,
                               uint32_t* shared) {
    uint64_t units = 0, tiles = 0;
    for (const MuonMatrix& m : mats) {
        const uint64_t ti = m.mp / tile, count = lower ? ti * (ti + 1) / 2 : ti * (m.np / tile);
        tiles += count;
        units += count * ((along_n ? m.np : m.mp) / bk);
    }
    const uint64_t target = tiles >= slots ? units : std::max<uint64_t>(least, (units + slots - 1) / slots);
    std::vector<MuonTask> out;
    *shared = 0;
    for (size_t k = 0; k < mats.size(); k++) {
        const MuonMatrix& m = mats[k];
        const uint32_t ti = m.mp / tile, tj = lower ? ti : m.np / tile, kt = (along_n ? m.np : m.mp) / bk;
        const uint32_t shares = (uint32_t)std::max<uint64_t>(1, kt / target);
        for (uint32_t g = 0; g < ti; g += 4)
            for (uint32_t j = 0; j < tj; j++)
                for (uint32_t i = g; i < std::min(g + 4, ti); i++) {
                    if (lower && j > i) continue;
                    for (uint32_t s = 0; s < shares; s++)
                        out.push_back({(uint32_t)k, i, j, (uint32_t)((uint64_t)kt * s / shares), (uint32_t)((uint64_t)kt * (s + 1) / shares), *shared, s, shares});
                    if (shares > 1) *shared += shares;
                }
    }
    deal(out);
    return out;
}

int env_int(const char* name, int dflt) { return tuning::get_int(name, dflt); }

template <class T> std::vector<char> bytes_of(const std::vector<T>& v) {
    std::vector<char> out(v.size() * sizeof(T));
    if (!v.empty()) memcpy(out.data(), v.data(), out.size());
    return out;
}

}  // namespace

Muon::Muon(const MuonProblem& pr) : pr_(pr) {
    HE_REQUIRE(!pr.shapes.empty() && pr.shapes.size() <= 65536, HE_ERR_INVALID, "muon: %zu matrices, 1 to 65536 are taken", pr.shapes.size());
    HE_REQUIRE(pr.dtype == HE_F16 || pr.dtype == HE_BF16 || pr.dtype == HE_F32, HE_ERR_INVALID, "muon does not take dtype %s", dtype_name(pr.dtype));
    HE_REQUIRE(pr.steps >= 1 && pr.steps <= 32, HE_ERR_INVALID, "muon: %d steps, 1 to 32 are taken", pr.steps);
    const uint32_t tile = (uint32_t)env_int("HELIUM_HIP_MUON_TILE", 128), stages = (uint32_t)env_int("HELIUM_HIP_MUON_STAGES", 2), bk = pr.split ? 32 : 64;
    const uint32_t waves_m = tile == 64 ? 2 : 2, waves_n = tile == 256 ? 4 : 2;
    threads_ = waves_m * waves_n * 64;
    uint64_t at = 0, parts = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    std::vector<MuonBlock> shares, blocks;
    for (size_t k = 0; k < pr.shapes.size(); k++) {
        const int64_t rows = pr.shapes[k][0], cols = pr.shapes[k][1];
        HE_REQUIRE(rows >= 1 && cols >= 1, HE_ERR_INVALID, "muon: matrix %zu is %lld x %lld", k, (long long)rows, (long long)cols);
        HE_REQUIRE(std::max(rows, cols) <= (1 << 20) && std::min(rows, cols) <= 32768, HE_ERR_UNSUPPORTED,
                   "muon: matrix %zu is %lld x %lld; extents up to 2^20 by 32768 are taken", k, (long long)rows, (long long)cols);
        MuonMatrix m{};
        m.rows = (uint32_t)rows, m.cols = (uint32_t)cols, m.tall = rows > cols;
        auto padded = [&](int64_t v) { return (uint32_t)((v + tile - 1) / tile * tile); };
        m.mp = padded(std::min(rows, cols)), m.np = padded(std::max(rows, cols));
        m.shape_scale = (float)std::sqrt(std::max(1.0, (double)rows / (double)cols));
        const uint64_t bytes = pr.split ? 4 : 2, x = m.mp * bytes * m.np, a = m.mp * bytes * m.mp;
        m.x = take(x), m.xt[0] = take(x), m.xt[1] = take(x), m.a = take(a), m.b = take(a);
        if (!pr.split) m.x_low = take(x);
        const uint64_t size = (uint64_t)rows * cols;
        m.first_part = (uint32_t)parts;
        m.parts = (uint32_t)((size + kPart - 1) / kPart);
        parts += m.parts;
        part_begin_.push_back((uint32_t)shares.size());
        block_begin_.push_back((uint32_t)blocks.size());
        for (uint32_t p = 0; p < m.parts; p++) shares.push_back({(uint32_t)k, p, 0});
        const uint32_t br = (m.tall ? m.np : m.mp) / kBlock, bc = (m.tall ? m.mp : m.np) / kBlock;
        for (uint32_t i = 0; i < br; i++)
            for (uint32_t j = 0; j < bc; j++) blocks.push_back({(uint32_t)k, i, j});
        matrices_.push_back(m);
        HE_REQUIRE(blocks.size() < (1u << 30) && shares.size() < (1u << 30), HE_ERR_UNSUPPORTED, "muon: too many elements for one group");
    }
    part_begin_.push_back((uint32_t)shares.size());
    block_begin_.push_back((uint32_t)blocks.size());
    const uint32_t slots = 256 * (tile == 256 ? 1 : 2), least = (uint32_t)env_int("HELIUM_HIP_MUON_LEAST", 8);
    uint32_t shared[3];
    const std::vector<MuonTask> gram = tasks_of(matrices_, tile, true, true, bk, slots, least, &shared[0]),
                                square = tasks_of(matrices_, tile, true, false, bk, slots, least, &shared[1]),
                                apply = tasks_of(matrices_, tile, false, false, bk, slots, least, &shared[2]);
    const uint32_t most = std::max({shared[0], shared[1], shared[2]});
    tickets_ = most;
    tickets_at_ = take((uint64_t)most * 4);
    shared_at_ = take((uint64_t)most * tile * tile * 4);
    // (a share's place among the sums is its block's, plus where its launch begins)
    for (size_t k = 0; k < pr.shapes.size(); k++)
        for (uint32_t p = part_begin_[k]; p < part_begin_[k + 1]; p++) shares[p].j = part_begin_[k / kGroup * kGroup];
    workspace_bytes_ = take(parts * sizeof(double)) + parts * sizeof(double);
    tables_[0] = bytes_of(matrices_), tables_[1] = bytes_of(gram), tables_[2] = bytes_of(square), tables_[3] = bytes_of(apply);
    tables_[4] = bytes_of(shares), tables_[5] = bytes_of(blocks);
    table_size_ = {(uint32_t)matrices_.size(), (uint32_t)gram.size(), (uint32_t)square.size(), (uint32_t)apply.size(), (uint32_t)shares.size(), (uint32_t)blocks.size()};
    for (int t = 0; t < kTables; t++) {
        table_at_[t] = table_bytes_;
        table_bytes_ += (tables_[t].size() + 255) / 256 * 256;
    }
    std::ostringstream s;
    s << "#define GROUP " << kGroup << "\n#define PART " << kPart << "ull\n#define STEPS " << pr.steps << "\n#define SPLIT " << (int)pr.split << "\n#define BF16 "
      << (pr.dtype == HE_BF16) << "\n#define F16 " << (pr.dtype == HE_F16) << "\n#define NORM_FLOOR 1e-7\n#define TILE " << tile << "\n#define WAVES_M " << waves_m
      << "\n#define WAVES_N " << waves_n << "\n#define STAGES " << stages << "\n#ifndef SHFL_XOR_F64\n#define SHFL_XOR_F64(v, m) __shfl_xor(v, m, 64)\n#endif\n";
    source_ = s.str() + kCommon + kElements + kProduct;
    auto make = [&](const char* entry) { return std::make_unique<JitKernel>(source_, entry); };
    norm_ = make("muon_norm"), convert_ = make("muon_convert"), finish_ = make("muon_finish");
    norm_step_ = make("muon_norm_step"), convert_step_ = make("muon_convert_step"), finish_step_ = make("muon_finish_step");
    gram_ = make("muon_gram"), square_ = make("muon_square"), apply_ = make("muon_apply");
    describe_ = strfmt("muon matrices=%zu steps=%d parts=%d tile=%u threads=%u stages=%u gram=%u square=%u apply=%u shared=%u,%u,%u shares=%u blocks=%u tickets_at=%zu shared_at=%zu workspace=%zu",
                       pr.shapes.size(), pr.steps, pr.split ? 2 : 1, tile, threads_, stages, table_size_[1], table_size_[2], table_size_[3], shared[0], shared[1], shared[2],
                       table_size_[4], table_size_[5], tickets_at_, shared_at_, workspace_bytes_);
}

Muon::~Muon() {
    for (auto& kv : per_stream_) {
        (void)hipFree(kv.second.tables);
        (void)hipFree(kv.second.workspace);
    }
}

Muon::Buffers Muon::buffers(hipStream_t stream) {
    auto it = per_stream_.find(stream);
    if (it != per_stream_.end()) return it->second;
    Buffers b;
    HE_HIP(hipMalloc((void**)&b.tables, table_bytes_));
    hipError_t e = hipMalloc((void**)&b.workspace, workspace_bytes_);
    if (e == hipSuccess && tickets_) e = hipMemset(b.workspace + tickets_at_, 0, (size_t)tickets_ * 4);
    for (int t = 0; t < kTables && e == hipSuccess; t++) e = hipMemcpy(b.tables + table_at_[t], tables_[t].data(), tables_[t].size(), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        (void)hipFree(b.tables);
        (void)hipFree(b.workspace);
        fail(HE_ERR_HIP, strfmt("muon: %zu bytes of workspace: %s", workspace_bytes_, hipGetErrorString(e)));
    }
    per_stream_[stream] = b;
    return b;
}

void Muon::products(char* ws, char* tables, hipStream_t stream) {
    const uint32_t block[3] = {threads_, 1, 1};
    char *mats = tables + table_at_[0], *shared = ws + shared_at_, *tickets = ws + tickets_at_;
    for (int k = 0; k < pr_.steps; k++)
        for (int stage = 1; stage <= 3; stage++) {
            uint32_t turn = (uint32_t)k & 1u, last = k == pr_.steps - 1;
            char* tasks = tables + table_at_[stage];
            const uint32_t grid[3] = {table_size_[stage], 1, 1};
            void* args[] = {&mats, &tasks, &ws, &shared, &tickets, &turn, &last};
            (stage == 1 ? gram_ : stage == 2 ? square_ : apply_)->launch(grid, block, 0, stream, args);
        }
}

void Muon::orthogonalize(const void* const* in, void* const* out, hipStream_t stream) {
    step_or_not(in, nullptr, nullptr, nullptr, out, nullptr, stream);
}

void Muon::step(const void* const* grads, const float* const* momenta, const float* const* weights, float* const* new_momenta, float* const* new_weights,
                const MuonStep& how, hipStream_t stream) {
    step_or_not(grads, momenta, weights, new_momenta, (void* const*)new_weights, &how, stream);
}

void Muon::step_or_not(const void* const* in, const float* const* momenta, const float* const* weights, float* const* new_momenta, void* const* out,
                       const MuonStep* how, hipStream_t stream) {
    auto aligned = [](const void* p) { return p && ((uintptr_t)p & 15) == 0; };
    HE_REQUIRE(in && out && (!how || (momenta && weights && new_momenta)), HE_ERR_INVALID, "muon: a list of operands is null");
    for (size_t k = 0; k < count(); k++)
        HE_REQUIRE(aligned(in[k]) && aligned(out[k]) && (!how || (aligned(momenta[k]) && aligned(weights[k]) && aligned(new_momenta[k]))), HE_ERR_INVALID,
                   "muon: an operand of matrix %zu is null or not 16-byte aligned", k);
    if (how)
        HE_REQUIRE(std::isfinite(how->learning_rate) && std::isfinite(how->momentum) && std::isfinite(how->weight_decay), HE_ERR_INVALID,
                   "muon: learning rate, momentum or weight decay is not finite");
    std::lock_guard<std::mutex> lk(mu_);
    const Buffers b = buffers(stream);
    char *mats = b.tables + table_at_[0], *ws = b.workspace;
    double* sums = (double*)(ws + workspace_bytes_ - table_size_[4] * sizeof(double));
    const uint32_t block[3] = {256, 1, 1};
    auto each_group = [&](auto&& launch) {
        for (size_t first = 0; first < count(); first += kGroup) {
            OperandsArg o{};
            const size_t last = std::min(first + kGroup, count());
            for (size_t k = first; k < last; k++) {
                o.in[k - first] = in[k], o.out[k - first] = out[k];
                if (how) o.momentum[k - first] = momenta[k], o.new_momentum[k - first] = new_momenta[k], o.weight[k - first] = weights[k];
            }
            o.first = (uint32_t)first;
            if (how) o.learning_rate = how->learning_rate, o.mu = how->momentum, o.weight_decay = how->weight_decay, o.nesterov = how->nesterov;
            launch(o, first, last);
        }
    };
    each_group([&](OperandsArg& o, size_t first, size_t last) {
        char* parts = b.tables + table_at_[4] + part_begin_[first] * sizeof(MuonBlock);
        const uint32_t grid[3] = {part_begin_[last] - part_begin_[first], 1, 1};
        void* args[] = {&mats, &parts, &sums, &o};
        (how ? norm_step_ : norm_)->launch(grid, block, 0, stream, args);
    });
    each_group([&](OperandsArg& o, size_t first, size_t last) {
        char* blocks = b.tables + table_at_[5] + block_begin_[first] * sizeof(MuonBlock);
        const uint32_t grid[3] = {block_begin_[last] - block_begin_[first], 1, 1};
        void* args[] = {&mats, &blocks, &sums, &ws, &o};
        (how ? convert_step_ : convert_)->launch(grid, block, 0, stream, args);
    });
    products(ws, b.tables, stream);
    each_group([&](OperandsArg& o, size_t first, size_t last) {
        char* blocks = b.tables + table_at_[5] + block_begin_[first] * sizeof(MuonBlock);
        const uint32_t grid[3] = {block_begin_[last] - block_begin_[first], 1, 1};
        void* args[] = {&mats, &blocks, &ws, &o};
        (how ? finish_step_ : finish_)->launch(grid, block, 0, stream, args, last == count());
    });
}

}  // namespace he

// ---- C ABI ------------------------------------------------------------------------------------------------
struct he_muon_s {
    he::Muon impl;
    explicit he_muon_s(const he::MuonProblem& pr) : impl(pr) {}
};

extern "C" {

int he_muon_create(he_muon_t* muon, const int64_t* shapes, int count, int dtype, int precision, int steps) {
    return he::guard([&] {
        HE_REQUIRE(muon && shapes && count >= 1, HE_ERR_INVALID, "bad argument");
        HE_REQUIRE(precision == HE_PREC_F32_F32 || precision == HE_PREC_F16_F32, HE_ERR_INVALID, "muon: precision %d is neither f32_f32 nor f16_f32", precision);
        he::MuonProblem pr;
        for (int k = 0; k < count; k++) pr.shapes.push_back({shapes[2 * k], shapes[2 * k + 1]});
        pr.dtype = dtype, pr.split = precision == HE_PREC_F32_F32, pr.steps = steps;
        *muon = new he_muon_s(pr);
    });
}

int he_muon_destroy(he_muon_t muon) {
    return he::guard([&] { delete muon; });
}

int he_muon_orthogonalize(he_muon_t muon, const void* const* in, void* const* out, int count, he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(muon, HE_ERR_INVALID, "null muon");
        HE_REQUIRE(count == (int)muon->impl.count(), HE_ERR_INVALID, "muon takes %zu matrices, got %d", muon->impl.count(), count);
        muon->impl.orthogonalize(in, out, stream ? stream->s : nullptr);
    });
}

int he_muon_step(he_muon_t muon, const void* const* gradients, const float* const* momenta, const float* const* weights, float* const* new_momenta,
                 float* const* new_weights, int count, float learning_rate, float momentum, float weight_decay, int nesterov, he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(muon, HE_ERR_INVALID, "null muon");
        HE_REQUIRE(count == (int)muon->impl.count(), HE_ERR_INVALID, "muon takes %zu matrices, got %d", muon->impl.count(), count);
        const he::MuonStep how{learning_rate, momentum, weight_decay, nesterov != 0};
        muon->impl.step(gradients, momenta, weights, new_momenta, new_weights, how, stream ? stream->s : nullptr);
    });
}

const char* he_muon_source(he_muon_t muon) { return muon ? muon->impl.source().c_str() : ""; }
const char* he_muon_describe(he_muon_t muon) { return muon ? muon->impl.describe().c_str() : ""; }

int he_muon_table(he_muon_t muon, int which, void* data, size_t capacity, size_t* bytes) {
    return he::guard([&] {
        HE_REQUIRE(muon && bytes && which >= 0 && which < he::Muon::kTables && (data || capacity == 0), HE_ERR_INVALID, "bad argument");
        const std::vector<char>& t = muon->impl.table(which);
        *bytes = t.size();
        if (capacity) memcpy(data, t.data(), std::min(capacity, t.size()));
    });
}

}  // extern "C"
