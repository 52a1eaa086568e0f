#include "muon.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <functional>
#include <future>
#include <sstream>

namespace he {

namespace {

constexpr int kGroup = 32;       // matrices whose operands one launch takes by value
constexpr uint32_t kBlock = 64;  // rows and columns of one block of the conversions
// A launch has fewer than 2^32 threads. So a group has fewer than 2^24 blocks: 2^36 values, whose workspace would be more than 500 GB.
constexpr uint64_t kThreads = 1ull << 32, kMostBlocks = kThreads / 256 - 1;

// Newton-Schulz iteration on f16 matrix cores. With X scaled to a Frobenius norm of at most 1, no singular value ever leaves
// [0, 1.21]: the step's polynomial a s + b s^3 + c s^5 maps [0, 1] there and [1, 1.21] into [0.68, 0.96]. So every entry has a known
// bound, and fixed powers of two keep f16 operands in range (X_SCALE, and the scales in plan_launches()). A value's f16 rounding has 11 bits; its remainder in a second f16
// gives 22, and three of the four products of such pairs (the fourth is 2^-22 of the result) run at three times f16's cost, where f32
// matrix instructions take sixteen times. Errors are 0.7 to 1.6 times those of f32 products (1e-6 to 4e-6 of the result's norm).
//
// Several steps at once. All matrices of an iteration commute, so its steps can be taken on the m x m side: with A = X X^T and
// Q_k = a I + b A_k + c A_k A_k, A_(k+1) = Q_k A_k Q_k, and X = Q_(r-1) ... Q_0 X after r steps - one product with X on either end
// instead of two per step, for 3 m x m products (half of them by symmetry) per step between. It costs digits: an error of A, which is
// relative to the largest singular value, meets the smallest squared. After runs of three and two errors are 0.8 to 2.5 times those of f32
// products, and up to 8 times (7e-6 of the norm against 9e-7) on 20 x 60 with a few directions 35 times as strong as the rest; five at once: 1e-4.
// So steps go in runs of three at most, one by one where the caller says so (HE_OPT_MUON_SEVERAL_STEPS) and
// where operands have one part.
const char* kCommon = R"HIP(
typedef unsigned short u16;
typedef unsigned int u32;
typedef unsigned long long u64;
typedef _Float16 f16_t;
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
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
#ifndef FREXP_EXP
#define FREXP_EXP(x) __builtin_amdgcn_frexp_exp(x)
#define LDEXP_F64(x, n) __builtin_amdgcn_ldexp(x, n)
#define LDEXP_F32(x, n) __builtin_amdgcn_ldexpf(x, n)
#endif
#ifndef WAIT_LOADS
#define WAIT_LOADS(n) (0x0070 | ((n) & 15) | (((n) >> 4) << 14))   /* vmcnt(n), and lgkmcnt(0): this wave's reads of LDS are done */
#endif
struct Matrix {
    u32 rows, cols, mp, np;
    u32 tall, first_part, parts;
    float shape_scale;
    u64 at[BUFFERS];
};
enum { X, XT, XT2, A, B, C, Q, Q2, X_LOW };   // places of a matrix's buffers in `at`
struct Block { u32 matrix, i, j; };
// R = c1 E1 + c2 E2 + cs P Q^T + ci I of one matrix: operands and results by their offsets in the workspace. parked_at: of the product's
// shares, in floats. (All that a workgroup has to look up lies together, one look behind its task.)
struct Product {
    u32 mp, np;
    float c1, c2, cs, ci;
    u64 p, q, e1, e2, out, turned, low, parked_at;
};
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

// What goes over the values once, bound by memory: the norm (of a step: the momenta too), U in f16 parts and both orientations, and the
// last X to where it goes. The 22 filters of a classifier, 11.7 M values, step in f32: 29 + 34 + 28 us at 4.8, 5.6 and 5.0 TB/s.
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
    __shared__ double totals[4];
    const Block t = blocks[blockIdx.x];
    const Matrix& m = mats[t.matrix];
    const u32 k = t.matrix - o.first, rows_p = m.tall ? m.np : m.mp, cols_p = m.tall ? m.mp : m.np, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    double s = 0.0;
    for (u32 p = threadIdx.x; p < m.parts; p += 256) s += sums[m.first_part + p];
    for (int d = 32; d > 0; d /= 2) s += SHFL_XOR_F64(s, d);
    if (lane == 0) totals[wave] = s;
    __syncthreads();
    const double total = totals[0] + totals[1] + totals[2] + totals[3];
    // (the factor as a mantissa and a power of two: a norm beyond 2^126 leaves no f32 of its reciprocal)
    const double factor = (double)X_SCALE / (sqrt(total) + (double)NORM_FLOOR);
    const int power = FREXP_EXP(factor);
    const float mantissa = (float)LDEXP_F64(factor, -power);
    f16_t *natural = (f16_t*)(ws + m.at[m.tall ? XT : X]), *turned = (f16_t*)(ws + m.at[m.tall ? X : XT]), *low = (f16_t*)(ws + m.at[X_LOW]);
    const u32 c = t.j * 64 + (lane & 7u) * 8;
#pragma unroll
    for (u32 pass = 0; pass < 2; pass++) {
        const u32 i = pass * 32 + wave * 8 + (lane >> 3), r = t.i * 64 + i;
        float v[8];
        updates_of<STEP>(o, k, r, c, m.rows, m.cols, v);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = LDEXP_F32(v[e] * mantissa, power);
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
    const f16_t *from = (const f16_t*)(ws + m.at[X]), *low = SPLIT ? nullptr : (const f16_t*)(ws + m.at[X_LOW]);
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

// One text for the three kinds of products, all of the form R = c1 E1 + c2 E2 + cs P Q^T + ci I with P, Q row-major and contiguous along
// the sum (X and its transpose are both kept for that; the others are symmetric):
//   gram    A = X X^T                      m x m along n; lower tiles, stored twice
//   inner   B = b A + c A A and the like   m x m along m; lower tiles, stored twice; up to two products of a launch
//   apply   X = a X + B X or Q X           m x n along m; stored as X and as XT
// A tile of 64 to 256 rows and columns per workgroup, its operands loaded straight into a ring of LDS stages, sums in registers; where a
// group has too few tiles for the chip, their sums are cut into shares that `join` adds up in their order (no atomics: the same bits
// every time).
//
// 4096 x 4096 in one part: apply 135 us, 1.02 PFLOP/s; the matrix instructions take 46% of its cycles at 2.1 GHz. About 30 us of it
// are the epilogue, which moves 160 MB (X and its low part in, both and XT out) with one tile per CU and nothing beside it; with two smaller
// workgroups per CU, whose epilogues overlap, the sums take longer (tiles of 128: 152 us). gram 80 and inner 86 us for their lower halves,
// 253 tiles of 192. In two parts: 1024 x 4096 and its like, apply 56 us (0.92 PFLOP/s over its three products), gram 43 + 8 for
// the shares, inner 19; a classifier's 22 filters 50, 31 + 5 and 9.3 us, the last bound by its 252 workgroups' latency.
const char* kProduct = R"HIP(
#define WAVES (WAVES_M * WAVES_N)
#define WTM (TILE / WAVES_M)
#define WTN (TILE / WAVES_N)
#define MB (WTM / 32)
#define NB (WTN / 32)
#define ROW 64                          /* halves of a row in a k-tile: 128 bytes, 8 chunks */
#define KS (4 / PARTS)                  /* matrix instructions along a k-tile */
#define STAGE_HALVES (2 * TILE * ROW)
#define LOADS (2 * TILE / 8 / WAVES)    /* direct loads of a wave per k-tile: 8 rows each; an even number */
#define READS (PARTS * (MB + NB))       /* fragments of one k-step */
#define MMAS ((SPLIT ? 3 : 1) * MB * NB)
#define SM (MB % 2 ? 1 : 2)             /* a wave's strip, in blocks of 32 x 32: what goes through LDS at a time */
#define SN (NB % 2 ? 1 : 2)
#define STRIP_FLOATS(sm, sn) ((sm) * 32 * ((sn) * 32 + 1))   /* odd pitch: rows and columns are both read without bank conflicts */
#define STRIPS_HALVES (2 * WAVES * STRIP_FLOATS(SM, SN))
#define LDS_HALVES (STAGES * STAGE_HALVES > STRIPS_HALVES ? STAGES * STAGE_HALVES : STRIPS_HALVES)
#define PARKED (TILE * TILE)            /* floats of a tile that waits to be added up */
enum { GRAM, INNER, APPLY };

__device__ __forceinline__ void strip_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Where results come together and go. Looked up ahead of the sums: at their end each look would be waited for.
struct Ends { const f16_t *e1, *e2; f16_t *plain, *turned, *low; };
template <int STAGE> __device__ __forceinline__ Ends ends_of(const Product& m, char* __restrict__ ws) {
    Ends n;
    n.e1 = (const f16_t*)(ws + m.e1), n.e2 = (const f16_t*)(ws + m.e2);
    n.plain = (f16_t*)(ws + m.out), n.turned = (f16_t*)(ws + m.turned);
    // (of X the low part counts in either precision: what f16 drops of a X in each step would stay dropped, and the small
    // singular values with it)
    n.low = STAGE == APPLY && !SPLIT ? (f16_t*)(ws + m.low) : nullptr;
    return n;
}

// The results of 32 RM x 32 RN sums at (row0, col0) of the product. A lane holds rows (e / 4) * 8 + half * 4 + e % 4 of column lane % 32
// of each 32 x 32 block; through a strip of LDS that belongs to the wave it gets 8 neighbours of a row, adds E, stores them, and
// puts them back for the transposed copy.
template <int STAGE, int RM, int RN>
__device__ __forceinline__ void finish(const f32x16 (&acc)[RM][RN], const Ends& ends, const Product& m, u32 row0, u32 col0, bool mirrored, float* strip) {
    constexpr u32 strip_pitch = RN * 32 + 1, row_lanes = RN * 4, col_lanes = RM * 4;   // lanes along a row of the strip, and along a column
    const u32 lane = threadIdx.x & 63u, half = lane >> 5;
    const u32 pitch = STAGE == APPLY ? m.np : m.mp;
#pragma unroll
    for (int i = 0; i < RM; i++)
#pragma unroll
        for (int j = 0; j < RN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) strip[(i * 32 + (e / 4) * 8 + half * 4 + e % 4) * strip_pitch + j * 32 + (lane & 31u)] = acc[i][j][e];
    strip_sync();
#pragma unroll
    for (u32 s = 0; s < RM * 32 * row_lanes / 64; s++) {
        const u32 r = s * (64 / row_lanes) + lane / row_lanes, c = lane % row_lanes * 8;
        float v[8], e1[8], e2[8];
        const bool has_e1 = STAGE != GRAM && m.c1 != 0.0f, has_e2 = STAGE == INNER && m.c2 != 0.0f;
        if (has_e1) get(ends.e1, row0 + r, col0 + c, pitch, e1, ends.low);
        if (has_e2) get(ends.e2, row0 + r, col0 + c, pitch, e2, nullptr);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = m.cs * strip[r * strip_pitch + c + e];
            if (has_e1) v[e] += m.c1 * e1[e];
            if (has_e2) v[e] += m.c2 * e2[e];
            if (STAGE == INNER && row0 + r == col0 + c + e) v[e] += m.ci;
            strip[r * strip_pitch + c + e] = v[e];
        }
        put(ends.plain, row0 + r, col0 + c, pitch, v, ends.low);
    }
    strip_sync();
    if (mirrored)
#pragma unroll
        for (u32 s = 0; s < RN * 32 * col_lanes / 64; s++) {
            const u32 c = s * (64 / col_lanes) + lane / col_lanes, r = lane % col_lanes * 8;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = strip[(r + e) * strip_pitch + c];
            put(ends.turned, col0 + c, row0 + r, m.mp, v, nullptr);
        }
    strip_sync();
}

struct Fragments { f16x8 a[PARTS][MB], b[PARTS][NB]; };
struct True { constexpr operator bool() const { return true; } };
struct False { constexpr operator bool() const { return false; } };

template <int STAGE> __device__ __forceinline__ void product(const Product* __restrict__ products, u32 matrices, const Task* __restrict__ tasks, char* __restrict__ ws, float* __restrict__ parked) {
    __shared__ __attribute__((aligned(16))) f16_t lds[LDS_HALVES];
    const Task t = tasks[blockIdx.x];
    const Product m = products[(STAGE == INNER ? blockIdx.y * matrices : 0u) + t.matrix];
    if (STAGE == INNER) parked += m.parked_at;
    const Ends ends = ends_of<STAGE>(m, ws);
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave_m = wave / WAVES_N, wave_n = wave % WAVES_N;
    const u32 k_len = (STAGE == GRAM ? m.np : m.mp) * PARTS;   // halves of a row
    const u32 p_limit = m.mp, q_limit = STAGE == APPLY ? m.np : m.mp;
    const f16_t *p_rows = (const f16_t*)(ws + m.p), *q_rows = (const f16_t*)(ws + m.q);
    // Direct loads: lane l of the load of rows 8 r .. 8 r + 7 takes row l / 8 and, so that fragment reads meet different banks, the chunk
    // (l % 8) ^ (row / 2 % 8) of its 128 bytes: two rows fill the 64 banks, so rows two apart must differ. (A tile that ends beyond the
    // matrix loads its first rows there: sums that nothing stores.)
    const u32 lane_row = (lane >> 3) * k_len, lane_off[2] = {lane_row + (((lane & 7u) ^ (lane >> 4)) << 3), lane_row + (((lane & 7u) ^ (4u + (lane >> 4))) << 3)};
    auto fetch = [&](u32 kt, u32 slot) {
        f16_t* base = lds + slot * STAGE_HALVES;
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const u32 row = (wave * LOADS + l) * 8;   // of P's rows, then Q's
            const bool is_p = row < TILE;
            const u32 at = is_p ? t.i * TILE + row : t.j * TILE + row - TILE, limit = is_p ? p_limit : q_limit;
            const f16_t* src = (is_p ? p_rows : q_rows) + (u64)(at < limit ? at : 0u) * k_len + (u64)kt * ROW + lane_off[l & 1];
            __builtin_amdgcn_global_load_lds((const GLOBAL_AS u32*)src, (LDS_AS u32*)(base + row * ROW), 16, 0, 0);
        }
    };
    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
    const u32 frag_row = lane & 31u, half = lane >> 5, swz = lane >> 1 & 7u;
    Fragments f[2];
#pragma unroll
    for (int part = 0; part < PARTS; part++) {
#pragma unroll
        for (int i = 0; i < MB; i++) f[1].a[part][i] = f16x8(f16_t(0.0f));
#pragma unroll
        for (int j = 0; j < NB; j++) f[1].b[part][j] = f16x8(f16_t(0.0f));
    }
    auto read = [&](Fragments& g, const f16_t* stage, int kk) {
        const f16_t *p = stage + (wave_m * WTM + frag_row) * ROW, *q = stage + (TILE + wave_n * WTN + frag_row) * ROW;
#pragma unroll
        for (int part = 0; part < PARTS; part++) {
            const u32 chunk = (((kk * 2 + half) * PARTS + part) ^ swz) * 8;
#pragma unroll
            for (int i = 0; i < MB; i++) g.a[part][i] = *(const f16x8*)(p + i * 32 * ROW + chunk);
#pragma unroll
            for (int j = 0; j < NB; j++) g.b[part][j] = *(const f16x8*)(q + j * 32 * ROW + chunk);
        }
    };
    auto multiply = [&](const Fragments& g) {
        // high x high, high x low, low x high
#pragma unroll
        for (int c = 0; c < (SPLIT ? 3 : 1); c++)
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int j = 0; j < NB; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(g.a[c == 2][i], g.b[c == 1][j], acc[i][j], 0, 0, 0);
    };
    // One k-tile. The loop is rotated by a k-step: the matrix instructions that the last k-tile left over cover the barrier's way, the
    // first reads of this one and the loads of the one to come; each further step's reads are issued between the instructions of
    // the step before. The order is asked for, since the compiler by itself reads, waits and multiplies in turn.
    u32 slot = 0;
    auto k_tile = [&](u32 kt, auto more) {
        // this wave's loads of the k-tile have landed (those of the STAGES - 2 behind it may be on their way), then the other waves'
        if (more) __builtin_amdgcn_s_waitcnt(WAIT_LOADS((STAGES - 2) * LOADS));
        else __builtin_amdgcn_s_waitcnt(WAIT_LOADS(0));
        // (the bare barrier: __syncthreads() would wait for all loads; no wave still reads the stage that is filled next)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const f16_t* stage = lds + slot * STAGE_HALVES;
        read(f[0], stage, 0);
        if (more) fetch(kt + STAGES - 1, slot + STAGES - 1 < STAGES ? slot + STAGES - 1 : slot - 1);
        multiply(f[1]);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
        for (int n = 0; n < MMAS; n++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
            for (int l = n * LOADS / MMAS; l < (n + 1) * LOADS / MMAS; l++)
                if (more) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        }
#pragma unroll
        for (int kk = 1; kk < KS; kk++) {
            read(f[kk & 1], stage, kk);
            multiply(f[(kk & 1) ^ 1]);
#pragma unroll
            for (int n = 0; n < MMAS; n++) {
                // (reads behind the first instruction: the wait for its operands is for all reads before it)
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (n * 2 < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                if (n * 2 + 1 < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        }
        slot = slot + 1 < STAGES ? slot + 1 : 0;
    };
    const u32 k_count = t.k_end - t.k_begin, ahead = STAGES - 1 < k_count ? STAGES - 1 : k_count;
    for (u32 s = 0; s < ahead; s++) fetch(t.k_begin + s, s);
    u32 kt = t.k_begin;
    for (; kt + ahead < t.k_end; kt++) k_tile(kt, True());
    for (; kt < t.k_end; kt++) k_tile(kt, False());
    multiply(f[1]);

    // A share of a tile's sum waits in memory for the launch that adds them up, block by block of 32 x 32, as the lanes hold it.
    if (t.shares > 1) {
        f32x4* to = (f32x4*)(parked + (u64)(t.slot + t.share) * PARKED);
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    f32x4 four = {acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
                    to[((wave_m * MB + i) * (TILE / 32) + wave_n * NB + j) * 256 + e * 64 + lane] = four;
                }
        return;
    }
    __syncthreads();   // the operand stages become the waves' strips
    float* strip = (float*)lds + wave * STRIP_FLOATS(SM, SN);
#pragma unroll
    for (int i = 0; i < MB; i += SM)
#pragma unroll
        for (int j = 0; j < NB; j += SN) {
            const u32 row0 = t.i * TILE + (wave_m * MB + i) * 32, col0 = t.j * TILE + (wave_n * NB + j) * 32;
            if (row0 >= p_limit || col0 >= q_limit) continue;
            f32x16 part[SM][SN];
#pragma unroll
            for (int di = 0; di < SM; di++)
#pragma unroll
                for (int dj = 0; dj < SN; dj++) part[di][dj] = acc[i + di][j + dj];
            finish<STAGE, SM, SN>(part, ends, m, row0, col0, STAGE == APPLY ? m.turned != m.out : t.i != t.j, strip);
        }
}

// The shares of a tile added up in their order: a wave per 32 x 32 block, four waves in a workgroup. `tiles`: the first share's task of each.
template <int STAGE> __device__ __forceinline__ void join(const Product* __restrict__ products, u32 matrices, const Task* __restrict__ tiles, char* __restrict__ ws, const float* __restrict__ parked) {
    __shared__ float strips[4 * STRIP_FLOATS(1, 1)];
    constexpr u32 blocks = (TILE / 32) * (TILE / 32);
    const Task t = tiles[blockIdx.x / (blocks / 4)];
    const Product m = products[(STAGE == INNER ? blockIdx.y * matrices : 0u) + t.matrix];
    if (STAGE == INNER) parked += m.parked_at;
    const Ends ends = ends_of<STAGE>(m, ws);
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block = blockIdx.x % (blocks / 4) * 4 + wave;
    const u32 row0 = t.i * TILE + block / (TILE / 32) * 32, col0 = t.j * TILE + block % (TILE / 32) * 32;
    if (row0 >= m.mp || col0 >= (STAGE == APPLY ? m.np : m.mp)) return;
    const f32x4* from = (const f32x4*)(parked + (u64)t.slot * PARKED) + block * 256 + lane;
    f32x16 sum[1][1];
#pragma unroll
    for (int e = 0; e < 16; e++) sum[0][0][e] = 0.0f;
    for (u32 s = 0; s < t.shares; s += 4) {
        f32x4 got[4][4];
#pragma unroll
        for (u32 d = 0; d < 4; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                got[d][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (s + d < t.shares) got[d][e] = from[(u64)(s + d) * (PARKED / 4) + e * 64];
            }
#pragma unroll
        for (u32 d = 0; d < 4; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) sum[0][0][e] += got[d][e / 4][e % 4];
    }
    finish<STAGE, 1, 1>(sum, ends, m, row0, col0, STAGE == APPLY ? m.turned != m.out : t.i != t.j, strips + wave * STRIP_FLOATS(1, 1));
}

#define KERNELS(name, stage) \
    extern "C" __global__ __launch_bounds__(WAVES * 64) KERNEL_ATTRS void muon_##name(const Product* __restrict__ products, u32 matrices, const Task* __restrict__ tasks, char* __restrict__ ws, float* __restrict__ parked) { product<stage>(products, matrices, tasks, ws, parked); } \
    extern "C" __global__ __launch_bounds__(256) void muon_join_##name(const Product* __restrict__ products, u32 matrices, const Task* __restrict__ tiles, char* __restrict__ ws, const float* __restrict__ parked) { join<stage>(products, matrices, tiles, ws, parked); }
)HIP";

constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;
enum { X, XT, XT2, A, B, C, Q, Q2, X_LOW };

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

// Tasks in the order of their blocks. The longest sums begin first, so that the chip empties evenly. Of each length, the 8 XCDs, to
// which blocks are dealt in turn and each of which has an L2 of its own, get an eighth of a sequence in which neighbours share rows
// and columns.
void deal(std::vector<MuonTask>& tasks) {
    auto length = [](const MuonTask& t) { return t.k_end - t.k_begin; };
    std::stable_sort(tasks.begin(), tasks.end(), [&](const MuonTask& a, const MuonTask& b) { return length(a) > length(b); });
    std::vector<MuonTask> queue[8];
    size_t turn = 0;  // who gets one more where a length's tasks do not divide by 8
    for (size_t begin = 0, end; begin < tasks.size(); begin = end) {
        for (end = begin; end < tasks.size() && length(tasks[end]) == length(tasks[begin]);) end++;
        const size_t n = end - begin;
        size_t at = begin;
        for (size_t x = 0; x < 8; x++) {
            const size_t count = n / 8 + ((x + 8 - turn) % 8 < n % 8);
            queue[x].insert(queue[x].end(), tasks.begin() + at, tasks.begin() + at + count);
            at += count;
        }
        turn = (turn + n) % 8;
    }
    // (whoever has the extra tasks comes first in every round of 8)
    size_t b = 0;
    for (size_t round = 0; b < tasks.size(); round++)
        for (size_t x = 0; x < 8; x++)
            if (round < queue[x].size()) tasks[b++] = queue[x][round];
}

// How a product's tiles are made: the waves of a workgroup, its ring of k-tiles in LDS, and the workgroups that a CU holds. And what
// the choice between them goes by, microseconds measured on products of 64 to 4096 rows: a task's `base`, and what a k-tile takes
// in a workgroup that has a CU to itself (`alone`) and on a full chip, for operands of one part and of two. Against every other tile
// forced upon one kind of product, the choice is within 2% of the best on 4096 x 4096, 1024 x 4096 pairs, a classifier's filters and odd
// extents; with the worst a whole call takes 1.1 to 1.7 times as long.
struct TileShape {
    uint32_t tile, waves_m, waves_n, stages, per_cu;
    const char* attrs;
    double base, alone[2], full[2];
    uint32_t threads() const { return waves_m * waves_n * 64; }
};
const TileShape kTiles[] = {
    {64, 2, 2, 4, 2, "", 2.5, {0.22, 0.28}, {0.42, 0.50}},
    {128, 2, 2, 2, 2, "__attribute__((amdgpu_waves_per_eu(2, 2)))", 3.5, {0.65, 0.85}, {1.17, 1.65}},
    {192, 2, 2, 3, 1, "__attribute__((amdgpu_waves_per_eu(1, 1)))", 5.0, {0.70, 0.85}, {1.13, 2.00}},
    {256, 2, 4, 2, 1, "__attribute__((amdgpu_waves_per_eu(2, 2)))", 6.0, {1.25, 2.00}, {1.80, 2.85}},
};
constexpr uint32_t kCUs = 256;

// How one product of every matrix is cut into tasks: tiles, and where there are too few of them to fill the chip or their sums are
// long, shares of `target` k-tiles or a little more of each sum, which a second launch adds up.
struct Tiles {
    uint32_t ti, tj, kt, shares;  // tile rows and columns, k-tiles of a sum and how many tasks share it
    Tiles(const MuonMatrix& m, uint32_t tile, bool lower, bool along_n, int parts, uint32_t target) {
        ti = (m.mp + tile - 1) / tile, tj = lower ? ti : (m.np + tile - 1) / tile;
        kt = (along_n ? m.np : m.mp) / (64 / parts), shares = std::max(1u, kt / target);
    }
};
// What a cut comes to, from counts alone: a large group has candidates of a thousand million tasks.
struct CutSize {
    uint64_t tasks = 0, parked = 0;  // parked: shares that wait in memory
    double estimate = 0;             // microseconds
};
CutSize size_cut(const std::vector<MuonMatrix>& mats, const TileShape& shape, bool lower, bool along_n, int parts, uint32_t target) {
    CutSize size;
    std::map<uint32_t, uint64_t, std::greater<uint32_t>> lengths;  // how many tasks have so many k-tiles, the longest first
    for (const MuonMatrix& m : mats) {
        const Tiles t(m, shape.tile, lower, along_n, parts, target);
        const uint64_t tiles = lower ? (uint64_t)t.ti * (t.ti + 1) / 2 : (uint64_t)t.ti * t.tj, longer = t.kt % t.shares;
        size.tasks += tiles * t.shares;
        if (t.shares > 1) size.parked += tiles * t.shares;
        if (longer) lengths[t.kt / t.shares + 1] += tiles * longer;
        lengths[t.kt / t.shares] += tiles * (t.shares - longer);
    }
    // Every task goes to the workgroup place that is free first; a k-tile takes the longer the fuller the chip is. `free_at`: how many
    // places are free from when on. Places that become free within one task's time of each other take turns, a task each.
    const uint64_t slots = (uint64_t)kCUs * shape.per_cu;
    const double f = std::min(1.0, (double)size.tasks / slots), each = shape.alone[parts - 1] + (shape.full[parts - 1] - shape.alone[parts - 1]) * f * f;
    std::map<double, uint64_t> free_at{{0.0, slots}};
    for (auto [length, count] : lengths) {
        const double time = shape.base + each * length;
        while (count) {
            const auto first = free_at.begin();
            if (count >= slots && free_at.rbegin()->first - first->first <= time) {
                const uint64_t rounds = count / slots;
                std::map<double, uint64_t> later;
                for (auto& [at, places] : free_at) later[at + rounds * time] += places;
                free_at = std::move(later);
                count -= rounds * slots;
                continue;
            }
            const uint64_t taken = std::min(count, first->second);
            free_at[first->first + time] += taken;
            if (taken == first->second) free_at.erase(first);
            else first->second -= taken;
            count -= taken;
        }
    }
    size.estimate = free_at.rbegin()->first;
    // (a launch, and the shares read at about 5 TB/s)
    if (size.parked) size.estimate += 2.5 + 4.0 * size.parked * shape.tile * shape.tile / 5e6;
    return size;
}
struct Cut {
    std::vector<MuonTask> tasks, joins;  // joins: a task of each tile that is shared
};
Cut cut_product(const std::vector<MuonMatrix>& mats, const TileShape& shape, bool lower, bool along_n, int parts, uint32_t target) {
    Cut cut;
    uint32_t parked = 0;
    for (size_t k = 0; k < mats.size(); k++) {
        const Tiles t(mats[k], shape.tile, lower, along_n, parts, target);
        for (uint32_t g = 0; g < t.ti; g += 4)  // bands of four tile rows, column by column
            for (uint32_t j = 0; j < t.tj; j++)
                for (uint32_t i = g; i < std::min(g + 4, t.ti); i++) {
                    if (lower && j > i) continue;
                    for (uint32_t s = 0; s < t.shares; s++)
                        cut.tasks.push_back({(uint32_t)k, i, j, (uint32_t)((uint64_t)t.kt * s / t.shares), (uint32_t)((uint64_t)t.kt * (s + 1) / t.shares), parked, s, t.shares});
                    if (t.shares > 1) {
                        cut.joins.push_back(cut.tasks.back());
                        parked += t.shares;
                    }
                }
    }
    deal(cut.tasks);
    return cut;
}
template <class T> std::vector<char> bytes_of(const std::vector<T>& v) {
    std::vector<char> out(v.size() * sizeof(T));
    if (!v.empty()) memcpy(out.data(), v.data(), out.size());
    return out;
}

std::atomic<bool> g_several_steps{true};

}  // namespace

void set_muon_several_steps(bool may) { g_several_steps = may; }

Muon::Muon(const MuonProblem& pr) : pr_(pr) {
    HE_REQUIRE(!pr.shapes.empty() && pr.shapes.size() <= 65536, HE_ERR_INVALID, "muon: %zu matrices, 1 to 65536 are taken", pr.shapes.size());
    HE_REQUIRE(pr.dtype == HE_F16 || pr.dtype == HE_BF16 || pr.dtype == HE_F32, HE_ERR_INVALID, "muon does not take dtype %s", dtype_name(pr.dtype));
    HE_REQUIRE(pr.steps >= 1 && pr.steps <= 32, HE_ERR_INVALID, "muon: %d steps, 1 to 32 are taken", pr.steps);
    uint64_t at = 0, parts = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    // Shares of the sums of squares: about a thousand, so that they fill the chip and a matrix has few of them to add up.
    uint64_t values = 0;
    for (auto& s : pr.shapes) values += (uint64_t)std::max<int64_t>(s[0], 0) * std::max<int64_t>(s[1], 0);
    uint64_t part = 2048;
    while (part < 65536 && part * 1024 < values) part *= 2;
    std::vector<MuonBlock> portions, blocks;
    for (size_t k = 0; k < pr.shapes.size(); k++) {
        const int64_t rows = pr.shapes[k][0], cols = pr.shapes[k][1];
        HE_REQUIRE(rows >= 1 && cols >= 1, HE_ERR_INVALID, "muon: matrix %zu is %lld x %lld", k, (long long)rows, (long long)cols);
        HE_REQUIRE(std::max(rows, cols) <= (1 << 20) && std::min(rows, cols) <= 32768, HE_ERR_UNSUPPORTED,
                   "muon: matrix %zu is %lld x %lld; extents up to 2^20 by 32768 are taken", k, (long long)rows, (long long)cols);
        MuonMatrix m{};
        m.rows = (uint32_t)rows, m.cols = (uint32_t)cols, m.tall = rows > cols;
        auto padded = [&](int64_t v) { return (uint32_t)((v + kBlock - 1) / kBlock * kBlock); };
        m.mp = padded(std::min(rows, cols)), m.np = padded(std::max(rows, cols));
        m.shape_scale = (float)std::sqrt(std::max(1.0, (double)rows / (double)cols));
        const uint64_t size = (uint64_t)rows * cols;
        m.first_part = (uint32_t)parts;
        m.parts = (uint32_t)((size + part - 1) / part);
        parts += m.parts;
        part_begin_.push_back((uint32_t)portions.size());
        block_begin_.push_back((uint32_t)blocks.size());
        HE_REQUIRE(blocks.size() + (uint64_t)(m.mp / kBlock) * (m.np / kBlock) <= kMostBlocks, HE_ERR_UNSUPPORTED, "muon: too many elements for one group");
        for (uint32_t p = 0; p < m.parts; p++) portions.push_back({(uint32_t)k, p, 0});
        const uint32_t br = (m.tall ? m.np : m.mp) / kBlock, bc = (m.tall ? m.mp : m.np) / kBlock;
        for (uint32_t i = 0; i < br; i++)
            for (uint32_t j = 0; j < bc; j++) blocks.push_back({(uint32_t)k, i, j});
        matrices_.push_back(m);
    }
    part_begin_.push_back((uint32_t)portions.size());
    block_begin_.push_back((uint32_t)blocks.size());
    // the kinds of products: A = X X^T along n, those of m x m matrices along m, and X from B X along m
    const char* names[3] = {"gram", "inner", "apply"};
    uint32_t most = 0;
    std::string cuts;
    for (int p = 0; p < 3; p++) {
        ProductKind& product = products_[p];
        const int forced = tuning::get_int("HELIUM_HIP_MUON_TILE", -1), only = forced >= 0 ? forced : tuning::get_int((std::string("HELIUM_HIP_MUON_TILE_") + names[p]).c_str(), -1);
        const TileShape* chosen = nullptr;
        CutSize size;
        uint32_t chosen_target = 0;
        for (const TileShape& candidate : kTiles)
            for (uint32_t target : {1u << 30, 64u, 32u, 16u, 8u, 4u}) {
                if (only >= 0 && candidate.tile != (uint32_t)only) continue;
                const CutSize c = size_cut(matrices_, candidate, p < 2, p == 0, pr.split ? 2 : 1, target);
                // (4 GB of shares are the most that is made; tiles of 64 that nobody shares are no more than the blocks, so one candidate is always left)
                if (c.tasks * candidate.threads() >= kThreads || c.parked * candidate.tile * candidate.tile >= (1u << 30) || (chosen && c.estimate >= size.estimate)) continue;
                size = c;
                chosen = &candidate;
                chosen_target = target;
            }
        HE_REQUIRE(chosen, HE_ERR_INVALID, "muon: there are no tiles of %d", only);
        const TileShape& shape = *chosen;
        const Cut cut = cut_product(matrices_, shape, p < 2, p == 0, pr.split ? 2 : 1, chosen_target);
        const std::vector<MuonTask>&tasks = cut.tasks, &joins = cut.joins;
        const uint32_t parked = (uint32_t)size.parked;
        tables_[1 + p] = bytes_of(tasks), tables_[4 + p] = bytes_of(joins);
        product.threads = shape.threads();
        product.grid = (uint32_t)tasks.size();
        product.join_grid = (uint32_t)joins.size() * (shape.tile / 32) * (shape.tile / 32) / 4;
        product.text = strfmt("#define TILE %u\n#define WAVES_M %u\n#define WAVES_N %u\n#define STAGES %u\n#ifndef KERNEL_ATTRS\n#define KERNEL_ATTRS %s\n#endif\n", shape.tile,
                              shape.waves_m, shape.waves_n, shape.stages, shape.attrs);
        product.parked = parked * shape.tile * shape.tile;
        product.estimate = size.estimate;
        most = std::max(most, product.parked * (p == 1 ? 2 : 1));
        cuts += strfmt("\nmuon_%s tile=%u threads=%u stages=%u grid=%u join_grid=%u parked=%u estimate=%.1f", names[p], shape.tile, product.threads, shape.stages, product.grid,
                       product.join_grid, parked * shape.tile * shape.tile, size.estimate);
    }
    // What the launches read and write, and no more: X's transpose a second time if there is a run after the first, C and the Q's if a
    // run has several steps.
    const std::vector<int> runs = choose_runs();
    const bool several = *std::max_element(runs.begin(), runs.end()) > 1;
    for (MuonMatrix& m : matrices_) {
        const uint64_t bytes = pr.split ? 4 : 2, x = m.mp * bytes * m.np, a = m.mp * bytes * m.mp;
        for (int k : {X, XT, A, B}) m.at[k] = take(k == X || k == XT ? x : a);
        if (runs.size() > 1) m.at[XT2] = take(x);
        if (several)
            for (int k : {C, Q, Q2}) m.at[k] = take(a);
        if (!pr.split) m.at[X_LOW] = take(x);
    }
    shared_at_ = take((uint64_t)most * 4);
    plan_launches(runs);
    // (a share's place among the sums is its block's, plus where its launch begins)
    for (size_t k = 0; k < pr.shapes.size(); k++)
        for (uint32_t p = part_begin_[k]; p < part_begin_[k + 1]; p++) portions[p].j = part_begin_[k / kGroup * kGroup];
    workspace_bytes_ = take(parts * sizeof(double)) + parts * sizeof(double);
    tables_[0] = bytes_of(matrices_), tables_[7] = bytes_of(portions), tables_[8] = bytes_of(blocks);
    shares_ = (uint32_t)portions.size();
    for (int t = 0; t < kTables; t++) {
        table_at_[t] = table_bytes_;
        table_bytes_ += (tables_[t].size() + 255) / 256 * 256;
    }
    std::ostringstream s;
    s << "#define GROUP " << kGroup << "\n#define PART " << part << "ull\n#define BUFFERS " << MuonMatrix::kBuffers << "\n#define SPLIT " << (int)pr.split << "\n#define BF16 "
      << (pr.dtype == HE_BF16) << "\n#define F16 " << (pr.dtype == HE_F16) << "\n#define NORM_FLOOR 1e-7\n#ifndef SHFL_XOR_F64\n#define SHFL_XOR_F64(v, m) __shfl_xor(v, m, 64)\n#endif\n";
    const std::string head = s.str() + kCommon;
    std::vector<std::pair<std::unique_ptr<JitKernel>*, std::pair<std::string, std::string>>> kernels;  // where to, text, entry
    const std::string elements = head + kElements;
    for (auto& k : {std::make_pair(&norm_, "muon_norm"), std::make_pair(&convert_, "muon_convert"), std::make_pair(&finish_, "muon_finish"), std::make_pair(&norm_step_, "muon_norm_step"),
                    std::make_pair(&convert_step_, "muon_convert_step"), std::make_pair(&finish_step_, "muon_finish_step")})
        kernels.push_back({k.first, {elements, k.second}});
    source_ = elements;
    for (int p = 0; p < 3; p++) {
        const std::string name = names[p];
        ProductKind& product = products_[p];
        product.text = head + product.text + kProduct + "KERNELS(" + name + ", " + (p == 0 ? "GRAM" : p == 1 ? "INNER" : "APPLY") + ")\n";
        source_ += "\n//// product " + name + "\n" + product.text;
        kernels.push_back({&product.kernel, {product.text, "muon_" + name}});
        if (product.join_grid) kernels.push_back({&product.join, {product.text, "muon_join_" + name}});
    }
    // (each text is compiled once, all of them side by side)
    std::map<std::string, std::future<void>> compiled;
    for (auto& k : kernels) {
        const std::string& text = k.second.first;
        if (!compiled.count(text)) compiled[text] = std::async(std::launch::async, [&text] { (void)rtc_compile(text, "muon", {}); });
    }
    for (auto& c : compiled) c.second.get();
    for (auto& k : kernels) k.first->reset(new JitKernel(k.second.first, k.second.second));
    describe_ = strfmt("muon matrices=%zu steps=%d parts=%d shares=%u blocks=%zu shared_at=%zu workspace=%zu", pr.shapes.size(), pr.steps, pr.split ? 2 : 1, shares_,
                       blocks.size(), shared_at_, workspace_bytes_) + cuts + launches_text_;
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
    for (int t = 0; t < kTables && e == hipSuccess; t++) e = hipMemcpy(b.tables + table_at_[t], tables_[t].data(), tables_[t].size(), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        (void)hipFree(b.tables);
        (void)hipFree(b.workspace);
        fail(HE_ERR_HIP, strfmt("muon: %zu bytes of workspace: %s", workspace_bytes_, hipGetErrorString(e)));
    }
    per_stream_[stream] = b;
    return b;
}

// How many steps at a time are taken on the m x m side.
std::vector<int> Muon::choose_runs() const {
    std::vector<int> runs(pr_.steps, 1);
    // Runs of three at most and as even as can be, the longest first, if that is estimated to save a tenth: always where n is well beyond
    // m, never where they are equal (a classifier's 22 filters, mostly 1 to 9: 569 -> 379 us; 1000 x 512 and 777 x 1203: 221 -> 245).
    if (pr_.split && g_several_steps.load() && !tuning::get_int("HELIUM_HIP_MUON_ONE_BY_ONE", 0)) {
        const int count = (pr_.steps + 2) / 3;
        std::vector<int> longer(count, pr_.steps / count);
        for (int k = 0; k < pr_.steps % count; k++) longer[k]++;
        auto cost = [&](const std::vector<int>& of) {
            double total = 0;
            for (int r : of) total += products_[0].estimate + products_[2].estimate + products_[1].estimate * (r == 1 ? 1 : r == 2 ? 5 : 9);
            return total;
        };
        if (cost(longer) < 0.9 * cost(runs) || tuning::get_int("HELIUM_HIP_MUON_RUNS", 0)) runs = longer;
    }
    return runs;
}

// What is launched between the conversions: runs of steps, each of them on the m x m side but for its ends.
void Muon::plan_launches(const std::vector<int>& runs) {
    // scales of what is in the buffers: of X, of A, B and C, and of Q after so many steps (its values are at most a, a^2, a^3)
    const double sx = 4096, sa = 8192, sq[4] = {0, 8192, 4096, 1024};
    // (what a launch computes lies in a table on the device: a kernel's own parameters come from host memory, and longer ones took
    // the 20 small launches of a 64 x 576 matrix 79 -> 96 us)
    std::vector<MuonProduct> table;
    struct Formula {
        uint32_t p, q, out, e1, e2, turned;  // places in MuonMatrix::at
        double c1, c2, cs, ci;
    };
    auto add = [&](int kind, const std::vector<Formula>& products) {
        launches_.push_back({kind, (uint32_t)products.size(), table.size() * sizeof(MuonProduct)});
        const char* names[3] = {"gram", "inner", "apply"};
        for (size_t k = 0; k < products.size(); k++) {
            const Formula& f = products[k];
            for (const MuonMatrix& m : matrices_)
                table.push_back({m.mp, m.np, (float)f.c1, (float)f.c2, (float)f.cs, (float)f.ci, m.at[f.p], m.at[f.q], m.at[f.e1], m.at[f.e2], m.at[f.out], m.at[f.turned],
                                 m.at[X_LOW], k * products_[kind].parked});
            launches_text_ += strfmt("\nlaunch %s of=%zu c1=%.9g c2=%.9g cs=%.9g ci=%.9g", names[kind], k, f.c1, f.c2, f.cs, f.ci);
        }
    };
    // (a result that is not stored transposed as well, or in its own place as symmetric ones are, is given its own place)
    auto product = [](uint32_t p, uint32_t q, uint32_t out, uint32_t e1, double c1, double cs, uint32_t e2 = X, double c2 = 0, double ci = 0, uint32_t turned = X) {
        return Formula{p, q, out, e1, e2, turned == X ? out : turned, c1, c2, cs, ci};
    };
    launches_text_ = "\nruns";
    for (size_t k = 0; k < runs.size(); k++) launches_text_ += strfmt("%c%d", k ? ',' : ' ', runs[k]);
    uint32_t from = XT, to = XT2;
    size_t done = 0;
    for (int r : runs) {
        add(0, {product(X, X, A, 0, 0, sa / (sx * sx))});
        uint32_t q = Q, q_new = Q2;  // of two steps and more; after the first one Q is a I + B, and B is in q
        std::vector<Formula> also;  // (waits for a launch to share)
        for (int j = 0; j < r; j++) {
            const uint32_t b = r > 1 && j == 0 ? q : (uint32_t)B;
            add(1, {product(A, A, b, A, kB, kC * sa / (sa * sa))});
            if (j > 0) {
                // Q = (a I + B) Q
                if (j == 1) also = {product(b, q, q_new, q, kA * sq[2] / sa, sq[2] / (sa * sa), b, kA * sq[2] / sa, kA * kA * sq[2])};
                else also = {product(b, q, q_new, q, kA * sq[j + 1] / sq[j], sq[j + 1] / (sa * sq[j]))};
                std::swap(q, q_new);
            }
            if (j + 1 < r) {
                also.insert(also.begin(), product(b, A, C, A, kA, sa / (sa * sa)));  // C = (a I + B) A
                add(1, also);
                also.clear();
                add(1, {product(C, b, A, C, kA, sa / (sa * sa))});  // A = C (a I + B)
            }
        }
        if (!also.empty()) add(1, also);
        done += r;
        const bool last = done == (size_t)pr_.steps;
        if (r == 1) add(2, {product(B, from, X, X, kA, 1 / sa, 0, 0, 0, last ? (uint32_t)X : to)});
        else add(2, {product(q, from, X, X, 0, 1 / sq[r], 0, 0, 0, last ? (uint32_t)X : to)});
        std::swap(from, to);
    }
    tables_[9] = bytes_of(table);
}

void Muon::products(char* ws, char* tables, hipStream_t stream) {
    const uint32_t join_block[3] = {256, 1, 1};
    char* parked = ws + shared_at_;
    uint32_t matrices = (uint32_t)matrices_.size();
    for (const Launch& l : launches_) {
        const ProductKind& kind = products_[l.kind];
        char *tasks = tables + table_at_[1 + l.kind], *joins = tables + table_at_[4 + l.kind];
        const uint32_t grid[3] = {kind.grid, l.count, 1}, block[3] = {kind.threads, 1, 1}, join_grid[3] = {kind.join_grid, l.count, 1};
        char* what = tables + table_at_[9] + l.products_at;
        void* args[] = {&what, &matrices, &tasks, &ws, &parked};
        kind.kernel->launch(grid, block, 0, stream, args);
        void* join_args[] = {&what, &matrices, &joins, &ws, &parked};
        if (kind.join_grid) kind.join->launch(join_grid, join_block, 0, stream, join_args);
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
    double* sums = (double*)(ws + workspace_bytes_ - shares_ * sizeof(double));
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
        char* parts = b.tables + table_at_[7] + part_begin_[first] * sizeof(MuonBlock);
        const uint32_t grid[3] = {part_begin_[last] - part_begin_[first], 1, 1};
        void* args[] = {&mats, &parts, &sums, &o};
        (how ? norm_step_ : norm_)->launch(grid, block, 0, stream, args);
    });
    each_group([&](OperandsArg& o, size_t first, size_t last) {
        char* blocks = b.tables + table_at_[8] + block_begin_[first] * sizeof(MuonBlock);
        const uint32_t grid[3] = {block_begin_[last] - block_begin_[first], 1, 1};
        void* args[] = {&mats, &blocks, &sums, &ws, &o};
        (how ? convert_step_ : convert_)->launch(grid, block, 0, stream, args);
    });
    products(ws, b.tables, stream);
    each_group([&](OperandsArg& o, size_t first, size_t last) {
        char* blocks = b.tables + table_at_[8] + block_begin_[first] * sizeof(MuonBlock);
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
        pr.dtype = dtype, pr.steps = steps;
        // (f16 matrices are worked on in two parts at any precision: their results have 11 bits, of which five steps with operands of 11
        // bits leave eight: 2.3e-3 of the norm off, where the result's rounding is 2e-4)
        pr.split = precision == HE_PREC_F32_F32 || dtype == HE_F16;
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
