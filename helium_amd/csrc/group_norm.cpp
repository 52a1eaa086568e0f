#include "group_norm.h"

#include <algorithm>
#include <cmath>
#include <future>
#include <numeric>
#include <sstream>

namespace he {

namespace {

// ---- device text ---------------------------------------------------------------------------------------------------
// One text for all kernels of a plan; the definitions ahead of it hold the shape and the tiling:
//   PIXELS, C, G, D (channels per group), V, T (threads), KG (groups per slice), SC (channels per slice), SLICES, CV (vectors
//   of a slice's pixel), TX, TY, NC (columns per thread), RPT, ROWS, CHUNKS, BF16 / F16 / F32, PARAM_SAME, ACT, EPS
const char* kCommon = R"HIP(
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
#if PARAM_SAME
typedef elem_t param_t;
#else
typedef float param_t;
#endif
#if V == 1
typedef elem_t vec_t;
#define AT(v, i) (v)
#else
typedef elem_t vec_t __attribute__((ext_vector_type(V)));
#define AT(v, i) (v)[i]
#endif
#ifndef HE_FAST_RCP
#define HE_FAST_RCP(x) __builtin_amdgcn_rcpf(x)
#endif
#ifndef HE_EXP2
#define HE_EXP2(x) __builtin_amdgcn_exp2f(x)
#endif

// A vector whose channels all lie in one group adds up to one number, one that spans groups to one per channel.
#define ACC ((D % V) == 0 ? 1 : V)
// Where the threads of a wave that share a column can meet by shuffles, a wave leaves one row of sums in LDS, otherwise each
// row of threads does.
#define BY_SHUFFLE(n) ((TX & (TX - 1)) == 0 && TX < 64)
#define RED_ROWS (BY_SHUFFLE(0) ? T / 64 : TY)

struct Place {
    u32 tx, ty, slice, chunk;
    int left;   // pixels of the workgroup from the thread's first one on (its own are every TY-th)
    u64 n;
};
__device__ __forceinline__ Place place() {
    Place p;
    p.tx = threadIdx.x % TX;
    p.ty = threadIdx.x / TX;
    // Blocks are dealt round-robin to the 8 XCDs, each with an L2 of its own: an XCD takes neighbours, whose slices share cache lines.
    const u32 xcd = blockIdx.x % 8u;
    u64 b = xcd * (BLOCKS / 8u) + (xcd < BLOCKS % 8u ? xcd : BLOCKS % 8u) + blockIdx.x / 8u;
    p.slice = (u32)(b % SLICES);
    b /= SLICES;
    p.chunk = (u32)(b % CHUNKS);
    p.n = b / CHUNKS;
    const u64 pixels = PIXELS - (u64)p.chunk * ROWS;
    p.left = p.ty < TY ? (int)(pixels < ROWS ? pixels : ROWS) - (int)p.ty : 0;
    return p;
}
// Element offset of the workgroup's first channel of the thread's first pixel.
__device__ __forceinline__ u64 origin(const Place& p) {
    return (p.n * PIXELS + (u64)p.chunk * ROWS + p.ty) * C + (u64)p.slice * SC + p.tx * V;
}
#define COLUMN(p, q) (CV % TX == 0 || (p).tx + (q) * TX < CV)
// (what holds for every thread is not asked of each)
#define HELD(p, r, q) ((WHOLE && ((r) + 1) * TY <= PIXELS ? TX * TY == T || (p).ty < TY : (r) * TY < (p).left) && COLUMN(p, q))

__device__ __forceinline__ void load_held(const elem_t* __restrict__ x, const Place& p, vec_t (&held)[RPT][NC]) {
    const u64 o = origin(p);
#pragma unroll
    for (int r = 0; r < RPT; r++)
#pragma unroll
        for (int q = 0; q < NC; q++) {
            held[r][q] = vec_t(elem_t(0.0f));
            if (HELD(p, r, q)) held[r][q] = *(const vec_t*)(x + o + (u64)r * TY * C + q * TX * V);
        }
}

// Adds up every thread's sums (N per column) over the workgroup's pixels: entry e of the slice's CV * N ends up in red[e] of the
// first row. The order is fixed.
template <int N> __device__ __forceinline__ void fold_rows(float (&a)[NC][N], const Place& p, float* red) {
    if (BY_SHUFFLE(0)) {
#pragma unroll
        for (int q = 0; q < NC; q++)
#pragma unroll
            for (int i = 0; i < N; i++)
                for (int m = TX; m < 64; m *= 2) a[q][i] += __shfl_xor(a[q][i], m, 64);
        if ((threadIdx.x & 63u) < TX)
#pragma unroll
            for (int q = 0; q < NC; q++)
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (COLUMN(p, q)) red[((threadIdx.x >> 6) * CV + p.tx + q * TX) * N + i] = a[q][i];
    } else if (p.ty < TY) {
#pragma unroll
        for (int q = 0; q < NC; q++)
#pragma unroll
            for (int i = 0; i < N; i++)
                if (COLUMN(p, q)) red[(p.ty * CV + p.tx + q * TX) * N + i] = a[q][i];
    }
    __syncthreads();
}
// The sums of fold_rows() per entry, out[e] for all E entries of a row: LANES neighbouring threads add one up. Where there is one row
// it is the sums already, and `out` is `red`: a pixel of 16384 channels leaves 128 KB of them, and a workgroup has 160 KB of LDS.
#define ONE_ROW (RED_ROWS == 1)
#define SUMS_APART (ONE_ROW ? 1 : SC * 2)
template <int E, int LANES> __device__ __forceinline__ void fold_entries(const float* red, float* out) {
    if (ONE_ROW) return;
    const u32 l = threadIdx.x % LANES;
    for (u32 e0 = 0; e0 < E; e0 += T / LANES) {
        const u32 e = e0 + threadIdx.x / LANES;
        float s = 0.0f;
        if (e < E)
            for (u32 row = l; row < RED_ROWS; row += LANES) s += red[row * E + e];
        for (int m = LANES / 2; m > 0; m /= 2) s += __shfl_xor(s, m, 64);
        if (e < E && l == 0) out[e] = s;
    }
    __syncthreads();
}
// The sums of fold_rows() per group: out[g], g < KG. Each group is added up by LPG neighbouring threads.
__device__ __forceinline__ void fold_groups(const float* red, float* out) {
    const u32 g = threadIdx.x / LPG, l = threadIdx.x % LPG;
    float s = 0.0f;
    const u32 per = (D / V) * V == D ? D / V : D;   // entries of a group in one row
    if (g < KG)
        for (u32 e = l; e < RED_ROWS * per; e += LPG) s += red[(e / per) * (CV * ACC) + g * per + e % per];
    for (int m = LPG / 2; m > 0; m /= 2) s += __shfl_xor(s, m, 64);
    if (g < KG && l == 0) out[g] = s;
    __syncthreads();
}
__device__ __forceinline__ u32 group_of(u32 channel) { return channel / D; }   // within the slice

// 1 / (1 + exp(-z)); z2 is -z log2(e)
#define SIGMOID(z2) HE_FAST_RCP(1.0f + HE_EXP2(z2))
#define NEG_LOG2E -1.44269504f
__device__ __forceinline__ float activate(float z) {
#if ACT == 1
    return z > 0.0f ? z : (z != z ? z : 0.0f);
#elif ACT == 2
    return z * SIGMOID(z * NEG_LOG2E);
#else
    return z;
#endif
}
// dz from dy: the activation's slope at z
__device__ __forceinline__ float slope_times(float dy, float z) {
#if ACT == 1
    return z > 0.0f ? dy : (z != z ? z : 0.0f);
#elif ACT == 2
    const float s = SIGMOID(z * NEG_LOG2E);
    return dy * (s + s * (z - z * s));
#else
    return dy;
#endif
}
#if STREAM
#define STORE(p, v) __builtin_nontemporal_store(v, p)
#else
#define STORE(p, v) (*(p) = (v))
#endif
)HIP";

// Statistics. A workgroup holds its part of a sample in registers, takes the mean of each group in it, then the sum of squared
// distances from that mean (not E[x^2] - E[x]^2, which loses all digits of a variance that is small beside the mean). Where a
// workgroup holds all pixels of its groups (WHOLE), it goes on and the tensor is read once. Otherwise the parts of a group are joined,
// M2 = sum of M2_i + n_i (mean_i - mean)^2 (by `apply` itself, or by `merge` where they are more than 32), and the tensor is read again.
// Sums are f32: a thread its own values, then trees.
//
// Bound by memory. WHOLE, 64 x 3136 x 256 bf16 in 32 groups: 47 us for one read and one write, 5.1 TB/s of what crosses the L2s' far
// side: in 105 MB, out 139 MB for 103 MB of results (a workgroup's 64 bytes of a pixel are half a cache line). In parts 52 us. In parts, 2 x 262144 x 128 bf16: statistics 22 us (6.1
// TB/s), merge 5, apply 41 (6.5 TB/s). 1 x 49 x 512: one launch of 3.7 us.
const char* kForward = R"HIP(
// mean[g] and m2[g] of the workgroup's pixels
__device__ __forceinline__ void part_statistics(const vec_t (&held)[RPT][NC], const Place& p, float count, float* red, float* mean_of, float* m2_of) {
    float a[NC][ACC];
#pragma unroll
    for (int q = 0; q < NC; q++)
#pragma unroll
        for (int i = 0; i < ACC; i++) a[q][i] = 0.0f;
#pragma unroll
    for (int r = 0; r < RPT; r++)
#pragma unroll
        for (int q = 0; q < NC; q++)
#pragma unroll
            for (int i = 0; i < V; i++) a[q][i % ACC] += (float)AT(held[r][q], i);
    fold_rows<ACC>(a, p, red);
    fold_groups(red, mean_of);
    const float inverse = 1.0f / count;
    for (u32 g = threadIdx.x; g < KG; g += T) mean_of[g] *= inverse;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NC; q++) {
        float mean[ACC];
#pragma unroll
        for (int i = 0; i < ACC; i++) {
            a[q][i] = 0.0f;
            mean[i] = COLUMN(p, q) ? mean_of[group_of((p.tx + q * TX) * V + i)] : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < RPT; r++)
            if (HELD(p, r, q))
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float d = (float)AT(held[r][q], i) - mean[i % ACC];
                    a[q][i % ACC] += d * d;
                }
    }
    fold_rows<ACC>(a, p, red);
    fold_groups(red, m2_of);
}

// act(gamma (x - mean) rstd + beta); mean_of and rstd_of: of the slice's groups, `step` apart
__device__ __forceinline__ void store_applied(const vec_t (&held)[RPT][NC], const Place& p, const param_t* __restrict__ gamma, const param_t* __restrict__ beta,
                                              const float* mean_of, const float* rstd_of, u32 step, elem_t* __restrict__ y) {
    const u64 o = origin(p);
#pragma unroll
    for (int q = 0; q < NC; q++) {
        if (!COLUMN(p, q)) continue;
        float mean[ACC], scale[V], shift[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const u32 c = (p.tx + q * TX) * V + i;
            mean[i % ACC] = mean_of[group_of(c) * step];
            scale[i] = rstd_of[group_of(c) * step] * (float)gamma[p.slice * SC + c];
            shift[i] = (float)beta[p.slice * SC + c];
        }
#pragma unroll
        for (int r = 0; r < RPT; r++)
            if (HELD(p, r, q)) {
                vec_t out;
#pragma unroll
                for (int i = 0; i < V; i++) AT(out, i) = (elem_t)activate(((float)AT(held[r][q], i) - mean[i % ACC]) * scale[i] + shift[i]);
                STORE((vec_t*)(y + o + (u64)r * TY * C + q * TX * V), out);
            }
    }
}

#if WHOLE
extern "C" __global__ __launch_bounds__(T) void group_norm_forward(const elem_t* __restrict__ x, const param_t* __restrict__ gamma,
                                                                   const param_t* __restrict__ beta, elem_t* __restrict__ y,
                                                                   float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    __shared__ float red[RED_ROWS * CV * ACC], mean_of[KG], m2_of[KG];
    const Place p = place();
    vec_t held[RPT][NC];
    load_held(x, p, held);
    const float count = (float)PIXELS * (float)D;
    part_statistics(held, p, count, red, mean_of, m2_of);
    for (u32 g = threadIdx.x; g < KG; g += T) {
        const float rstd = 1.0f / sqrtf(m2_of[g] / count + EPS);
        m2_of[g] = rstd;
        if (mean_out) mean_out[p.n * G + p.slice * KG + g] = mean_of[g];
        if (rstd_out) rstd_out[p.n * G + p.slice * KG + g] = rstd;
    }
    __syncthreads();
    store_applied(held, p, gamma, beta, mean_of, m2_of, 1, y);
}
#else
extern "C" __global__ __launch_bounds__(T) void group_norm_stats(const elem_t* __restrict__ x, float* __restrict__ parts) {
    __shared__ float red[RED_ROWS * CV * ACC], mean_of[KG], m2_of[KG];
    const Place p = place();
    vec_t held[RPT][NC];
    load_held(x, p, held);
    const u64 first = (u64)p.chunk * ROWS;
    part_statistics(held, p, (float)(PIXELS - first < ROWS ? PIXELS - first : ROWS) * (float)D, red, mean_of, m2_of);
    for (u32 g = threadIdx.x; g < KG; g += T) {
        float* to = parts + (((p.n * G + p.slice * KG + g) * CHUNKS) + p.chunk) * 2;
        to[0] = mean_of[g];
        to[1] = m2_of[g];
    }
}

// The parts c = first, first + step, ... of a group, weighted by their pixels: a thread's share of the mean, and of the sum of squared
// distances from it.
#define PIXELS_OF(c) (PIXELS - (u64)(c) * ROWS < ROWS ? PIXELS - (u64)(c) * ROWS : ROWS)
__device__ __forceinline__ float share_of_mean(const float* __restrict__ parts, u32 first, u32 step) {
    const float whole = (float)PIXELS * (float)D;
    float s = 0.0f;
    for (u32 c = first; c < CHUNKS; c += step) s += parts[c * 2] * ((float)PIXELS_OF(c) * (float)D / whole);
    return s;
}
__device__ __forceinline__ float share_of_m2(const float* __restrict__ parts, u32 first, u32 step, float mean) {
    float m2 = 0.0f;
    for (u32 c = first; c < CHUNKS; c += step) {
        const float d = parts[c * 2] - mean;
        m2 += parts[c * 2 + 1] + d * d * ((float)PIXELS_OF(c) * (float)D);
    }
    return m2;
}
__device__ __forceinline__ float rstd_from(float m2) { return 1.0f / sqrtf(m2 / ((float)PIXELS * (float)D) + EPS); }

#if MERGE
// The parts of a (sample, group) by one workgroup, which has a thread to each of up to 1024: the parts were written on other XCDs and
// every look at them is a long one.
__device__ __forceinline__ float over_mergers(float s, float* waves) {
    for (int m = 32; m > 0; m /= 2) s += __shfl_xor(s, m, 64);
    if ((threadIdx.x & 63u) == 0) waves[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0f;
#pragma unroll
    for (u32 w = 0; w < MERGERS / 64; w++) s += waves[w];
    return s;
}
extern "C" __global__ __launch_bounds__(MERGERS) void group_norm_merge(const float* __restrict__ parts, float* __restrict__ stats,
                                                                      float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    __shared__ float waves[2][MERGERS / 64];
    for (u64 of = blockIdx.x; of < BATCH * G; of += MERGE_BLOCKS) {
        const float* from = parts + of * CHUNKS * 2;
        const float mean = over_mergers(share_of_mean(from, threadIdx.x, MERGERS), waves[0]);
        const float m2 = over_mergers(share_of_m2(from, threadIdx.x, MERGERS, mean), waves[1]);
        if (threadIdx.x == 0) {
            const float rstd = rstd_from(m2);
            stats[of * 2] = mean;
            stats[of * 2 + 1] = rstd;
            if (mean_out) mean_out[of] = mean;
            if (rstd_out) rstd_out[of] = rstd;
        }
        // (the next group's sums take the places of this one's)
        if (BATCH * G > MERGE_BLOCKS) __syncthreads();
    }
}
#endif

// `from`: the groups' statistics, or (few parts) the parts themselves, which every workgroup then joins for its groups; the first of a
// sample also writes the statistics.
extern "C" __global__ __launch_bounds__(T) void group_norm_apply(const elem_t* __restrict__ x, const param_t* __restrict__ gamma,
                                                                 const param_t* __restrict__ beta, const float* __restrict__ from,
                                                                 elem_t* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    const Place p = place();
    vec_t held[RPT][NC];
    load_held(x, p, held);
#if MERGE
    const float* of = from + (p.n * G + p.slice * KG) * 2;
    store_applied(held, p, gamma, beta, of, of + 1, 2, y);
#else
    __shared__ float mean_of[KG], rstd_of[KG];
    const u32 g = threadIdx.x / LPG, l = threadIdx.x % LPG;
    const u64 at = p.n * G + p.slice * KG + (g < KG ? g : 0);
    float s = share_of_mean(from + at * CHUNKS * 2, l, LPG);
    for (int m = LPG / 2; m > 0; m /= 2) s += __shfl_xor(s, m, 64);
    float m2 = share_of_m2(from + at * CHUNKS * 2, l, LPG, s);
    for (int m = LPG / 2; m > 0; m /= 2) m2 += __shfl_xor(m2, m, 64);
    if (g < KG && l == 0) {
        mean_of[g] = s;
        rstd_of[g] = rstd_from(m2);
        if (mean_out && p.chunk == 0) mean_out[at] = s;
        if (rstd_out && p.chunk == 0) rstd_out[at] = rstd_of[g];
    }
    __syncthreads();
    store_applied(held, p, gamma, beta, mean_of, rstd_of, 1, y);
#endif
}
#endif
)HIP";

// Gradients. With dz = dy act'(z), a sample's sums over its pixels, A_c = sum dz and B_c = sum dz xh, give everything: dbeta and
// dgamma are their sums over the samples, and a group's s1 = sum gamma_c A_c / M, s2 = sum gamma_c B_c / M are what
// dx = rstd (gamma_c dz - s1 - xh s2) takes away. A workgroup that holds all pixels of its groups (WHOLE) reads x and dy once;
// otherwise `sums` and `gradient` read them both, with `fold` adding up the chunks of a sample between them.
//
// Bound by memory: 64 x 3136 x 256 bf16 with silu, in parts: sums 34 us (6.2 TB/s), fold 5, gradient 48 (6.4 TB/s). Once through
// memory would be 54, but x and dy of four groups (64 bytes of a pixel) take 400 KB, nearly all registers of a CU, so that nothing loads while a
// workgroup sums and stores: 128 x 784 x 512 took 90 to 107 us whole and 100 in parts. Small calls gain: 8 x 64 x 256 f32 3.7 + 2 us.
const char* kBackward = R"HIP(
struct Column { float mean[ACC], rstd[ACC], scale[V], shift[V]; };   // z = (x - mean) scale + shift
__device__ __forceinline__ void load_column(Column& k, const Place& p, int q, const param_t* __restrict__ gamma, const param_t* __restrict__ beta,
                                            const float* __restrict__ mean, const float* __restrict__ rstd) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        const u32 c = (p.tx + q * TX) * V + i;
        const u64 g = p.n * G + p.slice * KG + group_of(c);
        k.mean[i % ACC] = mean[g];
        k.rstd[i % ACC] = rstd[g];
        k.scale[i] = rstd[g] * (float)gamma[p.slice * SC + c];
        k.shift[i] = (float)beta[p.slice * SC + c];
    }
}
__device__ __forceinline__ float from_mean(const Column& k, int i, float x) { return x - k.mean[i % ACC]; }
__device__ __forceinline__ float dz_of(const Column& k, int i, float from_mean, float dy) { return slope_times(dy, from_mean * k.scale[i] + k.shift[i]); }

// A channel's sums over the pixels that a thread holds: dz, and dz (x - mean), which times rstd is dz xh.
__device__ __forceinline__ void add_to_sums(float (&a)[2 * V], int i, float from_mean, float dz) {
    a[2 * i] += dz;
    a[2 * i + 1] += dz * from_mean;
}
__device__ __forceinline__ void end_sums(float (&a)[2 * V], const Column& k) {
#pragma unroll
    for (int i = 0; i < V; i++) a[2 * i + 1] *= k.rstd[i % ACC];
}
// dx of one element: scale dz - (rstd s1 + (x - mean) rstd^2 s2)
struct Minus { float by[ACC], slope[ACC]; };
__device__ __forceinline__ elem_t dx_of(const Column& k, const Minus& s, int i, float from_mean, float dz) {
    return (elem_t)(k.scale[i] * dz - (from_mean * s.slope[i % ACC] + s.by[i % ACC]));
}
// The groups' s1 and s2 from the channels' sums over all pixels.
__device__ __forceinline__ void group_sums_of(const float* sums, const param_t* __restrict__ gamma, const Place& p, float* out) {
    const u32 g = threadIdx.x / LPG, l = threadIdx.x % LPG;
    float s1 = 0.0f, s2 = 0.0f;
    if (g < KG)
        for (u32 c = g * D + l; c < (g + 1) * D; c += LPG) {
            const float w = (float)gamma[p.slice * SC + c];
            s1 += w * sums[2 * c];
            s2 += w * sums[2 * c + 1];
        }
    for (int m = LPG / 2; m > 0; m /= 2) {
        s1 += __shfl_xor(s1, m, 64);
        s2 += __shfl_xor(s2, m, 64);
    }
    const float whole = (float)PIXELS * (float)D;
    if (g < KG && l == 0) {
        out[2 * g] = s1 / whole;
        out[2 * g + 1] = s2 / whole;
    }
    __syncthreads();
}
__device__ __forceinline__ void load_minus(Minus& s, const Column& k, const Place& p, int q, const float* group_sums) {
#pragma unroll
    for (int i = 0; i < ACC; i++) {
        const u32 g = group_of((p.tx + q * TX) * V + i);
        s.by[i] = k.rstd[i] * group_sums[2 * g];
        s.slope[i] = k.rstd[i] * k.rstd[i] * group_sums[2 * g + 1];
    }
}

// The samples' sums [batch][2][C] added up for the parameters, in an order that is fixed and with no chain of more than a few hundred
// additions. Up to 1024 samples: 64 channels to a workgroup, the samples shared by its waves. More of them are first added up 256 to a row, until
// 1024 rows or fewer are left (FINAL, FINAL_AT floats behind the samples): a workgroup takes 64 of the 2 C sums of 256 rows.
extern "C" __global__ __launch_bounds__(256) void group_norm_level(const float* __restrict__ from, float* __restrict__ to, u64 count) {
    __shared__ float part[4][64];
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u64 columns = (2 * C + 63) / 64, row = blockIdx.x / columns, e = blockIdx.x % columns * 64 + lane;
    const u64 end = row * 256 + 256 < count ? row * 256 + 256 : count;
    float s = 0.0f;
    if (e < 2 * C)
#pragma unroll 8
        for (u64 n = row * 256 + wave; n < end; n += 4) s += from[n * (2 * C) + e];
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && e < 2 * C) to[row * (2 * C) + e] = s + part[1][lane] + part[2][lane] + part[3][lane];
}
template <int WAVES> __device__ __forceinline__ void parameter_gradients(u64 block, const float* __restrict__ samples, float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float part[2][WAVES][64];
    const float* rows = samples + FINAL_AT;
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u64 c = block * 64 + lane;
    float a = 0.0f, b = 0.0f;
    if (c < C)
        for (u64 n = wave; n < FINAL; n += WAVES) {
            a += rows[(n * 2) * C + c];
            b += rows[(n * 2 + 1) * C + c];
        }
    part[0][wave][lane] = a;
    part[1][wave][lane] = b;
    __syncthreads();
    if (wave == 0 && c < C) {
        for (u32 w = 1; w < WAVES; w++) {
            a += part[0][w][lane];
            b += part[1][w][lane];
        }
        dbeta[c] = a;
        dgamma[c] = b;
    }
}

#if WHOLE
// (silu's slope costs more than the rest: dz is held in f32 then, instead of dy and a second round of slopes)
#define HOLD_DZ (ACT == 2)
extern "C" __global__ __launch_bounds__(T) void group_norm_backward(const elem_t* __restrict__ dy, const elem_t* __restrict__ x,
                                                                    const param_t* __restrict__ gamma, const param_t* __restrict__ beta,
                                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                    float* __restrict__ samples, elem_t* __restrict__ dx) {
    __shared__ float red[RED_ROWS * CV * V * 2], sums_apart[SUMS_APART], group_sums[KG * 2];
    float* sums = ONE_ROW ? red : sums_apart;
    const Place p = place();
    vec_t hx[RPT][NC], hd[RPT][NC];
    load_held(x, p, hx);
    load_held(dy, p, hd);
    float a[NC][2 * V];
#if HOLD_DZ
    float dz[RPT][NC][V];
#endif
#pragma unroll
    for (int q = 0; q < NC; q++) {
#pragma unroll
        for (int i = 0; i < 2 * V; i++) a[q][i] = 0.0f;
        if (p.ty < TY && COLUMN(p, q)) {
            Column k;
            load_column(k, p, q, gamma, beta, mean, rstd);
#pragma unroll
            for (int r = 0; r < RPT; r++) {
#if HOLD_DZ
#pragma unroll
                for (int i = 0; i < V; i++) dz[r][q][i] = 0.0f;
#endif
                if (HELD(p, r, q))
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float c = from_mean(k, i, (float)AT(hx[r][q], i)), d = dz_of(k, i, c, (float)AT(hd[r][q], i));
                        add_to_sums(a[q], i, c, d);
#if HOLD_DZ
                        dz[r][q][i] = d;
#endif
                    }
            }
            end_sums(a[q], k);
        }
    }
    fold_rows<2 * V>(a, p, red);
    fold_entries<SC * 2, LPE>(red, sums);
    for (u32 e = threadIdx.x; e < SC * 2; e += T) samples[(p.n * 2 + (e & 1)) * C + p.slice * SC + (e >> 1)] = sums[e];
    group_sums_of(sums, gamma, p, group_sums);
    const u64 o = origin(p);
#pragma unroll
    for (int q = 0; q < NC; q++) {
        if (p.ty >= TY || !COLUMN(p, q)) continue;
        Column k;
        load_column(k, p, q, gamma, beta, mean, rstd);
        Minus s;
        load_minus(s, k, p, q, group_sums);
#pragma unroll
        for (int r = 0; r < RPT; r++)
            if (HELD(p, r, q)) {
                vec_t out;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float c = from_mean(k, i, (float)AT(hx[r][q], i));
#if HOLD_DZ
                    AT(out, i) = dx_of(k, s, i, c, dz[r][q][i]);
#else
                    AT(out, i) = dx_of(k, s, i, c, dz_of(k, i, c, (float)AT(hd[r][q], i)));
#endif
                }
                STORE((vec_t*)(dx + o + (u64)r * TY * C + q * TX * V), out);
            }
    }
}

extern "C" __global__ __launch_bounds__(256) void group_norm_parameters(const float* __restrict__ samples, float* __restrict__ dgamma, float* __restrict__ dbeta) {
    parameter_gradients<4>(blockIdx.x, samples, dgamma, dbeta);
}
#else
// parts: [batch * CHUNKS][2][C]
extern "C" __global__ __launch_bounds__(T) void group_norm_sums(const elem_t* __restrict__ dy, const elem_t* __restrict__ x,
                                                                const param_t* __restrict__ gamma, const param_t* __restrict__ beta,
                                                                const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                float* __restrict__ parts) {
    __shared__ float red[RED_ROWS * CV * V * 2], sums_apart[SUMS_APART];
    float* sums = ONE_ROW ? red : sums_apart;
    const Place p = place();
    vec_t hx[RPT][NC], hd[RPT][NC];
    load_held(x, p, hx);
    load_held(dy, p, hd);
    float a[NC][2 * V];
#pragma unroll
    for (int q = 0; q < NC; q++) {
#pragma unroll
        for (int i = 0; i < 2 * V; i++) a[q][i] = 0.0f;
        if (p.ty < TY && COLUMN(p, q)) {
            Column k;
            load_column(k, p, q, gamma, beta, mean, rstd);
#pragma unroll
            for (int r = 0; r < RPT; r++)
                if (HELD(p, r, q))
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float c = from_mean(k, i, (float)AT(hx[r][q], i));
                        add_to_sums(a[q], i, c, dz_of(k, i, c, (float)AT(hd[r][q], i)));
                    }
            end_sums(a[q], k);
        }
    }
    fold_rows<2 * V>(a, p, red);
    fold_entries<SC * 2, LPE>(red, sums);
    for (u32 e = threadIdx.x; e < SC * 2; e += T) parts[((p.n * CHUNKS + p.chunk) * 2 + (e & 1)) * C + p.slice * SC + (e >> 1)] = sums[e];
}

// The chunks of a sample added up (one chunk is its sample's sums already, and none is launched): [batch][2][C]. A workgroup takes 32 of a sample's 2 C sums, its 32 rows of threads every 32nd chunk.
// Bound by the latency of reading what other XCDs wrote: four chunks at a time instead of one take the whole backward pass of 2 x 262144 x 128
// from 146 to 136 us.
extern "C" __global__ __launch_bounds__(1024) void group_norm_fold(const float* __restrict__ parts, float* __restrict__ samples) {
    __shared__ float part[32][33];
    const u64 per = (2 * C + 31) / 32;
    const u32 row = threadIdx.x >> 5, column = threadIdx.x & 31u;
    for (u64 b = blockIdx.x; b < BATCH * per; b += FOLD_BLOCKS) {
        const u64 n = b / per, e = b % per * 32 + column;
        float s = 0.0f;
        if (e < 2 * C)
            for (u64 k = row; k < CHUNKS; k += 128) {
                float of[4];   // (four on their way at a time)
#pragma unroll
                for (u32 d = 0; d < 4; d++) of[d] = k + d * 32 < CHUNKS ? parts[(n * CHUNKS + k + d * 32) * (2 * C) + e] : 0.0f;
#pragma unroll
                for (u32 d = 0; d < 4; d++) s += of[d];
            }
        part[row][column] = s;
        __syncthreads();
        // (transposed: a row's threads now hold one sum's 32 shares)
        s = part[column][row];
        for (int m = 16; m > 0; m /= 2) s += __shfl_xor(s, m, 64);
        const u64 mine = b % per * 32 + row;
        if (column == 0 && mine < 2 * C) samples[n * (2 * C) + mine] = s;
        if (BATCH * per > FOLD_BLOCKS) __syncthreads();
    }
}

// The workgroups behind the tensor's own add up the samples' sums.
extern "C" __global__ __launch_bounds__(T) void group_norm_gradient(const elem_t* __restrict__ dy, const elem_t* __restrict__ x,
                                                                    const param_t* __restrict__ gamma, const param_t* __restrict__ beta,
                                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                    const float* __restrict__ samples, elem_t* __restrict__ dx,
                                                                    float* __restrict__ dgamma, float* __restrict__ dbeta) {
    if (blockIdx.x >= BLOCKS) return parameter_gradients<T / 64>(blockIdx.x - BLOCKS, samples, dgamma, dbeta);
    __shared__ float sums[SC * 2], group_sums[KG * 2];
    const Place p = place();
    vec_t hx[RPT][NC], hd[RPT][NC];
    load_held(x, p, hx);
    load_held(dy, p, hd);
    for (u32 e = threadIdx.x; e < SC * 2; e += T) sums[e] = samples[(p.n * 2 + (e & 1)) * C + p.slice * SC + (e >> 1)];
    __syncthreads();
    group_sums_of(sums, gamma, p, group_sums);
    const u64 o = origin(p);
#pragma unroll
    for (int q = 0; q < NC; q++) {
        if (p.ty >= TY || !COLUMN(p, q)) continue;
        Column k;
        load_column(k, p, q, gamma, beta, mean, rstd);
        Minus s;
        load_minus(s, k, p, q, group_sums);
#pragma unroll
        for (int r = 0; r < RPT; r++)
            if (HELD(p, r, q)) {
                vec_t out;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float c = from_mean(k, i, (float)AT(hx[r][q], i));
                    AT(out, i) = dx_of(k, s, i, c, dz_of(k, i, c, (float)AT(hd[r][q], i)));
                }
                STORE((vec_t*)(dx + o + (u64)r * TY * C + q * TX * V), out);
            }
    }
}
#endif
)HIP";

int pow2_floor(int64_t x) {
    int p = 1;
    while ((int64_t)p * 2 <= x && p < (1 << 30)) p *= 2;
    return p;
}

// A launch has fewer than 2^32 threads. The tensor's own launches are refused beyond that; of the small ones between them, whose workgroups
// of up to 1024 threads come to it sooner, a workgroup then does the work of several.
constexpr uint64_t kThreads = 1ull << 32;
uint32_t fold_blocks(const GroupNormProblem& pr) { return (uint32_t)std::min<uint64_t>((uint64_t)pr.batch * ((2 * pr.channels + 31) / 32), (kThreads - 1) / 1024); }
uint32_t merge_blocks(const GroupNormProblem& pr, const GroupNormTiling& t) { return (uint32_t)std::min<uint64_t>((uint64_t)pr.batch * pr.groups, (kThreads - 1) / t.mergers()); }

// Rows of sums that the parameters' gradients come from: the samples', then fewer and fewer, one behind the other.
std::vector<uint64_t> sum_levels(const GroupNormProblem& pr) {
    std::vector<uint64_t> rows{(uint64_t)pr.batch};
    while (rows.back() > 1024) rows.push_back((rows.back() + 255) / 256);
    return rows;
}
uint64_t all_rows(const std::vector<uint64_t>& levels) { return std::accumulate(levels.begin(), levels.end(), (uint64_t)0); }

std::string definitions(const GroupNormProblem& pr, const GroupNormTiling& t) {
    const int64_t d = pr.channels / pr.groups;
    const std::vector<uint64_t> levels = sum_levels(pr);
    std::ostringstream s;
    s << "#define BATCH " << pr.batch << "ull\n#define FINAL " << levels.back() << "ull\n#define FINAL_AT " << (all_rows(levels) - levels.back()) * 2 * pr.channels
      << "ull\n#define PIXELS " << pr.pixels << "ull\n#define C " << pr.channels << "\n#define G " << pr.groups
      << "\n#define D " << d << "\n#define V " << t.vec << "\n#define T " << t.threads << "\n#define KG " << t.slice_groups << "\n#define SC "
      << t.slice << "\n#define SLICES " << pr.groups / t.slice_groups << "\n#define CV " << t.slice / t.vec << "\n#define TX " << t.tx
      << "\n#define TY " << t.ty << "\n#define NC " << t.columns << "\n#define RPT " << t.rows_per_thread << "\n#define ROWS " << t.rows()
      << "\n#define CHUNKS " << t.chunks << "\n#define BLOCKS " << t.grid << "ull\n#define LPG "
      << std::min(64, pow2_floor(t.threads / t.slice_groups)) << "\n#define BF16 " << (pr.dtype == HE_BF16) << "\n#define F16 "
      << (pr.dtype == HE_F16) << "\n#define PARAM_SAME " << (pr.param_dtype == pr.dtype) << "\n#define ACT " << pr.activation
      << "\n#define EPS " << strfmt("%.9ef", (double)pr.epsilon) << "\n#define WHOLE " << (int)t.whole << "\n#define STREAM " << (int)t.stream << "\n#define MERGE " << (int)t.merge << "\n#define MERGERS " << t.mergers()
      << "\n#define MERGE_BLOCKS " << merge_blocks(pr, t) << "ull\n#define FOLD_BLOCKS " << fold_blocks(pr) << "ull"
      << "\n#define LPE " << std::min<int64_t>(64, pow2_floor(std::max<int64_t>(1, t.threads / (2 * t.slice)))) << "\n";
    return s.str();
}

}  // namespace

std::string GroupNormTiling::describe() const {
    return strfmt("%s vec=%d threads=%d slice=%lld(%d groups) tx=%lld ty=%lld columns=%d rows_per_thread=%d chunks=%lld grid=%llu", whole ? "whole" : "parts", vec, threads,
                  (long long)slice, slice_groups, (long long)tx, (long long)ty, columns, rows_per_thread, (long long)chunks, (unsigned long long)grid);
}

GroupNormTiling plan_group_norm(const GroupNormProblem& pr, bool backward) {
    GroupNormTiling t;
    const int esz = (int)dtype_bits(pr.dtype) / 8;
    const int64_t d = pr.channels / pr.groups;
    t.vec = 16 / esz;
    while (pr.channels % t.vec) t.vec /= 2;
    // registers that one vector of a pixel takes: x; going back also dy, or what silu makes of it in f32
    const int raw = std::max(1, t.vec * esz / 4);
    const auto vector_regs = [&](bool whole) { return raw + (!backward ? 0 : whole && pr.activation == HE_ACT_SILU ? t.vec : raw); };
    t.stream = (uint64_t)pr.batch * pr.pixels * pr.channels * esz >= (4u << 20) && tuning::get_int("HELIUM_HIP_NORM_STREAM", 1);

    // Whole groups of a sample to a workgroup, if its registers hold them and that is estimated to take less than two ways through
    // memory: of slices the one that costs least, then as few threads as keep a thread's data in 32 registers. Microseconds, from
    // measurements of 0.1 to 270 MB: 5.5 MB are moved in one where a pixel's part of a slice is at least 64 bytes (32 bytes:
    // a third, 16: an eighth of that), one workgroup moves 45 KB, and a thousand workgroups take 1.5 to begin and end.
    const int forced_k = tuning::get_int("HELIUM_HIP_NORM_SLICE", 0), forced_t = tuning::get_int("HELIUM_HIP_NORM_THREADS", 0);
    const double bytes = (double)pr.batch * pr.pixels * pr.channels * esz, moved = backward ? 3 : 2;
    double best = backward ? 12 + 5 * bytes / 5.5e6 : 9 + 3 * bytes / 5.5e6;
    if (forced_k || forced_t) best = 1e30;
    for (int64_t k = 1; k <= pr.groups && !tuning::get_int("HELIUM_HIP_NORM_PARTS", 0); k++) {
        if (pr.groups % k || k * d % t.vec || (forced_k && k != forced_k)) continue;
        const int64_t tx = k * d / t.vec;
        int threads = 0;
        for (int candidate : {256, 512, 1024}) {
            if (k > candidate || tx > candidate || (forced_t && candidate != forced_t)) continue;
            const int64_t regs = (pr.pixels + candidate / tx - 1) / (candidate / tx) * vector_regs(true);
            if (regs > (candidate == 1024 ? 56 : 64)) continue;
            threads = candidate;
            if (regs <= 32) break;
        }
        if (!threads) continue;
        const double segment = (double)k * d * esz, eff = k == pr.groups || segment >= 64 ? 1.0 : std::pow(segment / 64, 1.5);
        const double cost = (backward ? 8 : 5) + 1.5e-3 * pr.batch * (pr.groups / k) + std::max(moved * bytes / (5.5e6 * eff * (backward ? 0.65 : 1.0)), moved * segment * pr.pixels / 45e3);
        if (cost >= best) continue;
        best = cost;
        t.whole = true;
        t.threads = threads, t.slice_groups = (int)k, t.slice = k * d, t.tx = tx, t.ty = threads / tx, t.columns = 1;
        t.rows_per_thread = (int)((pr.pixels + t.ty - 1) / t.ty), t.chunks = 1;
        t.grid = (uint64_t)pr.batch * (pr.groups / k);
    }
    if (t.whole) return t;

    // The narrowest slice of whole groups and whole vectors that is at least 256 bytes of a pixel.
    t.threads = 256;
    for (int64_t k = 1; k <= pr.groups; k++) {
        if (pr.groups % k || k * d % t.vec || k > t.threads) continue;
        t.slice_groups = (int)k;
        t.slice = k * d;
        if (t.slice * esz >= 256) break;
    }
    HE_REQUIRE(t.slice, HE_ERR_UNSUPPORTED, "group norm: no slice of %lld channels in %lld groups", (long long)pr.channels, (long long)pr.groups);
    const int64_t cv = t.slice / t.vec;
    t.tx = std::min<int64_t>(cv, t.threads);
    t.ty = t.threads / t.tx;
    t.columns = (int)((cv + t.tx - 1) / t.tx);
    // 64 registers of data per thread, half or less of that where that leaves compute units idle (forward below 1024 workgroups;
    // backward, whose parts are many sums that `fold` reads, below 512: 1 x 65536 x 64 bf16 19.3 -> 16.9 us, 8 x 4096 x 320 31.5 -> 30.2)
    int64_t rpt = std::max<int64_t>(1, 64 / (vector_regs(false) * t.columns));
    const int64_t slices = pr.groups / t.slice_groups;
    while (rpt > 1 && (t.ty * (rpt / 2) >= pr.pixels || (uint64_t)(pr.batch * slices) * ((pr.pixels + t.ty * rpt - 1) / (t.ty * rpt)) < (backward ? 512u : 1024u))) rpt /= 2;
    // (forward, a full chip does better with 48 registers of data: 2 x 262144 x 128 bf16 71 -> 68 us, 64 x 3136 x 256 54 -> 52, 32 x 784 x 512
    // f32 28.0 -> 27.4; backward 96 -> 98-103 for 32 or 96 instead of 64)
    if (!backward && rpt % 4 == 0 && rpt * vector_regs(false) * t.columns == 64) rpt = rpt / 4 * 3;
    t.rows_per_thread = (int)rpt;
    t.chunks = (pr.pixels + t.rows() - 1) / t.rows();
    t.merge = t.chunks > 32;
    t.grid = (uint64_t)pr.batch * slices * t.chunks;
    return t;
}

GroupNorm::GroupNorm(const GroupNormProblem& pr) : pr_(pr) {
    HE_REQUIRE(pr.batch >= 0 && pr.pixels >= 1 && pr.channels >= 1 && pr.groups >= 1, HE_ERR_INVALID,
               "group norm: batch %lld, pixels %lld, channels %lld, groups %lld", (long long)pr.batch, (long long)pr.pixels,
               (long long)pr.channels, (long long)pr.groups);
    HE_REQUIRE(pr.channels % pr.groups == 0, HE_ERR_INVALID, "group norm: %lld channels do not divide into %lld groups", (long long)pr.channels,
               (long long)pr.groups);
    HE_REQUIRE(pr.dtype == HE_F16 || pr.dtype == HE_BF16 || pr.dtype == HE_F32, HE_ERR_INVALID, "group norm does not take dtype %s", dtype_name(pr.dtype));
    HE_REQUIRE(pr.param_dtype == HE_F32 || pr.param_dtype == pr.dtype, HE_ERR_INVALID, "group norm: parameters are f32 or of the tensor's type, not %s",
               dtype_name(pr.param_dtype));
    HE_REQUIRE(pr.activation >= HE_ACT_NONE && pr.activation <= HE_ACT_SILU, HE_ERR_INVALID, "group norm: unknown activation %d", pr.activation);
    HE_REQUIRE(std::isfinite(pr.epsilon) && pr.epsilon >= 0, HE_ERR_INVALID, "group norm: epsilon %g", (double)pr.epsilon);
    // (a group's channels stay together: two sums of each of 16384 are 128 KB of a workgroup's 160 KB of LDS)
    HE_REQUIRE(pr.channels <= 16384, HE_ERR_UNSUPPORTED, "group norm: %lld channels, at most 16384 are taken", (long long)pr.channels);
    // (2^46 elements are beyond any memory, and leave products of counts their 64 bits)
    HE_REQUIRE((double)pr.batch * (double)pr.pixels * (double)pr.channels <= (double)(1ull << 46), HE_ERR_UNSUPPORTED, "group norm: extents too large");
    fwd_ = plan_group_norm(pr, false);
    bwd_ = plan_group_norm(pr, true);
    levels_ = sum_levels(pr);
    const uint64_t channel_blocks = (pr.channels + 63) / 64, level_blocks = levels_.size() > 1 ? levels_[1] * ((2 * pr.channels + 63) / 64) : 0;
    HE_REQUIRE(fwd_.grid < kThreads / fwd_.threads && bwd_.grid + channel_blocks < kThreads / bwd_.threads && level_blocks < kThreads / 256, HE_ERR_UNSUPPORTED,
               "group norm: the tensor is too large for one launch");
    const std::string forward = definitions(pr, fwd_) + kCommon + kForward, backward = definitions(pr, bwd_) + kCommon + kBackward;
    auto compiled = std::async(std::launch::async, [&] { (void)rtc_compile(backward, "group_norm", {}); });
    auto make = [](const std::string& text, const char* entry) { return std::make_unique<JitKernel>(text, entry); };
    if (fwd_.whole) {
        whole_forward_ = make(forward, "group_norm_forward");
    } else {
        stats_ = make(forward, "group_norm_stats");
        if (fwd_.merge) merge_ = make(forward, "group_norm_merge");
        apply_ = make(forward, "group_norm_apply");
    }
    compiled.get();
    if (levels_.size() > 1) level_ = make(backward, "group_norm_level");
    if (bwd_.whole) {
        whole_backward_ = make(backward, "group_norm_backward");
        parameters_ = make(backward, "group_norm_parameters");
    } else {
        sums_ = make(backward, "group_norm_sums");
        if (bwd_.chunks > 1) fold_ = make(backward, "group_norm_fold");
        gradient_ = make(backward, "group_norm_gradient");
    }
    const uint64_t rows = (uint64_t)pr.batch * pr.groups, sums = 2 * (uint64_t)pr.channels;
    scratch_floats_ = std::max(rows * 2 * (fwd_.chunks + 1), sums * (all_rows(levels_) + pr.batch * bwd_.chunks));
    source_ = forward + "\n" + backward;
    describe_ = "group_norm forward: " + fwd_.describe() + "\ngroup_norm backward: " + bwd_.describe() + " samples=";
    for (size_t k = 0; k < levels_.size(); k++) describe_ += (k ? "," : "") + std::to_string(levels_[k]);
}

GroupNorm::~GroupNorm() { scratch_.release(); }

void GroupNorm::check(std::initializer_list<const void*> tensors, std::initializer_list<const void*> params,
                      std::initializer_list<const void*> stats) const {
    const uintptr_t mask = (uintptr_t)fwd_.vec * dtype_bits(pr_.dtype) / 8 - 1, pmask = dtype_bits(pr_.param_dtype) / 8 - 1;
    for (const void* p : tensors)
        HE_REQUIRE(p && ((uintptr_t)p & mask) == 0, HE_ERR_INVALID, "group norm: a tensor is null or not aligned to %d bytes", (int)mask + 1);
    for (const void* p : params)
        HE_REQUIRE(p && ((uintptr_t)p & pmask) == 0, HE_ERR_INVALID, "group norm: gamma or beta is null or not aligned");
    for (const void* p : stats) HE_REQUIRE(((uintptr_t)p & 3) == 0, HE_ERR_INVALID, "group norm: statistics are not aligned");
}

void GroupNorm::forward(const void* x, const void* gamma, const void* beta, void* y, float* mean, float* rstd, hipStream_t stream) {
    if (pr_.batch == 0) return;
    check({x, y}, {gamma, beta}, {mean, rstd});
    const uint32_t grid[3] = {(uint32_t)fwd_.grid, 1, 1}, block[3] = {(uint32_t)fwd_.threads, 1, 1};
    if (fwd_.whole) {
        void* args[] = {&x, &gamma, &beta, &y, &mean, &rstd};
        whole_forward_->launch(grid, block, 0, stream, args, true);
        return;
    }
    const uint64_t rows = (uint64_t)pr_.batch * pr_.groups;
    std::lock_guard<std::mutex> lk(mu_);
    float* parts = scratch_.get(scratch_floats_, 0, stream).floats;
    float* stats = parts + rows * fwd_.chunks * 2;
    const uint32_t merge_grid[3] = {merge_blocks(pr_, fwd_), 1, 1}, merge_block[3] = {(uint32_t)fwd_.mergers(), 1, 1};
    void* a[] = {&x, &parts};
    stats_->launch(grid, block, 0, stream, a);
    void* b[] = {&parts, &stats, &mean, &rstd};
    if (fwd_.merge) merge_->launch(merge_grid, merge_block, 0, stream, b);
    void* c[] = {&x, &gamma, &beta, fwd_.merge ? &stats : &parts, &y, &mean, &rstd};
    apply_->launch(grid, block, 0, stream, c, true);
}

void GroupNorm::add_levels(float* samples, hipStream_t stream) {
    const uint64_t sums = 2 * (uint64_t)pr_.channels, columns = (sums + 63) / 64;
    const uint32_t block[3] = {256, 1, 1};
    for (size_t k = 1; k < levels_.size(); k++) {
        uint64_t count = levels_[k - 1];
        float* to = samples + count * sums;
        const uint32_t grid[3] = {(uint32_t)(levels_[k] * columns), 1, 1};
        void* args[] = {&samples, &to, &count};
        level_->launch(grid, block, 0, stream, args);
        samples = to;
    }
}

void GroupNorm::backward(const void* dy, const void* x, const void* gamma, const void* beta, const float* mean, const float* rstd, void* dx,
                         float* dgamma, float* dbeta, hipStream_t stream) {
    HE_REQUIRE(dgamma && dbeta, HE_ERR_INVALID, "group norm: the parameters' gradients are null");
    if (pr_.batch) {
        check({dy, x, dx}, {gamma, beta}, {mean, rstd, dgamma, dbeta});
        HE_REQUIRE(mean && rstd, HE_ERR_INVALID, "group norm: the backward pass needs the statistics of the forward pass");
    }
    const uint64_t sums = 2 * (uint64_t)pr_.channels;
    std::lock_guard<std::mutex> lk(mu_);
    float *samples = scratch_.get(scratch_floats_, 0, stream).floats, *parts = fold_ ? samples + sums * all_rows(levels_) : samples;
    const uint32_t channel_blocks = (uint32_t)((pr_.channels + 63) / 64), small[3] = {256, 1, 1};
    const uint32_t grid[3] = {(uint32_t)bwd_.grid, 1, 1}, block[3] = {(uint32_t)bwd_.threads, 1, 1};
    if (bwd_.whole) {
        const uint32_t last_grid[3] = {channel_blocks, 1, 1};
        void* a[] = {&dy, &x, &gamma, &beta, &mean, &rstd, &samples, &dx};
        if (pr_.batch) whole_backward_->launch(grid, block, 0, stream, a);
        add_levels(samples, stream);
        void* b[] = {&samples, &dgamma, &dbeta};
        parameters_->launch(last_grid, small, 0, stream, b, true);
        return;
    }
    if (pr_.batch) {
        const uint32_t fold_grid[3] = {fold_blocks(pr_), 1, 1}, fold_block[3] = {1024, 1, 1};
        void* a[] = {&dy, &x, &gamma, &beta, &mean, &rstd, &parts};
        sums_->launch(grid, block, 0, stream, a);
        void* b[] = {&parts, &samples};
        if (fold_) fold_->launch(fold_grid, fold_block, 0, stream, b);
        add_levels(samples, stream);
    }
    // (without samples only the parameters' gradients are left, all zero)
    const uint32_t last_grid[3] = {(uint32_t)bwd_.grid + channel_blocks, 1, 1};
    void* c[] = {&dy, &x, &gamma, &beta, &mean, &rstd, &samples, &dx, &dgamma, &dbeta};
    gradient_->launch(last_grid, block, 0, stream, c, true);
}

}  // namespace he

// ---- C ABI ------------------------------------------------------------------------------------------------
struct he_group_norm_s {
    he::GroupNorm impl;
    explicit he_group_norm_s(const he::GroupNormProblem& pr) : impl(pr) {}
};

extern "C" {

int he_group_norm_create(he_group_norm_t* norm, int64_t batch, int64_t pixels, int64_t channels, int64_t groups, int dtype, int param_dtype,
                         int activation, float epsilon) {
    return he::guard([&] {
        HE_REQUIRE(norm, HE_ERR_INVALID, "bad argument");
        he::GroupNormProblem pr;
        pr.batch = batch, pr.pixels = pixels, pr.channels = channels, pr.groups = groups;
        pr.dtype = dtype, pr.param_dtype = param_dtype, pr.activation = activation, pr.epsilon = epsilon;
        *norm = new he_group_norm_s(pr);
    });
}

int he_group_norm_destroy(he_group_norm_t norm) {
    return he::guard([&] { delete norm; });
}

int he_group_norm_forward(he_group_norm_t norm, const void* x, const void* gamma, const void* beta, void* y, float* mean, float* rstd,
                          he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(norm, HE_ERR_INVALID, "null group norm");
        norm->impl.forward(x, gamma, beta, y, mean, rstd, stream ? stream->s : nullptr);
    });
}

int he_group_norm_backward(he_group_norm_t norm, const void* dy, const void* x, const void* gamma, const void* beta, const float* mean,
                           const float* rstd, void* dx, float* dgamma, float* dbeta, he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(norm, HE_ERR_INVALID, "null group norm");
        norm->impl.backward(dy, x, gamma, beta, mean, rstd, dx, dgamma, dbeta, stream ? stream->s : nullptr);
    });
}

const char* he_group_norm_source(he_group_norm_t norm) { return norm ? norm->impl.source().c_str() : ""; }
const char* he_group_norm_describe(he_group_norm_t norm) { return norm ? norm->impl.describe().c_str() : ""; }

}  // extern "C"
