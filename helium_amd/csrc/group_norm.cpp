#include "group_norm.h"

#include <algorithm>
#include <cmath>
#include <future>
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
    u64 b = blockIdx.x;
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
#define COLUMN(p, q) ((p).tx + (q) * TX < CV)
#define HELD(p, r, q) ((r) * TY < (p).left && COLUMN(p, q))

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

__device__ __forceinline__ float activate(float z) {
#if ACT == 1
    return z > 0.0f ? z : (z != z ? z : 0.0f);
#elif ACT == 2
    return z * HE_FAST_RCP(1.0f + __expf(-z));
#else
    return z;
#endif
}
// dz from dy: the activation's slope at z
__device__ __forceinline__ float slope_times(float dy, float z) {
#if ACT == 1
    return z > 0.0f ? dy : (z != z ? z : 0.0f);
#elif ACT == 2
    const float s = HE_FAST_RCP(1.0f + __expf(-z));
    return dy * (s + z * s * (1.0f - s));
#else
    return dy;
#endif
}
)HIP";

// Statistics. A workgroup holds its part of a sample in registers, takes the mean of each group in it, then the sum of squared
// distances from that mean (not E[x^2] - E[x]^2, which loses all digits of a variance that is small beside the mean). `merge`
// joins the parts of a group: M2 = sum of M2_i + n_i (mean_i - mean)^2.
const char* kForward = R"HIP(
extern "C" __global__ __launch_bounds__(T) void group_norm_stats(const elem_t* __restrict__ x, float* __restrict__ parts) {
    __shared__ float red[RED_ROWS * CV * ACC], group_mean[KG], group_m2[KG];
    const Place p = place();
    vec_t held[RPT][NC];
    load_held(x, p, held);
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
    fold_groups(red, group_mean);
    const u64 first = (u64)p.chunk * ROWS;
    const float count = (float)(PIXELS - first < ROWS ? PIXELS - first : ROWS) * (float)D, inverse = 1.0f / count;
#pragma unroll
    for (int q = 0; q < NC; q++) {
        float mean[ACC];
#pragma unroll
        for (int i = 0; i < ACC; i++) {
            a[q][i] = 0.0f;
            mean[i] = COLUMN(p, q) ? group_mean[group_of((p.tx + q * TX) * V + i)] * inverse : 0.0f;
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
    fold_groups(red, group_m2);
    for (u32 g = threadIdx.x; g < KG; g += T) {
        float* to = parts + (((p.n * G + p.slice * KG + g) * CHUNKS) + p.chunk) * 2;
        to[0] = group_mean[g] * inverse;
        to[1] = group_m2[g];
    }
}

// One wave per (sample, group).
extern "C" __global__ __launch_bounds__(256) void group_norm_merge(const float* __restrict__ parts, float* __restrict__ stats,
                                                                  float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    const u64 of = (u64)blockIdx.x * 4 + (threadIdx.x >> 6);
    const u32 lane = threadIdx.x & 63u;
    const bool mine = of < (u64)BATCH * G;
    const float* from = parts + (mine ? of : 0) * CHUNKS * 2;
    const float whole = (float)PIXELS * (float)D;
    float s = 0.0f;
    for (u32 c = lane; c < CHUNKS; c += 64) {
        const u64 left = PIXELS - (u64)c * ROWS;
        s += from[c * 2] * ((float)(left < ROWS ? left : ROWS) * (float)D / whole);
    }
    for (int m = 32; m > 0; m /= 2) s += __shfl_xor(s, m, 64);
    float m2 = 0.0f;
    for (u32 c = lane; c < CHUNKS; c += 64) {
        const u64 left = PIXELS - (u64)c * ROWS;
        const float d = from[c * 2] - s;
        m2 += from[c * 2 + 1] + d * d * ((float)(left < ROWS ? left : ROWS) * (float)D);
    }
    for (int m = 32; m > 0; m /= 2) m2 += __shfl_xor(m2, m, 64);
    if (mine && lane == 0) {
        const float rstd = 1.0f / sqrtf(m2 / whole + EPS);
        stats[of * 2] = s;
        stats[of * 2 + 1] = rstd;
        if (mean_out) mean_out[of] = s;
        if (rstd_out) rstd_out[of] = rstd;
    }
}

extern "C" __global__ __launch_bounds__(T) void group_norm_apply(const elem_t* __restrict__ x, const param_t* __restrict__ gamma,
                                                                 const param_t* __restrict__ beta, const float* __restrict__ stats,
                                                                 elem_t* __restrict__ y) {
    const Place p = place();
    vec_t held[RPT][NC];
    load_held(x, p, held);
    const u64 o = origin(p);
#pragma unroll
    for (int q = 0; q < NC; q++) {
        if (!COLUMN(p, q)) continue;
        float mean[ACC], scale[V], shift[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const u32 c = (p.tx + q * TX) * V + i;
            const float* st = stats + (p.n * G + p.slice * KG + group_of(c)) * 2;
            mean[i % ACC] = st[0];
            scale[i] = st[1] * (float)gamma[p.slice * SC + c];
            shift[i] = (float)beta[p.slice * SC + c];
        }
#pragma unroll
        for (int r = 0; r < RPT; r++)
            if (HELD(p, r, q)) {
                vec_t out;
#pragma unroll
                for (int i = 0; i < V; i++) AT(out, i) = (elem_t)activate(((float)AT(held[r][q], i) - mean[i % ACC]) * scale[i] + shift[i]);
                *(vec_t*)(y + o + (u64)r * TY * C + q * TX * V) = out;
            }
    }
}
)HIP";

// Gradients. With dz = dy act'(z), a sample's sums over its pixels, A_c = sum dz and B_c = sum dz xh, give everything: dbeta and
// dgamma are their sums over the samples, and a group's s1 = sum gamma_c A_c / M, s2 = sum gamma_c B_c / M are what
// dx = rstd (gamma_c dz - s1 - xh s2) takes away.
const char* kBackward = R"HIP(
struct Column { float mean[V], rstd[V], gamma[V], beta[V]; };
__device__ __forceinline__ void load_column(Column& k, const Place& p, int q, const param_t* __restrict__ gamma, const param_t* __restrict__ beta,
                                            const float* __restrict__ mean, const float* __restrict__ rstd) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        const u32 c = (p.tx + q * TX) * V + i;
        const u64 g = p.n * G + p.slice * KG + group_of(c);
        k.mean[i] = mean[g];
        k.rstd[i] = rstd[g];
        k.gamma[i] = (float)gamma[p.slice * SC + c];
        k.beta[i] = (float)beta[p.slice * SC + c];
    }
}

// parts: [batch * CHUNKS][2][C]
extern "C" __global__ __launch_bounds__(T) void group_norm_sums(const elem_t* __restrict__ dy, const elem_t* __restrict__ x,
                                                                const param_t* __restrict__ gamma, const param_t* __restrict__ beta,
                                                                const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                float* __restrict__ parts) {
    __shared__ float red[RED_ROWS * CV * V * 2];
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
                        const float xh = ((float)AT(hx[r][q], i) - k.mean[i]) * k.rstd[i];
                        const float dz = slope_times((float)AT(hd[r][q], i), xh * k.gamma[i] + k.beta[i]);
                        a[q][2 * i] += dz;
                        a[q][2 * i + 1] += dz * xh;
                    }
        }
    }
    fold_rows<2 * V>(a, p, red);
    for (u32 e = threadIdx.x; e < CV * V * 2; e += T) {
        float s = 0.0f;
        for (u32 row = 0; row < RED_ROWS; row++) s += red[row * (CV * V * 2) + e];
        parts[((p.n * CHUNKS + p.chunk) * 2 + (e & 1)) * C + p.slice * SC + (e >> 1)] = s;
    }
}

// The chunks of a sample joined: its channels' sums [batch][2][C], and s1, s2 of its groups [batch][G][2]. One wave per group.
extern "C" __global__ __launch_bounds__(256) void group_norm_fold(const float* __restrict__ parts, const param_t* __restrict__ gamma,
                                                                  float* __restrict__ samples, float* __restrict__ group_sums) {
    const u64 of = (u64)blockIdx.x * 4 + (threadIdx.x >> 6);
    const u32 lane = threadIdx.x & 63u;
    if (of >= (u64)BATCH * G) return;
    const u64 n = of / G;
    const u32 g = (u32)(of % G);
    float s1 = 0.0f, s2 = 0.0f;
    for (u32 c = g * D + lane; c < (g + 1) * D; c += 64) {
        float a = 0.0f, b = 0.0f;
        for (u32 k = 0; k < CHUNKS; k++) {
            a += parts[((n * CHUNKS + k) * 2) * C + c];
            b += parts[((n * CHUNKS + k) * 2 + 1) * C + c];
        }
        samples[(n * 2) * C + c] = a;
        samples[(n * 2 + 1) * C + c] = b;
        s1 += (float)gamma[c] * a;
        s2 += (float)gamma[c] * b;
    }
    for (int m = 32; m > 0; m /= 2) {
        s1 += __shfl_xor(s1, m, 64);
        s2 += __shfl_xor(s2, m, 64);
    }
    const float whole = (float)PIXELS * (float)D;
    if (lane == 0) {
        group_sums[of * 2] = s1 / whole;
        group_sums[of * 2 + 1] = s2 / whole;
    }
}

// The workgroups behind the tensor's own add up the samples' sums: 64 channels each, a quarter of the samples per wave.
__device__ __forceinline__ void parameter_gradients(u64 block, const float* __restrict__ samples, float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float part[2][T / 64][64];
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u64 c = block * 64 + lane;
    float a = 0.0f, b = 0.0f;
    if (c < C)
        for (u64 n = wave; n < BATCH; n += T / 64) {
            a += samples[(n * 2) * C + c];
            b += samples[(n * 2 + 1) * C + c];
        }
    part[0][wave][lane] = a;
    part[1][wave][lane] = b;
    __syncthreads();
    if (wave == 0 && c < C) {
        for (u32 w = 1; w < T / 64; w++) {
            a += part[0][w][lane];
            b += part[1][w][lane];
        }
        dbeta[c] = a;
        dgamma[c] = b;
    }
}

extern "C" __global__ __launch_bounds__(T) void group_norm_gradient(const elem_t* __restrict__ dy, const elem_t* __restrict__ x,
                                                                    const param_t* __restrict__ gamma, const param_t* __restrict__ beta,
                                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                    const float* __restrict__ samples, const float* __restrict__ group_sums,
                                                                    elem_t* __restrict__ dx, float* __restrict__ dgamma, float* __restrict__ dbeta) {
    if (blockIdx.x >= BLOCKS) return parameter_gradients(blockIdx.x - BLOCKS, samples, dgamma, dbeta);
    const Place p = place();
    vec_t hx[RPT][NC], hd[RPT][NC];
    load_held(x, p, hx);
    load_held(dy, p, hd);
    const u64 o = origin(p);
#pragma unroll
    for (int q = 0; q < NC; q++) {
        if (p.ty >= TY || !COLUMN(p, q)) continue;
        Column k;
        load_column(k, p, q, gamma, beta, mean, rstd);
        float s1[V], s2[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const u64 g = p.n * G + p.slice * KG + group_of((p.tx + q * TX) * V + i);
            s1[i] = group_sums[g * 2];
            s2[i] = group_sums[g * 2 + 1];
        }
#pragma unroll
        for (int r = 0; r < RPT; r++)
            if (HELD(p, r, q)) {
                vec_t out;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float xh = ((float)AT(hx[r][q], i) - k.mean[i]) * k.rstd[i];
                    const float dz = slope_times((float)AT(hd[r][q], i), xh * k.gamma[i] + k.beta[i]);
                    AT(out, i) = (elem_t)(k.rstd[i] * (k.gamma[i] * dz - s1[i] - xh * s2[i]));
                }
                *(vec_t*)(dx + o + (u64)r * TY * C + q * TX * V) = out;
            }
    }
}
)HIP";

int pow2_floor(int64_t x) {
    int p = 1;
    while ((int64_t)p * 2 <= x && p < (1 << 30)) p *= 2;
    return p;
}

std::string definitions(const GroupNormProblem& pr, const GroupNormTiling& t) {
    const int64_t d = pr.channels / pr.groups;
    std::ostringstream s;
    s << "#define BATCH " << pr.batch << "ull\n#define PIXELS " << pr.pixels << "ull\n#define C " << pr.channels << "\n#define G " << pr.groups
      << "\n#define D " << d << "\n#define V " << t.vec << "\n#define T " << t.threads << "\n#define KG " << t.slice_groups << "\n#define SC "
      << t.slice << "\n#define SLICES " << pr.groups / t.slice_groups << "\n#define CV " << t.slice / t.vec << "\n#define TX " << t.tx
      << "\n#define TY " << t.ty << "\n#define NC " << t.columns << "\n#define RPT " << t.rows_per_thread << "\n#define ROWS " << t.rows()
      << "\n#define CHUNKS " << t.chunks << "\n#define BLOCKS " << t.grid << "ull\n#define LPG "
      << std::min(64, pow2_floor(t.threads / t.slice_groups)) << "\n#define BF16 " << (pr.dtype == HE_BF16) << "\n#define F16 "
      << (pr.dtype == HE_F16) << "\n#define PARAM_SAME " << (pr.param_dtype == pr.dtype) << "\n#define ACT " << pr.activation
      << "\n#define EPS " << strfmt("%.9gf", (double)pr.epsilon) << "\n";
    return s.str();
}

}  // namespace

std::string GroupNormTiling::describe() const {
    return strfmt("vec=%d threads=%d slice=%lld(%d groups) tx=%lld ty=%lld columns=%d rows_per_thread=%d chunks=%lld grid=%llu", vec, threads,
                  (long long)slice, slice_groups, (long long)tx, (long long)ty, columns, rows_per_thread, (long long)chunks, (unsigned long long)grid);
}

GroupNormTiling plan_group_norm(const GroupNormProblem& pr, bool backward) {
    GroupNormTiling t;
    const int esz = (int)dtype_bits(pr.dtype) / 8;
    const int64_t d = pr.channels / pr.groups;
    t.vec = 16 / esz;
    while (pr.channels % t.vec) t.vec /= 2;
    // The narrowest slice of whole groups and whole vectors that is at least 256 bytes of a pixel.
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
    // 64 registers of data per thread, fewer where that leaves compute units idle
    const int64_t vector_regs = std::max(1, t.vec * esz / 4) * (backward ? 2 : 1);
    int64_t rpt = std::max<int64_t>(1, 64 / (vector_regs * t.columns));
    const int64_t slices = pr.groups / t.slice_groups;
    while (rpt > 1 && (t.ty * (rpt / 2) >= pr.pixels || (uint64_t)(pr.batch * slices) * ((pr.pixels + t.ty * rpt - 1) / (t.ty * rpt)) < 1024)) rpt /= 2;
    t.rows_per_thread = (int)rpt;
    t.chunks = (pr.pixels + t.rows() - 1) / t.rows();
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
    // (kernels count channels, and vectors of LDS, in 32 bits)
    HE_REQUIRE(pr.channels <= 16384, HE_ERR_UNSUPPORTED, "group norm: %lld channels, at most 16384 are taken", (long long)pr.channels);
    HE_REQUIRE(pr.pixels <= (int64_t)1 << 40 && pr.batch <= (int64_t)1 << 31, HE_ERR_UNSUPPORTED, "group norm: extents too large");
    fwd_ = plan_group_norm(pr, false);
    bwd_ = plan_group_norm(pr, true);
    HE_REQUIRE(std::max(fwd_.grid, bwd_.grid) < (1ull << 31) - 16384, HE_ERR_UNSUPPORTED, "group norm: the tensor is too large for one launch");
    const std::string forward = definitions(pr, fwd_) + kCommon + kForward, backward = definitions(pr, bwd_) + kCommon + kBackward;
    auto make = [](const std::string& text, const char* entry) {
        return std::async(std::launch::async, [&text, entry] { return std::make_unique<JitKernel>(text, entry); });
    };
    auto f = make(forward, "group_norm_stats"), b = make(backward, "group_norm_sums");
    stats_ = f.get();
    sums_ = b.get();
    // (the other entries of the same texts: compiled already)
    merge_.reset(new JitKernel(forward, "group_norm_merge"));
    apply_.reset(new JitKernel(forward, "group_norm_apply"));
    fold_.reset(new JitKernel(backward, "group_norm_fold"));
    gradient_.reset(new JitKernel(backward, "group_norm_gradient"));
    const uint64_t rows = (uint64_t)pr.batch * pr.groups, sums = (uint64_t)pr.batch * 2 * pr.channels;
    scratch_floats_ = std::max(rows * 2 * (fwd_.chunks + 1), sums * (bwd_.chunks + 1) + rows * 2);
    source_ = forward + "\n" + backward;
    describe_ = "group_norm forward: " + fwd_.describe() + "\ngroup_norm backward: " + bwd_.describe();
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
    const uint64_t rows = (uint64_t)pr_.batch * pr_.groups;
    std::lock_guard<std::mutex> lk(mu_);
    float* parts = scratch_.get(scratch_floats_, 0, stream).floats;
    float* stats = parts + rows * fwd_.chunks * 2;
    const uint32_t grid[3] = {(uint32_t)fwd_.grid, 1, 1}, block[3] = {(uint32_t)fwd_.threads, 1, 1};
    const uint32_t merge_grid[3] = {(uint32_t)((rows + 3) / 4), 1, 1}, merge_block[3] = {256, 1, 1};
    void* a[] = {&x, &parts};
    stats_->launch(grid, block, 0, stream, a);
    void* b[] = {&parts, &stats, &mean, &rstd};
    merge_->launch(merge_grid, merge_block, 0, stream, b);
    void* c[] = {&x, &gamma, &beta, &stats, &y};
    apply_->launch(grid, block, 0, stream, c, true);
}

void GroupNorm::backward(const void* dy, const void* x, const void* gamma, const void* beta, const float* mean, const float* rstd, void* dx,
                         float* dgamma, float* dbeta, hipStream_t stream) {
    HE_REQUIRE(dgamma && dbeta, HE_ERR_INVALID, "group norm: the parameters' gradients are null");
    if (pr_.batch) {
        check({dy, x, dx}, {gamma, beta}, {mean, rstd, dgamma, dbeta});
        HE_REQUIRE(mean && rstd, HE_ERR_INVALID, "group norm: the backward pass needs the statistics of the forward pass");
    }
    const uint64_t rows = (uint64_t)pr_.batch * pr_.groups, sums = (uint64_t)pr_.batch * 2 * pr_.channels;
    std::lock_guard<std::mutex> lk(mu_);
    float* parts = scratch_.get(scratch_floats_, 0, stream).floats;
    float *samples = parts + sums * bwd_.chunks, *group_sums = samples + sums;
    const uint32_t block[3] = {(uint32_t)bwd_.threads, 1, 1};
    if (pr_.batch) {
        const uint32_t grid[3] = {(uint32_t)bwd_.grid, 1, 1};
        const uint32_t fold_grid[3] = {(uint32_t)((rows + 3) / 4), 1, 1}, fold_block[3] = {256, 1, 1};
        void* a[] = {&dy, &x, &gamma, &beta, &mean, &rstd, &parts};
        sums_->launch(grid, block, 0, stream, a);
        void* b[] = {&parts, &gamma, &samples, &group_sums};
        fold_->launch(fold_grid, fold_block, 0, stream, b);
    }
    // (without samples only the parameters' gradients are left, all zero)
    const uint32_t grid[3] = {(uint32_t)(bwd_.grid + (pr_.channels + 63) / 64), 1, 1};
    void* c[] = {&dy, &x, &gamma, &beta, &mean, &rstd, &samples, &group_sums, &dx, &dgamma, &dbeta};
    gradient_->launch(grid, block, 0, stream, c, true);
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
