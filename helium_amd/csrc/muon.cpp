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
struct Matrix {
    u32 rows, cols, mp, np;
    u32 tall, first_part, parts;
    float shape_scale;
    u64 x[2], xt[2][2], a[2], b[2];
};
struct Tile { u32 matrix, i, j; };
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

// The matrix that is orthogonalised, element by element: the operand itself, or the step's update from the gradient and the new momentum.
template <bool STEP> __device__ __forceinline__ float update_of(const Operands& o, u32 k, u64 e) {
    const float g = (float)o.in[k][e];
    if (!STEP) return g;
    const float m = o.new_momentum[k][e];
    return o.nesterov ? g + o.mu * m : m;
}
)HIP";

const char* kElements = R"HIP(
// Shares of |U|^2, in 64 bits: squares of f32 neither overflow nor vanish there. The step's first pass also writes the new momenta.
template <bool STEP> __device__ __forceinline__ void norm_part(const Matrix* __restrict__ mats, const Tile* __restrict__ parts, double* __restrict__ sums, const Operands& o) {
    __shared__ double wave_sums[4];
    const Tile t = parts[blockIdx.x];
    const u32 k = t.matrix - o.first;
    const u64 size = (u64)mats[t.matrix].rows * mats[t.matrix].cols, begin = (u64)t.i * PART, end = begin + PART < size ? begin + PART : size;
    double s = 0.0;
    for (u64 e = begin + threadIdx.x; e < end; e += 256) {
        float u = (float)o.in[k][e];
        if (STEP) {
            const float m = o.mu * o.momentum[k][e] + u;
            o.new_momentum[k][e] = m;
            u = o.nesterov ? u + o.mu * m : m;
        }
        s += (double)u * (double)u;
    }
    for (int m = 32; m > 0; m /= 2) s += SHFL_XOR_F64(s, m);
    if ((threadIdx.x & 63u) == 0) wave_sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) sums[blockIdx.x + t.j] = wave_sums[0] + wave_sums[1] + wave_sums[2] + wave_sums[3];
}

__device__ __forceinline__ void store_split(f16_t* __restrict__ high, f16_t* __restrict__ low, u64 at, float v, bool with_low) {
    const f16_t h = (f16_t)v;
    high[at] = h;
    if (with_low) low[at] = (f16_t)(v - (float)h);
}

// U / (|U| + floor) in f16 parts, in both orientations, zeros beyond the matrix. A block of 64 x 64.
template <bool STEP> __device__ __forceinline__ void convert_block(const Matrix* __restrict__ mats, const Tile* __restrict__ blocks, const double* __restrict__ sums, char* __restrict__ ws, const Operands& o) {
    __shared__ float tile[64][65];
    __shared__ double total;
    const Tile t = blocks[blockIdx.x];
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
    f16_t *nh = (f16_t*)(ws + (m.tall ? m.xt[0][0] : m.x[0])), *nl = (f16_t*)(ws + (m.tall ? m.xt[0][1] : m.x[1]));
    f16_t *th = (f16_t*)(ws + (m.tall ? m.x[0] : m.xt[0][0])), *tl = (f16_t*)(ws + (m.tall ? m.x[1] : m.xt[0][1]));
    const u32 c = t.j * 64 + lane;
    for (u32 i = wave; i < 64; i += 4) {
        const u32 r = t.i * 64 + i;
        float v = 0.0f;
        if (r < m.rows && c < m.cols) v = (float)((double)update_of<STEP>(o, k, (u64)r * m.cols + c) * scale);
        tile[i][lane] = v;
        store_split(nh, nl, (u64)r * cols_p + c, v, SPLIT || !m.tall);
    }
    __syncthreads();
    for (u32 i = wave; i < 64; i += 4) store_split(th, tl, (u64)(t.j * 64 + i) * rows_p + t.i * 64 + lane, tile[lane][i], SPLIT || m.tall);
}

template <bool STEP> __device__ __forceinline__ void finish_block(const Matrix* __restrict__ mats, const Tile* __restrict__ blocks, const char* __restrict__ ws, const Operands& o) {
    const Tile t = blocks[blockIdx.x];
    const Matrix& m = mats[t.matrix];
    const u32 k = t.matrix - o.first, cols_p = m.tall ? m.mp : m.np, c = t.j * 64 + (threadIdx.x & 63u);
    const f16_t *h = (const f16_t*)(ws + (m.tall ? m.xt[STEPS & 1][0] : m.x[0])), *l = (const f16_t*)(ws + (m.tall ? m.xt[STEPS & 1][1] : m.x[1]));
    for (u32 i = threadIdx.x >> 6; i < 64; i += 4) {
        const u32 r = t.i * 64 + i;
        if (r >= m.rows || c >= m.cols) continue;
        const u64 at = (u64)r * cols_p + c, e = (u64)r * m.cols + c;
        float v = (float)h[at];
        v += (float)l[at];
        v *= 1.0f / X_SCALE;
        if (STEP) {
            const float w = o.weight[k][e];
            ((float*)o.out[k])[e] = (w - o.learning_rate * o.weight_decay * w) - o.learning_rate * m.shape_scale * v;
        } else {
            ((elem_t*)o.out[k])[e] = (elem_t)v;
        }
    }
}

extern "C" __global__ __launch_bounds__(256) void muon_norm(const Matrix* __restrict__ mats, const Tile* __restrict__ parts, double* __restrict__ sums, Operands o) { norm_part<false>(mats, parts, sums, o); }
extern "C" __global__ __launch_bounds__(256) void muon_norm_step(const Matrix* __restrict__ mats, const Tile* __restrict__ parts, double* __restrict__ sums, Operands o) { norm_part<true>(mats, parts, sums, o); }
extern "C" __global__ __launch_bounds__(256) void muon_convert(const Matrix* __restrict__ mats, const Tile* __restrict__ blocks, const double* __restrict__ sums, char* __restrict__ ws, Operands o) { convert_block<false>(mats, blocks, sums, ws, o); }
extern "C" __global__ __launch_bounds__(256) void muon_convert_step(const Matrix* __restrict__ mats, const Tile* __restrict__ blocks, const double* __restrict__ sums, char* __restrict__ ws, Operands o) { convert_block<true>(mats, blocks, sums, ws, o); }
extern "C" __global__ __launch_bounds__(256) void muon_finish(const Matrix* __restrict__ mats, const Tile* __restrict__ blocks, const char* __restrict__ ws, Operands o) { finish_block<false>(mats, blocks, ws, o); }
extern "C" __global__ __launch_bounds__(256) void muon_finish_step(const Matrix* __restrict__ mats, const Tile* __restrict__ blocks, const char* __restrict__ ws, Operands o) { finish_block<true>(mats, blocks, ws, o); }
)HIP";

// One kernel for the three products of a step, each of the form R = alpha P Q^T + beta E with P, Q row-major and contiguous along the
// sum (X and its transpose are both kept for that; A and B are symmetric):
//   gram    A = X X^T           P = Q = X            lower tiles, stored twice
//   square  B = b A + c A A     P = Q = A, E = A     lower tiles, stored twice
//   apply   X = a X + B X       P = B, Q = XT, E = X  whole, stored as X and as XT
const char* kProduct = R"HIP(
#define BM TILE
#define BN TILE
#define BK 64
#define WAVES (WAVES_M * WAVES_N)
#define WTM (BM / WAVES_M)
#define WTN (BN / WAVES_N)
#define MB (WTM / 32)
#define NB (WTN / 32)
#define STAGE_HALVES ((BM + BN) * BK)
#define LOADS ((BM + BN) / 8 / WAVES)   /* direct loads of a wave per k-tile: 8 rows of 128 bytes each */
#define STRIP_PITCH 72                  /* of a wave's 64 x 64 strip in LDS, in halves: rows stay 16-byte aligned */
enum { GRAM, SQUARE, APPLY };

// Waits until this wave's direct loads have landed, then for the other waves'.
__device__ __forceinline__ void tile_ready() {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
}

template <int STAGE> __device__ __forceinline__ void product(const Matrix* __restrict__ mats, const Tile* __restrict__ tiles, char* __restrict__ ws, u32 turn) {
    __shared__ __attribute__((aligned(16))) f16_t lds[2 * STAGE_HALVES];
    const Tile t = tiles[blockIdx.x];
    const Matrix& m = mats[t.matrix];
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave_m = wave / WAVES_N, wave_n = wave % WAVES_N;
    const u32 k_len = STAGE == GRAM ? m.np : m.mp, k_tiles = k_len / BK;
    const f16_t *p_plane[2], *q_plane[2];
#pragma unroll
    for (int part = 0; part < 2; part++) {
        p_plane[part] = (const f16_t*)(ws + (STAGE == GRAM ? m.x[part] : STAGE == SQUARE ? m.a[part] : m.b[part])) + (u64)t.i * BM * k_len;
        q_plane[part] = (const f16_t*)(ws + (STAGE == GRAM ? m.x[part] : STAGE == SQUARE ? m.a[part] : m.xt[turn][part])) + (u64)t.j * BN * k_len;
    }
    // Direct loads: lane l of the load of rows 8 r .. 8 r + 7 takes row l / 8 and, so that fragment reads of 8 neighbouring rows
    // meet 8 different bank groups, the chunk (l % 8) ^ (l / 8) of its 128 bytes.
    const u32 lane_off = (lane >> 3) * k_len + (((lane & 7u) ^ (lane >> 3)) << 3);
    // (parts: high x high, high x low, low x high)
    const u32 all = SPLIT ? 3 * k_tiles : k_tiles;
    auto fetch = [&](u32 kt, u32 slot) {
        const u32 pass = SPLIT ? kt / k_tiles : 0, k0 = (kt - pass * k_tiles) * BK;
        const f16_t *p = p_plane[pass == 2], *q = q_plane[pass == 1];
        f16_t* base = lds + slot * STAGE_HALVES;
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const u32 row = (wave * LOADS + l) * 8;   // of P's rows, then Q's
            const f16_t* src = (row < BM ? p + (u64)row * k_len : q + (u64)(row - BM) * k_len) + k0 + lane_off;
            __builtin_amdgcn_global_load_lds((const GLOBAL_AS u32*)src, (LDS_AS u32*)(base + row * BK), 16, 0, 0);
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
    fetch(0, 0);
    for (u32 kt = 0; kt < all; kt++) {
        tile_ready();
        if (kt + 1 < all) fetch(kt + 1, (kt + 1) & 1u);
        const f16_t *p = lds + (kt & 1u) * STAGE_HALVES + (wave_m * WTM + frag_row) * BK, *q = lds + (kt & 1u) * STAGE_HALVES + (BM + wave_n * WTN + frag_row) * BK;
#pragma unroll
        for (int kk = 0; kk < BK / 16; kk++) {
            f16x8 a[MB], b[NB];
            const u32 chunk = ((kk * 2 + half) ^ swz) * 8;
#pragma unroll
            for (int i = 0; i < MB; i++) a[i] = *(const f16x8*)(p + i * 32 * BK + chunk);
#pragma unroll
            for (int j = 0; j < NB; j++) b[j] = *(const f16x8*)(q + j * 32 * BK + chunk);
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int j = 0; j < NB; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    }
    __syncthreads();   // the operand stages become the waves' strips

    // Results: a lane holds rows (e / 4) * 8 + half * 4 + e % 4 of column lane % 32 of each 32 x 32 block. Strips of 64 x 64 go through
    // LDS into whole rows, once as they are and once transposed.
    const u32 out_pitch = STAGE == APPLY ? m.np : m.mp;
    f16_t* strip = lds + wave * 64 * STRIP_PITCH;
    const u64 row0 = (u64)t.i * BM + wave_m * WTM, col0 = (u64)t.j * BN + wave_n * WTN;
    const bool mirrored = STAGE == APPLY || t.i != t.j;
#pragma unroll
    for (int i = 0; i < MB; i += 2)
#pragma unroll
        for (int j = 0; j < NB; j += 2) {
            float v[2][2][16];
#pragma unroll
            for (int di = 0; di < 2; di++)
#pragma unroll
                for (int dj = 0; dj < 2; dj++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float s = acc[i + di][j + dj][e];
                        if (STAGE == GRAM) {
                            v[di][dj][e] = s * (A_SCALE / (X_SCALE * X_SCALE));
                            continue;
                        }
                        const u64 at = (row0 + (i + di) * 32 + (e / 4) * 8 + half * 4 + e % 4) * out_pitch + col0 + (j + dj) * 32 + frag_row;
                        float other = (float)((const f16_t*)(ws + (STAGE == SQUARE ? m.a[0] : m.x[0])))[at];
                        // (of X the low part counts in either precision: what f16 drops of a X in each step would stay dropped, and
                        // the small singular values with it)
                        if (SPLIT || STAGE == APPLY) other += (float)((const f16_t*)(ws + (STAGE == SQUARE ? m.a[1] : m.x[1])))[at];
                        v[di][dj][e] = STAGE == SQUARE ? NS_B * other + (NS_C * B_SCALE / (A_SCALE * A_SCALE)) * s : NS_A * other + (1.0f / B_SCALE) * s;
                    }
#pragma unroll
            for (int part = 0; part < 2; part++) {
                const bool keep_plain = SPLIT || part == 0 || STAGE == APPLY, keep_mirror = mirrored && (SPLIT || part == 0 || STAGE == APPLY);
                if (!keep_plain) continue;
                f16_t *plain = (f16_t*)(ws + (STAGE == GRAM ? m.a[part] : STAGE == SQUARE ? m.b[part] : m.x[part]));
                f16_t *mirror = (f16_t*)(ws + (STAGE == GRAM ? m.a[part] : STAGE == SQUARE ? m.b[part] : m.xt[turn ^ 1u][part]));
#pragma unroll
                for (int way = 0; way < 2; way++) {
                    if (way == 1 && !keep_mirror) continue;
                    __syncthreads();
#pragma unroll
                    for (int di = 0; di < 2; di++)
#pragma unroll
                        for (int dj = 0; dj < 2; dj++)
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                const u32 r = di * 32 + (e / 4) * 8 + half * 4 + e % 4, c = dj * 32 + frag_row;
                                const f16_t high = (f16_t)v[di][dj][e];
                                strip[way ? c * STRIP_PITCH + r : r * STRIP_PITCH + c] = part ? (f16_t)(v[di][dj][e] - (float)high) : high;
                            }
                    __syncthreads();
                    f16_t* to = way ? mirror + (col0 + j * 32) * (STAGE == APPLY ? m.mp : m.mp) + row0 + i * 32 : plain + (row0 + i * 32) * out_pitch + col0 + j * 32;
                    const u32 pitch = way ? m.mp : out_pitch;
#pragma unroll
                    for (int s = 0; s < 8; s++) {
                        const u32 r = s * 8 + (lane >> 3), c = (lane & 7u) * 8;
                        *(u32x4*)(to + (u64)r * pitch + c) = *(const u32x4*)(strip + r * STRIP_PITCH + c);
                    }
                }
            }
        }
}

extern "C" __global__ __launch_bounds__(WAVES * 64) void muon_gram(const Matrix* __restrict__ mats, const Tile* __restrict__ tiles, char* __restrict__ ws, u32 turn) { product<GRAM>(mats, tiles, ws, turn); }
extern "C" __global__ __launch_bounds__(WAVES * 64) void muon_square(const Matrix* __restrict__ mats, const Tile* __restrict__ tiles, char* __restrict__ ws, u32 turn) { product<SQUARE>(mats, tiles, ws, turn); }
extern "C" __global__ __launch_bounds__(WAVES * 64) void muon_apply(const Matrix* __restrict__ mats, const Tile* __restrict__ tiles, char* __restrict__ ws, u32 turn) { product<APPLY>(mats, tiles, ws, turn); }
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

// Tiles in the order of their blocks: blocks are dealt round-robin to the 8 XCDs, each with an L2 of its own, so XCD x gets the
// x-th eighth of a sequence in which neighbours share rows and columns.
void deal(std::vector<MuonTile>& tiles) {
    const size_t n = tiles.size(), whole = n / 8, over = n % 8;
    std::vector<MuonTile> out(n);
    for (size_t b = 0; b < n; b++) {
        const size_t x = b % 8;
        out[b] = tiles[x * whole + std::min(x, over) + b / 8];
    }
    tiles.swap(out);
}

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
    const uint32_t tile = 128;
    uint64_t at = 0, parts = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    std::vector<MuonTile> lower, whole, shares, blocks;
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
        const uint64_t x = (uint64_t)m.mp * m.np * 2, a = (uint64_t)m.mp * m.mp * 2;
        for (int part = 0; part < 2; part++) {
            m.x[part] = take(x);  // (its low part counts in either precision; the transpose's does where the result is tall)
            for (int turn = 0; turn < 2; turn++) m.xt[turn][part] = take(x);
            if (part == 0 || pr.split) m.a[part] = take(a), m.b[part] = take(a);
        }
        const uint32_t ti = m.mp / tile, tj = m.np / tile;
        for (uint32_t g = 0; g < ti; g += 4)  // bands of four tile rows, column by column
            for (uint32_t j = 0; j < std::max(ti, tj); j++)
                for (uint32_t i = g; i < std::min(g + 4, ti); i++) {
                    if (j < tj) whole.push_back({(uint32_t)k, i, j});
                    if (j <= i) lower.push_back({(uint32_t)k, i, j});
                }
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
    deal(lower);
    deal(whole);
    // (a share's place among the sums is its block's, plus where its launch begins)
    for (size_t k = 0; k < pr.shapes.size(); k++)
        for (uint32_t p = part_begin_[k]; p < part_begin_[k + 1]; p++) shares[p].j = part_begin_[k / kGroup * kGroup];
    workspace_bytes_ = take(parts * sizeof(double)) + parts * sizeof(double);
    tables_[0] = bytes_of(matrices_), tables_[1] = bytes_of(lower), tables_[2] = bytes_of(whole), tables_[3] = bytes_of(shares), tables_[4] = bytes_of(blocks);
    table_size_ = {(uint32_t)matrices_.size(), (uint32_t)lower.size(), (uint32_t)whole.size(), (uint32_t)shares.size(), (uint32_t)blocks.size()};
    for (int t = 0; t < 5; t++) {
        table_at_[t] = table_bytes_;
        table_bytes_ += (tables_[t].size() + 255) / 256 * 256;
    }
    const int waves_m = 2, waves_n = 2;
    std::ostringstream s;
    s << "#define GROUP " << kGroup << "\n#define PART " << kPart << "ull\n#define STEPS " << pr.steps << "\n#define SPLIT " << (int)pr.split << "\n#define BF16 "
      << (pr.dtype == HE_BF16) << "\n#define F16 " << (pr.dtype == HE_F16) << "\n#define NORM_FLOOR 1e-7\n#define TILE " << tile << "\n#define WAVES_M " << waves_m
      << "\n#define WAVES_N " << waves_n << "\n#ifndef SHFL_XOR_F64\n#define SHFL_XOR_F64(v, m) __shfl_xor(v, m, 64)\n#endif\n";
    source_ = s.str() + kCommon + kElements + kProduct;
    auto make = [&](const char* entry) { return std::make_unique<JitKernel>(source_, entry); };
    norm_ = make("muon_norm"), convert_ = make("muon_convert"), finish_ = make("muon_finish");
    norm_step_ = make("muon_norm_step"), convert_step_ = make("muon_convert_step"), finish_step_ = make("muon_finish_step");
    gram_ = make("muon_gram"), square_ = make("muon_square"), apply_ = make("muon_apply");
    describe_ = strfmt("muon matrices=%zu steps=%d parts=%d tile=%u threads=%d lower=%u whole=%u shares=%u blocks=%u workspace=%zu", pr.shapes.size(), pr.steps,
                       pr.split ? 2 : 1, tile, waves_m * waves_n * 64, table_size_[1], table_size_[2], table_size_[3], table_size_[4], workspace_bytes_);
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
    for (int t = 0; t < 5 && e == hipSuccess; t++) e = hipMemcpy(b.tables + table_at_[t], tables_[t].data(), tables_[t].size(), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        (void)hipFree(b.tables);
        (void)hipFree(b.workspace);
        fail(HE_ERR_HIP, strfmt("muon: %zu bytes of workspace: %s", workspace_bytes_, hipGetErrorString(e)));
    }
    per_stream_[stream] = b;
    return b;
}

void Muon::products(char* ws, char* tables, hipStream_t stream) {
    const uint32_t block[3] = {256, 1, 1}, lower[3] = {table_size_[1], 1, 1}, whole[3] = {table_size_[2], 1, 1};
    char *mats = tables + table_at_[0], *lower_tiles = tables + table_at_[1], *whole_tiles = tables + table_at_[2];
    for (int k = 0; k < pr_.steps; k++) {
        uint32_t turn = (uint32_t)k & 1u;
        void *sym[] = {&mats, &lower_tiles, &ws, &turn}, *all[] = {&mats, &whole_tiles, &ws, &turn};
        gram_->launch(lower, block, 0, stream, sym);
        square_->launch(lower, block, 0, stream, sym);
        apply_->launch(whole, block, 0, stream, all);
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
    double* sums = (double*)(ws + workspace_bytes_ - table_size_[3] * sizeof(double));
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
        char* parts = b.tables + table_at_[3] + part_begin_[first] * sizeof(MuonTile);
        const uint32_t grid[3] = {part_begin_[last] - part_begin_[first], 1, 1};
        void* args[] = {&mats, &parts, &sums, &o};
        (how ? norm_step_ : norm_)->launch(grid, block, 0, stream, args);
    });
    each_group([&](OperandsArg& o, size_t first, size_t last) {
        char* blocks = b.tables + table_at_[4] + block_begin_[first] * sizeof(MuonTile);
        const uint32_t grid[3] = {block_begin_[last] - block_begin_[first], 1, 1};
        void* args[] = {&mats, &blocks, &sums, &ws, &o};
        (how ? convert_step_ : convert_)->launch(grid, block, 0, stream, args);
    });
    products(ws, b.tables, stream);
    each_group([&](OperandsArg& o, size_t first, size_t last) {
        char* blocks = b.tables + table_at_[4] + block_begin_[first] * sizeof(MuonTile);
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
        HE_REQUIRE(muon && bytes && which >= 0 && which < 5 && (data || capacity == 0), HE_ERR_INVALID, "bad argument");
        const std::vector<char>& t = muon->impl.table(which);
        *bytes = t.size();
        if (capacity) memcpy(data, t.data(), std::min(capacity, t.size()));
    });
}

}  // extern "C"
