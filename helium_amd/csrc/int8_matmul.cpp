#include "int8_matmul.h"

#include <algorithm>
#include <cmath>
#include <future>
#include <map>
#include <sstream>

#include "rms_norm.h"

namespace he {

namespace {

// ---- device text ---------------------------------------------------------------------------------------------------
// y[t][n] = (sum over k of x[t][k] w[n][k]) x_scale[t] w_scale[n] + bias[n]. The sums are whole numbers in 32 bits and exact (fewer than 2^17
// products of at most 2^14), so that no cut of a sum changes a result. The definitions ahead of the text hold the type of the result (BF16, F16)
// and the shape: of tiles TN, TM, WAVES_N, WAVES_M, STAGES, AHEAD; of streams BN, BM, WAVES, STEPS (of 64 bytes of k, on their way at a time, twice).
//
// Weights are the instruction's rows and tokens its columns: a lane then has four neighbouring channels of one token at a time.
const char* kCommon = R"HIP(
typedef unsigned char u8;
typedef unsigned short u16;
typedef unsigned int u32;
typedef unsigned long long u64;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
#if BF16
typedef __bf16 out_t;
#elif F16
typedef _Float16 out_t;
#else
typedef float out_t;
#endif
typedef out_t out4 __attribute__((ext_vector_type(4)));
#define PER (16 / (int)sizeof(out_t))
typedef out_t out_v __attribute__((ext_vector_type(PER)));
// (rows of y begin where the row before ends: at any whole value)
typedef out_t out_any __attribute__((ext_vector_type(PER), aligned(sizeof(out_t))));
#ifndef MFMA_32
#define MFMA_32(a, b, c) __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0)
#define MFMA_16(a, b, c) __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0)
#define LDS_AS __attribute__((address_space(3)))
#define GLOBAL_AS __attribute__((address_space(1)))
#define AS_F32(f) asm("" : "+v"(f))
#else
#define AS_F32(f)
#endif
struct Call {
    const u8 *x, *w;
    const float *x_scales, *w_scales, *bias;
    out_t* y;
    u32 tokens, channels, pitch;   // pitch: bytes of an operand's row
    u32 blocks, shares;            // of one share; a share's sums wait in `parked`, rows of `parked_pitch` channels, for the launch that adds them up
    u32 parked_pitch;
    int* parked;
};
__device__ __forceinline__ i32x4* parked_at(const Call& c, u32 share, u32 m, u32 n) {
    return (i32x4*)(c.parked + ((u64)share * c.tokens + m) * c.parked_pitch + n);
}
// One rounding of the sum to f32, one of its product with the token's scale, one with the channel's and the bias added, and that to the result's type: the same
// in every shape and cut. (To f16 the compiler would take the last two as one where it can, some channels of a tile among them.)
__device__ __forceinline__ float scaled(int sum, float x_scale, float w_scale, float bias) {
    float f = __builtin_fmaf((float)sum * x_scale, w_scale, bias);
#if F16
    AS_F32(f);
#endif
    return f;
}
typedef out_t out4_any __attribute__((ext_vector_type(4), aligned(sizeof(out_t))));
struct Scales { float x, w[4], bias[4]; };   // of a token and four channels, of which the last may be missing
__device__ __forceinline__ Scales scales_of(const Call& c, u32 m, u32 n) {
    Scales s;
    s.x = c.x_scales[m < c.tokens ? m : c.tokens - 1];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const u32 of = n + k < c.channels ? n + k : c.channels - 1;
        s.w[k] = c.w_scales[of];
        s.bias[k] = c.bias ? c.bias[of] : 0.0f;
    }
    return s;
}
__device__ __forceinline__ void store_four(const Call& c, u32 m, u32 n, i32x4 sum, const Scales& s) {
    out_t* to = c.y + (u64)m * c.channels + n;
    out4_any out;
#pragma unroll
    for (int k = 0; k < 4; k++) out[k] = (out_t)scaled(sum[k], s.x, s.w[k], s.bias[k]);
    if (n + 4 <= c.channels) *(out4_any*)to = out;
    else
#pragma unroll
        for (u32 k = 0; k < 4; k++)
            if (n + k < c.channels) to[k] = out[k];
}
)HIP";

// Tiles. Rows of 128 bytes of k go from memory straight into a ring of STAGES k-tiles in LDS and from there, 16 bytes to a lane, into the
// matrix instructions (32 x 32 x 32).
//
// 256 x 256: 4096 x 4096 x 4096 62 us (2220 TOPS), 8192 x 8192 x 8192 449 (2450). The instructions alone, on zeros, take 25 us of the 62, on numbers like the
// operands' 40: the card lowers its clock under them. Loads alone take 39, reads of LDS 10; without the reads it is 62 as well, without the loads 55; some
// 10 us are beginning and end, where results leave that no sums hide. Waves of 64 x 128, four along the channels or two, 62 us, four waves of
// 128 x 128 65; tiles of 128 x 256 70, 192 x 192 77.
const char* kTile = R"HIP(
#define WTN (TN / WAVES_N)
#define WTM (TM / WAVES_M)
#define NB (WTN / 32)
#define MB (WTM / 32)
#define ROW 128
#define STAGE_BYTES ((TN + TM) * ROW)
#define LOADS ((TN + TM) / 8 / (WAVES_N * WAVES_M))
#define READS (NB + MB)
#define MMAS (NB * MB)
#define WAIT_LOADS(n) (0x0070 | ((n) & 15) | (((n) >> 4) << 14))   /* vmcnt(n), and lgkmcnt(0): this wave's reads of LDS are done */
// a wave's strip of 32 tokens; two rows are apart by what a token's pair of lanes writes, so that they meet different banks
#define STRIP_PITCH (WTN + 8)
#define STRIP_VALUES (32 * STRIP_PITCH)
#define STRIPS ((WAVES_N * WAVES_M + STAGES - 1) / STAGES)   /* in a stage's room */
static_assert(STRIPS * STRIP_VALUES * sizeof(out_t) <= STAGE_BYTES, "");

struct Fragments { i32x4 w[NB], x[MB]; };

// What a wave stores of its sums: 32 tokens at a time through its strip, so that whole vectors of channels go out.
__device__ __forceinline__ void store_sums(const i32x16 (&acc)[NB][MB], const Call& c, u32 n0, u32 m0, const float (&x_scales)[MB], const float* w_scales, const float* bias, out_t* strip) {
    const u32 lane = threadIdx.x & 63u, half = lane >> 5;
    const bool past = (u64)c.tokens * c.channels >= (1u << 21);   // (results of 4 MB and more bypass the caches: 4096 x 4096 x 4096 67.5 -> 66.5 us)
#pragma unroll
    for (int j = 0; j < MB; j++) {
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32 n = i * 32 + e * 8 + half * 4;
                const f32x4 ws = *(const f32x4*)(w_scales + n), b = *(const f32x4*)(bias + n);
                out4 out;
#pragma unroll
                for (int k = 0; k < 4; k++) out[k] = (out_t)scaled(acc[i][j][e * 4 + k], x_scales[j], ws[k], b[k]);
                *(out4*)(strip + (lane & 31u) * STRIP_PITCH + n) = out;
            }
        // (the strip is the wave's own: what it wrote is there when its LDS accesses are done, which the reads' own waits see to)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        constexpr u32 lanes = WTN / PER;   // of a token
#pragma unroll
        for (u32 s = 0; s < 32 * lanes / 64; s++) {
            const u32 token = s * (64 / lanes) + lane / lanes, n = lane % lanes * PER;
            const out_v out = *(const out_v*)(strip + token * STRIP_PITCH + n);
            if (m0 + j * 32 + token >= c.tokens) continue;
            out_t* to = c.y + (u64)(m0 + j * 32 + token) * c.channels + n0 + n;
            if (n0 + n + PER > c.channels) {
#pragma unroll
                for (u32 k = 0; k < PER; k++)
                    if (n0 + n + k < c.channels) to[k] = out[k];
            } else if (past) __builtin_nontemporal_store(out, (out_any*)to);
            else *(out_any*)to = out;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}
// Which tile a block makes. Blocks are dealt to the 8 XCDs in turn, each with an L2 of its own: an XCD takes neighbours, in groups of
// four rows of tiles, whose weights and tokens they share.
__device__ __forceinline__ void place(const Call& c, u32& tn, u32& tm) {
    const u32 tiles_n = (c.channels + TN - 1) / TN, tiles_m = (c.tokens + TM - 1) / TM, xcd = blockIdx.x % 8u;
    const u32 t = xcd * (c.blocks / 8u) + (xcd < c.blocks % 8u ? xcd : c.blocks % 8u) + blockIdx.x / 8u;
    const u32 group = t / (4 * tiles_n), in = t % (4 * tiles_n), high = tiles_m - group * 4 < 4 ? tiles_m - group * 4 : 4;
    tm = group * 4 + in % high;
    tn = in / high;
}

// What a wave fetches of a k-tile. Direct loads: lane l of the load of rows 8 r .. 8 r + 7 takes row l / 8 and, so that fragment reads meet different
// banks, the chunk (l % 8) ^ (row / 2 % 8) of its 128 bytes: two rows fill the 64 banks, so rows two apart must differ. (A tile that ends beyond an
// operand loads its last row there: sums that nothing stores. Behind a row's end its last chunk is loaded once more: what is read there of the tokens
// counts as zeros.)
struct Source { u32 wave, chunks, off[LOADS], chunk[2]; };
// What it reads of a stage: the first of its rows of weights and of tokens, its half of a k-step's chunks, and where those lie.
struct Reader { u32 w_at, x_at, half, swz; };
__device__ __forceinline__ void fetch(u8* stage, const u8* w, const u8* x, const Source& s, u32 kt) {
    u32 behind[2];   // by how many chunks a lane's lies behind the row's last, which it loads then
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const u32 last = s.chunks - 1, mine = kt * 8 + s.chunk[e];
        behind[e] = mine > last ? mine - last : 0;
    }
#pragma unroll
    for (int l = 0; l < LOADS; l++) {
        const u32 row = (s.wave * LOADS + l) * 8;   // of the weights, then of the tokens
        const u8* src = (row < TN ? w : x) + (u64)kt * ROW + (s.off[l] - behind[l & 1] * 16);
        __builtin_amdgcn_global_load_lds((const GLOBAL_AS u32*)src, (LDS_AS u32*)(stage + row * ROW), 16, 0, 0);
    }
}
__device__ __forceinline__ void read(const u8* stage, const Reader& r, int kk, Fragments& g, bool whole, u32 chunks_left) {
    const u8 *w = stage + r.w_at, *x = stage + r.x_at;
    const u32 at = ((kk * 2 + r.half) ^ r.swz) * 16;
#pragma unroll
    for (int i = 0; i < NB; i++) g.w[i] = *(const i32x4*)(w + i * 32 * ROW + at);
#pragma unroll
    for (int j = 0; j < MB; j++) {
        g.x[j] = *(const i32x4*)(x + j * 32 * ROW + at);
        if (!whole && kk * 2 + r.half >= chunks_left) g.x[j] = i32x4{0, 0, 0, 0};
    }
}
__device__ __forceinline__ void multiply(const Fragments& g, i32x16 (&acc)[NB][MB]) {
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) acc[i][j] = MFMA_32(g.w[i], g.x[j], acc[i][j]);
}
// One k-tile, from `from`; the one to come goes to `to`. The loop is rotated by AHEAD k-steps: the matrix instructions that the last k-tile left over cover
// the barrier's way, the first reads of this one and the loads of the one to come; the reads of further steps are issued between the instructions of
// those before. The order is asked for, since the compiler by itself reads, waits and multiplies in turn.
//
// Each stage is an array of its own, and the calls of a round of the ring name theirs: only so does the compiler know that a direct load does not write where
// a read looks. Otherwise it has the reads wait for all loads that are on their way: 4096 x 4096 x 4096 66 us for 62, 512 x 4096 x 4096 17.9 for 14.7.
template <bool MORE> __device__ __forceinline__ void k_tile(const u8* from, u8* to, const u8* w, const u8* x, const Source& s, const Reader& r, u32 kt, Fragments (&f)[2][AHEAD],
                                                           i32x16 (&acc)[NB][MB]) {
    // This wave's loads of the k-tile have landed (those of the STAGES - 2 behind it may be on their way), then the other waves'. No wave still reads the
    // stage that is filled next. (The bare barrier: __syncthreads() would wait for all loads.)
    __builtin_amdgcn_s_waitcnt(WAIT_LOADS(MORE ? (STAGES - 2) * LOADS : 0));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int g = 0; g < 4 / AHEAD; g++) {
#pragma unroll
        for (int k = 0; k < AHEAD; k++) read(from, r, g * AHEAD + k, f[g & 1][k], MORE, s.chunks - kt * 8);
        if (g == 0 && MORE) fetch(to, w, x, s, kt + STAGES - 1);
#pragma unroll
        for (int k = 0; k < AHEAD; k++) multiply(f[(g & 1) ^ 1][k], acc);
        if (g == 0) {
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
            for (int n = 0; n < AHEAD * MMAS; n++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
                for (int l = n * LOADS / (AHEAD * MMAS); l < (n + 1) * LOADS / (AHEAD * MMAS); l++)
                    if (MORE) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            }
        } else {
#pragma unroll
            for (int n = 0; n < AHEAD * MMAS; n++) {
                // (reads behind the first instruction: the wait for its operands is for all reads before it)
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (n * 2 < AHEAD * READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                if (n * 2 + 1 < AHEAD * READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        }
    }
}

extern "C" __global__ __launch_bounds__(WAVES_N * WAVES_M * 64) KERNEL_ATTRS void int8_product(Call c) {
    __shared__ __attribute__((aligned(16))) u8 s0[STAGE_BYTES], s1[STAGE_BYTES];
#if STAGES > 2
    __shared__ __attribute__((aligned(16))) u8 s2[STAGE_BYTES];
#else
    u8* const s2 = s1;
#endif
#if STAGES > 3
    __shared__ __attribute__((aligned(16))) u8 s3[STAGE_BYTES];
#else
    u8* const s3 = s2;   // (the last)
#endif
    __shared__ __attribute__((aligned(16))) float w_scales[TN], bias[TN];
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave_n = wave / WAVES_M, wave_m = wave % WAVES_M;
    u32 tn, tm;
    place(c, tn, tm);
    const u32 n0 = tn * TN, m0 = tm * TM;
    const u32 k_tiles = (c.pitch + ROW - 1) / ROW, halvings = __builtin_ctz(c.shares);   // (shares are a power of two)
    const u32 k_begin = k_tiles * blockIdx.y >> halvings, k_end = k_tiles * (blockIdx.y + 1) >> halvings;
    const u8 *w = c.w + (u64)n0 * c.pitch, *x = c.x + (u64)m0 * c.pitch;
    Source source{wave, c.pitch / 16, {}, {(lane & 7u) ^ (lane >> 4), (lane & 7u) ^ (4u + (lane >> 4))}};
#pragma unroll
    for (int l = 0; l < LOADS; l++) {
        const u32 row = (wave * LOADS + l) * 8, of = row < TN ? row : row - TN, last = (row < TN ? c.channels - n0 : c.tokens - m0) - 1, mine = of + (lane >> 3);
        source.off[l] = (mine < last ? mine : last) * c.pitch + source.chunk[l & 1] * 16;
    }
    const u32 frag_row = lane & 31u, half = lane >> 5;
    const Reader reader{(wave_n * WTN + frag_row) * ROW, (TN + wave_m * WTM + frag_row) * ROW, half, lane >> 1 & 7u};
    i32x16 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
    Fragments f[2][AHEAD];
#pragma unroll
    for (int s = 0; s < AHEAD; s++) {
#pragma unroll
        for (int i = 0; i < NB; i++) f[1][s].w[i] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < MB; j++) f[1][s].x[j] = i32x4{0, 0, 0, 0};
    }
    // The scales and the bias, asked for before the k-tiles, so that nothing waits for them.
    const u32 n = n0 + threadIdx.x % TN, n_at = n < c.channels ? n : c.channels - 1;
    const float my_scale = c.w_scales[n_at], my_bias = c.bias ? c.bias[n_at] : 0.0f;
    float x_scales[MB];
#pragma unroll
    for (int j = 0; j < MB; j++) {
        const u32 m = m0 + wave_m * WTM + j * 32 + frag_row;
        x_scales[j] = c.x_scales[m < c.tokens ? m : c.tokens - 1];
    }
    // Whole rounds of the ring, each call with its own stages (see k_tile); what is left takes them as they come.
    const u32 k_count = k_end - k_begin, ahead = STAGES - 1 < k_count ? STAGES - 1 : k_count;
    u32 kt = k_begin;
    if (k_count >= 2 * STAGES - 1) {
        fetch(s0, w, x, source, kt);
        if (STAGES > 2) fetch(s1, w, x, source, kt + 1);
        if (STAGES > 3) fetch(s2, w, x, source, kt + 2);
        do {
            k_tile<true>(s0, s3, w, x, source, reader, kt, f, acc);
            k_tile<true>(s1, s0, w, x, source, reader, kt + 1, f, acc);
            if (STAGES > 2) k_tile<true>(s2, s1, w, x, source, reader, kt + 2, f, acc);
            if (STAGES > 3) k_tile<true>(s3, s2, w, x, source, reader, kt + 3, f, acc);
            kt += STAGES;
        } while (kt + 2 * STAGES - 1 <= k_end);
    } else {
        if (ahead > 0) fetch(s0, w, x, source, kt);
        if (STAGES > 2 && ahead > 1) fetch(s1, w, x, source, kt + 1);
        if (STAGES > 3 && ahead > 2) fetch(s2, w, x, source, kt + 2);
    }
    u8 *from = s0, *to = s3;
    for (; kt + ahead < k_end; kt++) {
        k_tile<true>(from, to, w, x, source, reader, kt, f, acc);
        to = from;
        from = from == s0 ? s1 : from == s1 ? s2 : s3;
    }
    for (; kt < k_end; kt++) {
        k_tile<false>(from, to, w, x, source, reader, kt, f, acc);
        from = from == s3 ? s0 : from == s0 ? s1 : from == s1 ? s2 : s3;
    }
#pragma unroll
    for (int s = 0; s < AHEAD; s++) multiply(f[1][s], acc);

    if (c.shares > 1) {
#pragma unroll
        for (int j = 0; j < MB; j++) {
            const u32 m = m0 + wave_m * WTM + j * 32 + frag_row;
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const u32 n = n0 + wave_n * WTN + i * 32 + e * 8 + half * 4;
                    if (m < c.tokens && n < c.parked_pitch) *parked_at(c, blockIdx.y, m, n) = i32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
                }
        }
        return;
    }
    if (threadIdx.x < TN) w_scales[threadIdx.x] = my_scale, bias[threadIdx.x] = my_bias;
    __syncthreads();   // the operand stages become the waves' strips
    store_sums(acc, c, n0 + wave_n * WTN, m0 + wave_m * WTM, x_scales, w_scales + wave_n * WTN, bias + wave_n * WTN, (out_t*)(wave % STAGES == 0 ? s0 : wave % STAGES == 1 ? s1 : wave % STAGES == 2 ? s2 : s3) + wave / STAGES * STRIP_VALUES);
}

)HIP";

// Streams. Reading the weights once is nearly all there is to do for few tokens, so they go straight into registers, as many loads on their way as
// there is room for; the tokens come out of the L2. The matrix instructions (16 x 16 x 64) are far from being a bound.
//
// One token, 4096 x 4096: 5.4 us (5.7 where the scales are read when the sums are there), 3 of them a launch, and 6.2 with weights that are in no cache; such weights of 8192 inputs and 16384
// channels (134 MB) 24.6 us (5.5 TB/s), of 28672 channels 40.1 (5.9 TB/s), where the estimate below takes tiles of 64 x 64, in 31.0 and 43.6.
const char* kStream = R"HIP(
extern "C" __global__ __launch_bounds__(WAVES * 64) void int8_stream(Call c) {
    __shared__ __attribute__((aligned(16))) int sums[WAVES][BM * 16][BN * 16 + 4];
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, tiles_n = (c.channels + BN * 16 - 1) / (BN * 16);
    const u32 n0 = blockIdx.x % tiles_n * (BN * 16), m0 = blockIdx.x / tiles_n * (BM * 16);
    // (the waves take turns along k, STEPS steps each: together they read long pieces of a row)
    const u32 chunks = c.pitch / 16, groups = (c.pitch + 64 * STEPS - 1) / (64 * STEPS), part = blockIdx.y * WAVES + wave, parts = c.shares * WAVES;
    // (four channels to a thread, whose scales are there when the sums are)
    static_assert(BM * 16 * BN * 4 <= WAVES * 64, "");
    const u32 j = threadIdx.x / (BN * 4), i = threadIdx.x % (BN * 4) * 4, m = m0 + j, n = n0 + i;
    const Scales scales = scales_of(c, m, n);
    const u8 *w[BN], *x[BM];
#pragma unroll
    for (int i = 0; i < BN; i++) {
        const u32 n = n0 + i * 16 + (lane & 15u);
        w[i] = c.w + (u64)(n < c.channels ? n : c.channels - 1) * c.pitch;
    }
#pragma unroll
    for (int j = 0; j < BM; j++) {
        const u32 m = m0 + j * 16 + (lane & 15u);
        x[j] = c.x + (u64)(m < c.tokens ? m : c.tokens - 1) * c.pitch;
    }
    i32x4 acc[BN][BM];
#pragma unroll
    for (int i = 0; i < BN; i++)
#pragma unroll
        for (int j = 0; j < BM; j++) acc[i][j] = i32x4{0, 0, 0, 0};
    struct Operands { i32x4 w[STEPS][BN], x[STEPS][BM]; } f[2];
    auto load = [&](Operands& o, u32 group) {
#pragma unroll
        for (int d = 0; d < STEPS; d++) {
            const u32 chunk = (group * STEPS + d) * 4 + (lane >> 4);
            const bool there = chunk < chunks;
#pragma unroll
            for (int i = 0; i < BN; i++) {
                o.w[d][i] = i32x4{0, 0, 0, 0};
                if (there) o.w[d][i] = *(const i32x4*)(w[i] + chunk * 16);
            }
#pragma unroll
            for (int j = 0; j < BM; j++) {
                o.x[d][j] = i32x4{0, 0, 0, 0};
                if (there) o.x[d][j] = *(const i32x4*)(x[j] + chunk * 16);
            }
        }
    };
    auto multiply = [&](const Operands& o) {
#pragma unroll
        for (int d = 0; d < STEPS; d++)
#pragma unroll
            for (int i = 0; i < BN; i++)
#pragma unroll
                for (int j = 0; j < BM; j++) acc[i][j] = MFMA_16(o.w[d][i], o.x[d][j], acc[i][j]);
    };
    // (two groups on their way; what is behind the rows' end is zeros)
    load(f[0], part);
    for (u32 g = part; g < groups; g += 2 * parts) {
        load(f[1], g + parts);
        multiply(f[0]);
        load(f[0], g + 2 * parts);
        multiply(f[1]);
    }
#pragma unroll
    for (int i = 0; i < BN; i++)
#pragma unroll
        for (int j = 0; j < BM; j++) *(i32x4*)&sums[wave][j * 16 + (lane & 15u)][i * 16 + (lane >> 4) * 4] = acc[i][j];
    __syncthreads();
    if (j >= BM * 16 || m >= c.tokens || n >= c.channels) return;
    i32x4 sum = *(const i32x4*)&sums[0][j][i];
#pragma unroll
    for (int v = 1; v < WAVES; v++) sum += *(const i32x4*)&sums[v][j][i];
    if (c.shares > 1) *parked_at(c, blockIdx.y, m, n) = sum;
    else store_four(c, m, n, sum, scales);
}
)HIP";

// The shares of a call's sums added up: four channels of a token to a thread.
const char* kJoin = R"HIP(
extern "C" __global__ __launch_bounds__(256) void int8_join(Call c) {
    const u32 fours = (c.channels + 3) / 4;
    const u64 at = (u64)blockIdx.x * 256 + threadIdx.x;
    if (at >= (u64)c.tokens * fours) return;
    const u32 m = (u32)(at / fours), n = (u32)(at % fours) * 4;
    const Scales scales = scales_of(c, m, n);
    i32x4 sum = *parked_at(c, 0, m, n);
#pragma unroll 4
    for (u32 s = 1; s < c.shares; s++) sum += *parked_at(c, s, m, n);
    store_four(c, m, n, sum, scales);
}
)HIP";

constexpr uint64_t kThreads = 1ull << 32;  // a launch has fewer
constexpr uint64_t kCUs = 256;
constexpr uint64_t kMostParked = 1 << 22;  // sums of all shares together, for which the scratch has room

// What the choice goes by (cut_of below), of tiles from products of 33 to 8192 tokens: microseconds of a call, of a k-tile in a workgroup that has a CU to itself and
// on full CUs, and of beginning and ending a workgroup there. The small tiles, whose waves have few matrix instructions to a k-step, read two steps ahead
// (1024 x 4096 x 4096 with 128 x 128 22.9 -> 21.2 us); 256 x 256 has no registers for that (61.7, and 63.1 with the spills). Waves of 64 x 32 in a 64 x 128
// tile 13.95 us with 512 x 4096 x 4096, of 32 x 64 14.7; four stages of 64 x 64 rather than three 9.4 for 10.7 with 128 x 4096 x 4096.
const Int8Shape kShapes[] = {
    {256, 256, 4, 2, 2, 1, 1, 8.3, 1.03, 1.57, 9.5},
    {128, 128, 2, 4, 4, 1, 2, 4.3, 0.37, 0.56, 2.8},
    {64, 128, 1, 4, 3, 2, 2, 3.6, 0.29, 0.61, 1.7},
    {64, 64, 2, 2, 4, 2, 2, 3.1, 0.20, 0.39, 1.1},
    {0, 0, 0, 0, 0, 1, 1, 0, 0, 0, 0, 1, 1, 8, 4},
    {0, 0, 0, 0, 0, 1, 1, 0, 0, 0, 0, 1, 2, 8, 4},
    {0, 0, 0, 0, 0, 1, 1, 0, 0, 0, 0, 1, 3, 8, 2},
    {0, 0, 0, 0, 0, 1, 1, 0, 0, 0, 0, 1, 4, 16, 1},
    {0, 0, 0, 0, 0, 1, 1, 0, 0, 0, 0, 2, 4, 16, 1},
};
constexpr int kCount = sizeof(kShapes) / sizeof(kShapes[0]);

std::string definitions(int dtype, const Int8Shape* t) {
    std::ostringstream s;
    s << "#define BF16 " << (dtype == HE_BF16) << "\n#define F16 " << (dtype == HE_F16) << "\n";
    if (t && t->stream()) s << "#define BN " << t->blocks_n << "\n#define BM " << t->blocks_m << "\n#define WAVES " << t->waves << "\n#define STEPS " << t->steps << "\n";
    else if (t)
        s << "#define TN " << t->tile_n << "\n#define TM " << t->tile_m << "\n#define WAVES_N " << t->waves_n << "\n#define WAVES_M " << t->waves_m
          << "\n#define STAGES " << t->stages << "\n#define AHEAD " << t->ahead << "\n#ifndef KERNEL_ATTRS\n#define KERNEL_ATTRS __attribute__((amdgpu_waves_per_eu("
          << t->waves_n * t->waves_m * t->per_cu / 4 << ", " << t->waves_n * t->waves_m * t->per_cu / 4 << ")))\n#endif\n";
    return s.str();
}

uint64_t cut(int64_t extent, int by) { return ((uint64_t)extent + by - 1) / by; }
int64_t parked_pitch(const Int8Problem& pr) { return (int64_t)cut(pr.channels, 4) * 4; }

// How long a call would take, in microseconds. Streams: a CU reads 36 KB in one, of weights and tokens alike, the weights come out of memory at 6 TB/s at
// best, and a workgroup that follows another on its CU takes a while to begin and end. Shares cost a second launch.
//
// Tiles have no such bound by memory here, so that for a token or two of large layers they are taken for faster than they are. In us, weights in no cache, each side's best but
// for the tiles' shares, which are the chosen ones:
//   inputs, channels    1 token: tiles, stream    8 tokens: tiles, stream
//   4096, 14336                  14.2    14.1               14.3    16.3
//   4096, 28672                  26.8    23.3               27.2    28.4
//   4096, 128256                 91      87                 95      111
//   8192, 8192                   18.4    14.0               18.8    16.2
//   8192, 16384                  31.0    24.6               30.8    29.5
//   8192, 28672                  43.6    40.1               43.8    49.9
//   14336, 4096                  15.1    12.9               15.4    15.2
// (4096 and 4096 are the stream's: 6.2, tiles 8.6.)
Int8Cut cut_of(const Int8Problem& pr, int64_t tokens, int shape, uint32_t shares) {
    const Int8Shape& t = kShapes[shape];
    Int8Cut c;
    c.shape = shape, c.shares = shares, c.blocks = cut(pr.channels, t.channels()) * cut(tokens, t.tokens());
    const double pitch = (double)quantized_pitch(pr.inputs), blocks = (double)c.blocks * shares;
    c.estimate = shares > 1 ? 2.2 + (double)shares * tokens * pr.channels * 4 / 3e6 : 0;
    if (t.stream()) {
        const double sums = t.blocks_n * t.blocks_m, rows = 16.0 * t.blocks_n + std::min<double>(16.0 * t.blocks_m, (double)tokens);
        // (sums of four blocks and more fill a CU's LDS with one workgroup)
        const double rounds = sums >= 4 && blocks < 4 * kCUs ? std::ceil(blocks / kCUs) : std::max(1.0, blocks / kCUs);
        c.estimate += 2.5 + 0.08 * sums + std::max(rounds * rows * pitch / shares / 36e3, pr.channels * pitch / 6e6) + (rounds - 1) * (0.2 + 0.02 * t.waves * sums);
        return c;
    }
    const double k_tiles = std::ceil(pitch / 128 / shares), slots = (double)kCUs * t.per_cu, rounds = blocks < 4 * slots ? std::ceil(blocks / slots) : blocks / slots;
    const bool alone = t.per_cu > 1 ? blocks <= kCUs : blocks <= kCUs / 2;
    c.estimate += t.base + (alone ? k_tiles * t.alone : rounds * (k_tiles * t.full + t.round) - (t.per_cu > 1 ? 0 : t.round));
    return c;
}

struct CallArg {
    const void *x, *w;
    const float *x_scales, *w_scales, *bias;
    void* y;
    uint32_t tokens, channels, pitch, blocks, shares, parked_pitch;
    int32_t* parked;
};

}  // namespace

struct Int8Kernels {
    std::string source;
    std::unique_ptr<JitKernel> product[kCount], join;
    std::mutex mu;  // a call's two launches follow each other on their stream: they share the stream's scratch, which all products have in common
    ReduceScratch scratch;
    ~Int8Kernels() { scratch.release(); }

    explicit Int8Kernels(int dtype) {
        std::vector<std::string> texts(kCount);
        const std::string joining = definitions(dtype, nullptr) + kCommon + kJoin;
        std::vector<std::future<void>> compiled;
        for (int k = 0; k < kCount; k++) {
            texts[k] = definitions(dtype, &kShapes[k]) + kCommon + (kShapes[k].stream() ? kStream : kTile);
            compiled.push_back(std::async(std::launch::async, [&texts, k] { (void)rtc_compile(texts[k], "int8_product", {}); }));
            source += "//// shape\n" + texts[k];
        }
        for (auto& f : compiled) f.get();
        for (int k = 0; k < kCount; k++) product[k] = std::make_unique<JitKernel>(texts[k], kShapes[k].stream() ? "int8_stream" : "int8_product");
        join = std::make_unique<JitKernel>(joining, "int8_join");
        source += "//// shape\n" + joining;
    }

    static std::shared_ptr<Int8Kernels> of(int dtype) {
        static std::mutex mu;
        static std::map<int, std::weak_ptr<Int8Kernels>> made;
        std::lock_guard<std::mutex> lk(mu);
        std::shared_ptr<Int8Kernels> k = made[dtype].lock();
        if (!k) made[dtype] = k = std::make_shared<Int8Kernels>(dtype);
        return k;
    }
};

std::string Int8Cut::describe() const {
    const Int8Shape& t = kShapes[shape];
    const std::string how = t.stream() ? strfmt("int8 stream shape=%d blocks_n=%d blocks_m=%d waves=%d", shape, t.blocks_n, t.blocks_m, t.waves)
                                       : strfmt("int8 tiles shape=%d tile=%dx%d waves=%dx%d stages=%d", shape, t.tile_n, t.tile_m, t.waves_n, t.waves_m, t.stages);
    return how + strfmt(" threads=%d grid=%llu shares=%u estimate=%.1f", t.threads(), (unsigned long long)blocks, shares, estimate);
}

// Of all shapes and numbers of shares the one with the least estimate. A share is at least four k-tiles long, or what a stream's waves need to have four
// steps of it each.
Int8Cut plan_int8(const Int8Problem& pr, int64_t tokens) {
    const int forced = std::clamp(tuning::get_int("HELIUM_HIP_INT8_SHAPE", 0), 0, kCount), forced_shares = tuning::get_int("HELIUM_HIP_INT8_SHARES", 0);
    Int8Cut best = cut_of(pr, tokens, forced ? forced - 1 : 0, 1);
    if (forced_shares) best.estimate = 1e30;
    for (int k = 0; k < kCount; k++) {
        const Int8Shape& t = kShapes[k];
        if (forced ? k != forced - 1 : t.stream() && t.blocks_m != (int)std::min<uint64_t>(4, cut(tokens, 16))) continue;
        const uint64_t least = t.stream() ? (uint64_t)t.waves * 256 : 512;  // bytes of k
        for (uint32_t shares = 1; shares <= 16; shares *= 2) {
            if (shares > 1 && ((uint64_t)shares * tokens * parked_pitch(pr) > kMostParked || (uint64_t)quantized_pitch(pr.inputs) < least * shares)) break;
            if (forced_shares && shares != (uint32_t)forced_shares) continue;
            const Int8Cut c = cut_of(pr, tokens, k, shares);
            if (c.estimate < best.estimate) best = c;
        }
    }
    return best;
}

Int8Matmul::Int8Matmul(const Int8Problem& pr) : pr_(pr) {
    HE_REQUIRE(pr.inputs >= 1 && pr.channels >= 1, HE_ERR_INVALID, "int8 product: %lld inputs, %lld channels", (long long)pr.inputs, (long long)pr.channels);
    // (2^17 products of two bytes are less than 2^31 in any case)
    HE_REQUIRE(pr.inputs < (1 << 17) && pr.channels <= (1 << 24), HE_ERR_UNSUPPORTED, "int8 product: %lld inputs (131071 are taken), %lld channels (2^24 are taken)",
               (long long)pr.inputs, (long long)pr.channels);
    HE_REQUIRE(pr.dtype == HE_F16 || pr.dtype == HE_BF16 || pr.dtype == HE_F32, HE_ERR_INVALID, "int8 product does not give dtype %s", dtype_name(pr.dtype));
    kernels_ = Int8Kernels::of(pr.dtype);
}

const std::string& Int8Matmul::source() const { return kernels_->source; }

void Int8Matmul::multiply(int64_t tokens, const void* x, const float* x_scales, const void* weights, const float* weight_scales, const float* bias, void* y,
                          hipStream_t stream) {
    HE_REQUIRE(tokens >= 0, HE_ERR_INVALID, "int8 product: %lld tokens", (long long)tokens);
    if (tokens == 0) return;
    HE_REQUIRE(tokens <= (1 << 24), HE_ERR_UNSUPPORTED, "int8 product: %lld tokens, at most 2^24 are taken", (long long)tokens);
    const auto check = [](const char* what, const void* p, uintptr_t alignment) {
        HE_REQUIRE(p && (uintptr_t)p % alignment == 0, HE_ERR_INVALID, "int8 product: %s null or not aligned to %d bytes", what, (int)alignment);
    };
    check("the tokens are", x, 16);
    check("the weights are", weights, 16);
    check("the tokens' scales are", x_scales, 4);
    check("the weights' scales are", weight_scales, 4);
    check("the result is", y, dtype_bits(pr_.dtype) / 8);
    HE_REQUIRE((uintptr_t)bias % 4 == 0, HE_ERR_INVALID, "int8 product: the bias is not aligned to 4 bytes");
    const Int8Cut c = plan_int8(pr_, tokens);
    const Int8Shape& t = kShapes[c.shape];
    HE_REQUIRE(c.blocks < kThreads / t.threads(), HE_ERR_UNSUPPORTED, "int8 product: %lld tokens of %lld channels are too many for one launch", (long long)tokens,
               (long long)pr_.channels);
    CallArg call{x, weights, x_scales, weight_scales, bias, y, (uint32_t)tokens, (uint32_t)pr_.channels, (uint32_t)quantized_pitch(pr_.inputs), (uint32_t)c.blocks, c.shares,
                 (uint32_t)parked_pitch(pr_), nullptr};
    const uint32_t grid[3] = {(uint32_t)c.blocks, c.shares, 1}, block[3] = {(uint32_t)t.threads(), 1, 1};
    void* args[] = {&call};
    if (c.shares == 1) {
        kernels_->product[c.shape]->launch(grid, block, 0, stream, args, true);
        return;
    }
    const uint32_t join_grid[3] = {(uint32_t)cut(tokens * (int64_t)cut(pr_.channels, 4), 256), 1, 1}, join_block[3] = {256, 1, 1};
    std::lock_guard<std::mutex> lk(kernels_->mu);
    call.parked = (int32_t*)kernels_->scratch.get(kMostParked, 0, stream).floats;
    kernels_->product[c.shape]->launch(grid, block, 0, stream, args);
    kernels_->join->launch(join_grid, join_block, 0, stream, args, true);
}

}  // namespace he

// ---- C ABI ------------------------------------------------------------------------------------------------
struct he_int8_matmul_s {
    he::Int8Matmul impl;
    explicit he_int8_matmul_s(const he::Int8Problem& pr) : impl(pr) {}
};

extern "C" {

int he_int8_matmul_create(he_int8_matmul_t* matmul, int64_t inputs, int64_t channels, int dtype) {
    return he::guard([&] {
        HE_REQUIRE(matmul, HE_ERR_INVALID, "bad argument");
        he::Int8Problem pr;
        pr.inputs = inputs, pr.channels = channels, pr.dtype = dtype;
        *matmul = new he_int8_matmul_s(pr);
    });
}

int he_int8_matmul_destroy(he_int8_matmul_t matmul) {
    return he::guard([&] { delete matmul; });
}

int he_int8_matmul(he_int8_matmul_t matmul, int64_t tokens, const void* x, const float* x_scales, const void* weights, const float* weight_scales, const float* bias,
                   void* y, he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(matmul, HE_ERR_INVALID, "null int8 product");
        matmul->impl.multiply(tokens, x, x_scales, weights, weight_scales, bias, y, stream ? stream->s : nullptr);
    });
}

const char* he_int8_matmul_source(he_int8_matmul_t matmul) { return matmul ? matmul->impl.source().c_str() : ""; }

int he_int8_matmul_describe(he_int8_matmul_t matmul, int64_t tokens, char* text, size_t capacity) {
    return he::guard([&] {
        HE_REQUIRE(matmul && text && capacity && tokens >= 1, HE_ERR_INVALID, "bad argument");
        snprintf(text, capacity, "%s", matmul->impl.describe(tokens).c_str());
    });
}

}  // extern "C"
