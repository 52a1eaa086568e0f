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
// in every shape and cut.
__device__ __forceinline__ float scaled(int sum, float x_scale, float w_scale, float bias) { return __builtin_fmaf((float)sum * x_scale, w_scale, bias); }
typedef out_t out4_any __attribute__((ext_vector_type(4), aligned(sizeof(out_t))));
__device__ __forceinline__ void store_four(const Call& c, u32 m, u32 n, i32x4 sum) {
    const float x_scale = c.x_scales[m];
    out_t* to = c.y + (u64)m * c.channels + n;
    out4_any out;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const u32 of = n + k < c.channels ? n + k : c.channels - 1;
        out[k] = (out_t)scaled(sum[k], x_scale, c.w_scales[of], c.bias ? c.bias[of] : 0.0f);
    }
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
// 256 x 256: 4096 x 4096 x 4096 64 to 66 us (2100 TOPS; the instructions alone would take 31 at the 2.1 GHz that such products run at), 10 of them beginning and
// end: results leave when no sums are left to hide them. Per k-tile a CU reads 192 KB of LDS and writes 64, 2048 clocks, as many as its instructions
// take, and both together take 1.75 us (3700 clocks). Waves of 64 x 128, four along the channels, 64 us, 128 x 64 66, 32 x 256 71; raised priority for the
// instructions 69; four waves of 128 x 128 69.
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
#define STRIP_BYTES (STRIP_VALUES * WAVES_N * WAVES_M * (int)sizeof(out_t))
#define LDS_BYTES (STAGES * STAGE_BYTES > STRIP_BYTES ? STAGES * STAGE_BYTES : STRIP_BYTES)

__device__ __attribute__((aligned(16))) const u32 nothing[4] = {0, 0, 0, 0};   // what lies behind a row's end

struct Fragments { i32x4 w[NB], x[MB]; };
struct True { static constexpr int value = 1; constexpr operator bool() const { return true; } };
struct False { static constexpr int value = 0; constexpr operator bool() const { return false; } };

// What a wave stores of its sums: 32 tokens at a time through its strip, so that whole vectors of channels go out.
__device__ __forceinline__ void store_sums(const i32x16 (&acc)[NB][MB], const Call& c, u32 n0, u32 m0, const float* w_scales, const float* bias, out_t* strip) {
    const u32 lane = threadIdx.x & 63u, half = lane >> 5;
    const bool past = (u64)c.tokens * c.channels >= (1u << 21);   // (results of 4 MB and more bypass the caches: 4096 x 4096 x 4096 67.5 -> 66.5 us)
#pragma unroll
    for (int j = 0; j < MB; j++) {
        const u32 m = m0 + j * 32 + (lane & 31u);
        const float x_scale = c.x_scales[m < c.tokens ? m : c.tokens - 1];
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32 n = i * 32 + e * 8 + half * 4;
                const f32x4 ws = *(const f32x4*)(w_scales + n), b = *(const f32x4*)(bias + n);
                out4 out;
#pragma unroll
                for (int k = 0; k < 4; k++) out[k] = (out_t)scaled(acc[i][j][e * 4 + k], x_scale, ws[k], b[k]);
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
// The scales and the bias of the tile's channels, in LDS: 1 and 0 where there are none.
__device__ __forceinline__ void load_channels(const Call& c, u32 n0, float* w_scales, float* bias) {
    for (u32 n = threadIdx.x; n < TN; n += WAVES_N * WAVES_M * 64) {
        const bool there = n0 + n < c.channels;
        w_scales[n] = there ? c.w_scales[n0 + n] : 1.0f;
        bias[n] = there && c.bias ? c.bias[n0 + n] : 0.0f;
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

extern "C" __global__ __launch_bounds__(WAVES_N * WAVES_M * 64) KERNEL_ATTRS void int8_product(Call c) {
    __shared__ __attribute__((aligned(16))) u8 lds[LDS_BYTES];
    __shared__ __attribute__((aligned(16))) float w_scales[TN], bias[TN];
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave_n = wave / WAVES_M, wave_m = wave % WAVES_M;
    u32 tn, tm;
    place(c, tn, tm);
    const u32 n0 = tn * TN, m0 = tm * TM;
    const u8 *w_rows = c.w + (u64)n0 * c.pitch, *x_rows = c.x + (u64)m0 * c.pitch;
    const u32 k_tiles = (c.pitch + ROW - 1) / ROW, chunks = c.pitch / 16;
    const u32 k_begin = (u32)((u64)k_tiles * blockIdx.y / c.shares), k_end = (u32)((u64)k_tiles * (blockIdx.y + 1) / c.shares);
    // Direct loads: lane l of the load of rows 8 r .. 8 r + 7 takes row l / 8 and, so that fragment reads meet different banks, the chunk
    // (l % 8) ^ (row / 2 % 8) of its 128 bytes: two rows fill the 64 banks, so rows two apart must differ. (A tile that ends beyond an
    // operand loads its last row there: sums that nothing stores.)
    u32 off[LOADS], chunk[2] = {(lane & 7u) ^ (lane >> 4), (lane & 7u) ^ (4u + (lane >> 4))};
#pragma unroll
    for (int l = 0; l < LOADS; l++) {
        const u32 row = (wave * LOADS + l) * 8;   // of the weights, then of the tokens
        const u32 of = row < TN ? row : row - TN, last = (row < TN ? c.channels - n0 : c.tokens - m0) - 1, mine = of + (lane >> 3);
        off[l] = (mine < last ? mine : last) * c.pitch + chunk[l & 1] * 16;
    }
    auto fetch = [&](u32 kt, u32 slot) {
        u8* base = lds + slot * STAGE_BYTES;
        const bool whole = kt * 8 + 8 <= chunks;
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const u32 row = (wave * LOADS + l) * 8;
            const u8* src = (row < TN ? w_rows : x_rows) + (u64)kt * ROW + off[l];
            if (!whole && kt * 8 + chunk[l & 1] >= chunks) src = (const u8*)nothing;
            __builtin_amdgcn_global_load_lds((const GLOBAL_AS u32*)src, (LDS_AS u32*)(base + row * ROW), 16, 0, 0);
        }
    };
    i32x16 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
    const u32 frag_row = lane & 31u, half = lane >> 5, swz = lane >> 1 & 7u;
    auto read = [&](Fragments& g, const u8* stage, int kk) {
        const u8 *w = stage + (wave_n * WTN + frag_row) * ROW, *x = stage + (TN + wave_m * WTM + frag_row) * ROW;
        const u32 at = ((kk * 2 + half) ^ swz) * 16;
#pragma unroll
        for (int i = 0; i < NB; i++) g.w[i] = *(const i32x4*)(w + i * 32 * ROW + at);
#pragma unroll
        for (int j = 0; j < MB; j++) g.x[j] = *(const i32x4*)(x + j * 32 * ROW + at);
    };
    auto multiply = [&](const Fragments& g) {
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < MB; j++) acc[i][j] = MFMA_32(g.w[i], g.x[j], acc[i][j]);
    };
    u32 slot = 0;
    // This wave's loads of a k-tile have landed (those of the STAGES - 2 behind it may be on their way), then the other waves'. No wave still reads the
    // stage that is filled next. (The bare barrier: __syncthreads() would wait for all loads.)
    auto meet = [&](auto more) {
        if (more) __builtin_amdgcn_s_waitcnt(WAIT_LOADS((STAGES - 2) * LOADS));
        else __builtin_amdgcn_s_waitcnt(WAIT_LOADS(0));
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    auto fetch_ahead = [&](u32 kt) { fetch(kt + STAGES - 1, slot + STAGES - 1 < STAGES ? slot + STAGES - 1 : slot - 1); };
    const u32 k_count = k_end - k_begin, ahead = STAGES - 1 < k_count ? STAGES - 1 : k_count;
    load_channels(c, n0, w_scales, bias);
    for (u32 s = 0; s < ahead; s++) fetch(k_begin + s, s);
    u32 kt = k_begin;
    Fragments f[2][AHEAD];
#pragma unroll
    for (int s = 0; s < AHEAD; s++) {
#pragma unroll
        for (int i = 0; i < NB; i++) f[1][s].w[i] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < MB; j++) f[1][s].x[j] = i32x4{0, 0, 0, 0};
    }
#if AHEAD == 1
    // The loop is rotated by a k-step: the matrix instructions that the last k-tile left over cover the barrier's way, the
    // first reads of this one and the loads of the one to come; each further step's reads are issued between the instructions of
    // the step before. The order is asked for, since the compiler by itself reads, waits and multiplies in turn.
    auto k_tile = [&](u32 kt, auto more) {
        meet(more);
        const u8* stage = lds + slot * STAGE_BYTES;
        read(f[0][0], stage, 0);
        if (more) fetch_ahead(kt);
        multiply(f[1][0]);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
        for (int n = 0; n < MMAS; n++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
            for (int l = n * LOADS / MMAS; l < (n + 1) * LOADS / MMAS; l++)
                if (more) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        }
#pragma unroll
        for (int kk = 1; kk < 4; kk++) {
            read(f[kk & 1][0], stage, kk);
            multiply(f[(kk & 1) ^ 1][0]);
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
    for (; kt + ahead < k_end; kt++) k_tile(kt, True());
    for (; kt < k_end; kt++) k_tile(kt, False());
    multiply(f[1][0]);
#else
    // A wave of a small tile has few matrix instructions to a k-step, fewer than an LDS read takes to come: the loop is rotated by a whole
    // k-tile, whose instructions cover the barrier and all reads of the next one.
    auto k_tile = [&](u32 kt, auto more, auto odd) {
        constexpr int now = decltype(odd)::value;
        meet(more);
#pragma unroll
        for (int kk = 0; kk < 4; kk++) read(f[now][kk], lds + slot * STAGE_BYTES, kk);
        if (more) fetch_ahead(kt);
#pragma unroll
        for (int kk = 0; kk < 4; kk++) multiply(f[now ^ 1][kk]);
        slot = slot + 1 < STAGES ? slot + 1 : 0;
        // (all reads and loads first)
        __builtin_amdgcn_sched_group_barrier(0x100, 4 * READS, 0);
        if (more) __builtin_amdgcn_sched_group_barrier(0x020, LOADS, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 4 * MMAS, 0);
    };
    auto either = [&](u32 kt, auto more) {
        if ((kt - k_begin) & 1) k_tile(kt, more, True());
        else k_tile(kt, more, False());
    };
    for (; kt + ahead + 1 < k_end; kt += 2) {
        k_tile(kt, True(), False());
        k_tile(kt + 1, True(), True());
    }
    for (; kt + ahead < k_end; kt++) either(kt, True());
    for (; kt < k_end; kt++) either(kt, False());
    if (k_count & 1)
#pragma unroll
        for (int kk = 0; kk < 4; kk++) multiply(f[0][kk]);
    else
#pragma unroll
        for (int kk = 0; kk < 4; kk++) multiply(f[1][kk]);
#endif

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
    __syncthreads();   // the operand stages become the waves' strips
    store_sums(acc, c, n0 + wave_n * WTN, m0 + wave_m * WTM, w_scales + wave_n * WTN, bias + wave_n * WTN, (out_t*)lds + wave * STRIP_VALUES);
}

)HIP";

// Streams. Reading the weights once is nearly all there is to do for few tokens, so they go straight into registers, as many loads on their way as
// there is room for; the tokens come out of the L2. The matrix instructions (16 x 16 x 64) are far from being a bound.
//
// One token, 4096 x 4096: 5.6 us, 3 of them a launch; 8192 inputs, 16384 channels (134 MB, more than the caches hold with two others) 25 us (5.3 TB/s).
const char* kStream = R"HIP(
extern "C" __global__ __launch_bounds__(WAVES * 64) void int8_stream(Call c) {
    __shared__ __attribute__((aligned(16))) int sums[WAVES][BM * 16][BN * 16 + 4];
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, tiles_n = (c.channels + BN * 16 - 1) / (BN * 16);
    const u32 n0 = blockIdx.x % tiles_n * (BN * 16), m0 = blockIdx.x / tiles_n * (BM * 16);
    // (the waves take turns along k, STEPS steps each: together they read long pieces of a row)
    const u32 chunks = c.pitch / 16, groups = (c.pitch + 64 * STEPS - 1) / (64 * STEPS), part = blockIdx.y * WAVES + wave, parts = c.shares * WAVES;
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
    // (four channels to a thread)
    for (u32 e = threadIdx.x; e < BM * 16 * BN * 4; e += WAVES * 64) {
        const u32 j = e / (BN * 4), i = e % (BN * 4) * 4, m = m0 + j, n = n0 + i;
        if (m >= c.tokens || n >= c.channels) continue;
        i32x4 sum = *(const i32x4*)&sums[0][j][i];
#pragma unroll
        for (int v = 1; v < WAVES; v++) sum += *(const i32x4*)&sums[v][j][i];
        if (c.shares > 1) *parked_at(c, blockIdx.y, m, n) = sum;
        else store_four(c, m, n, sum);
    }
}
)HIP";

// The shares of a call's sums added up: four channels of a token to a thread.
const char* kJoin = R"HIP(
extern "C" __global__ __launch_bounds__(256) void int8_join(Call c) {
    const u32 fours = (c.channels + 3) / 4;
    const u64 at = (u64)blockIdx.x * 256 + threadIdx.x;
    if (at >= (u64)c.tokens * fours) return;
    const u32 m = (u32)(at / fours), n = (u32)(at % fours) * 4;
    i32x4 sum = *parked_at(c, 0, m, n);
#pragma unroll 4
    for (u32 s = 1; s < c.shares; s++) sum += *parked_at(c, s, m, n);
    store_four(c, m, n, sum);
}
)HIP";

constexpr uint64_t kThreads = 1ull << 32;  // a launch has fewer
constexpr uint64_t kCUs = 256;
constexpr uint64_t kMostParked = 1 << 22;  // sums of all shares together, for which the scratch has room

// What the choice goes by (cut_of below), from products of 1 to 8192 tokens: microseconds of a call, of a k-tile in a workgroup that has a CU to itself and
// on full CUs, and of beginning and ending a workgroup there. The small tiles, whose waves
// have few matrix instructions to a k-step, read a whole k-tile ahead: 1024 x 4096 x 4096 28.1 -> 25.9 us with 64 x 128 (128 x 128 24.6), 512 tokens
// 22.6 -> 17.9, 2048 x 1024 x 1024 7.4 -> 6.8. Of 256 x 256 four waves along the channels read less from LDS than two: 66.4 -> 64.
const Int8Shape kShapes[] = {
    {256, 256, 4, 2, 2, 1, 1, 9.0, 1.24, 1.76, 6.5},
    {128, 128, 2, 4, 4, 1, 4, 5.2, 0.46, 0.61, 3.3},
    {64, 128, 2, 2, 3, 2, 4, 3.6, 0.42, 0.60, 3.2},
    {64, 64, 2, 2, 3, 3, 4, 3.5, 0.33, 0.43, 2.0},
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
    const int forced = tuning::get_int("HELIUM_HIP_INT8_SHAPE", 0), forced_shares = tuning::get_int("HELIUM_HIP_INT8_SHARES", 0);
    Int8Cut best = cut_of(pr, tokens, forced ? std::min(forced, kCount) - 1 : 0, 1);
    if (forced_shares) best.estimate = 1e30;
    for (int k = 0; k < kCount; k++) {
        const Int8Shape& t = kShapes[k];
        if (forced ? k != std::min(forced, kCount) - 1 : t.stream() && t.blocks_m != (int)std::min<uint64_t>(4, cut(tokens, 16))) continue;
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
