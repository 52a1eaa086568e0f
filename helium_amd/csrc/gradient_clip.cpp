#include "gradient_clip.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <sstream>

namespace he {

namespace {

constexpr uint32_t kGroup = 128;          // tensors whose addresses one launch takes by value
constexpr uint64_t kChunk = 16384;        // bytes
constexpr uint32_t kBlocks = 1024;        // workgroups of all groups together, about: the four to a CU that registers allow
constexpr uint64_t kKept = 12288;         // chunks (192 MB) that the second launch finds in the Infinity Cache
constexpr size_t kMostTensors = 65536;

// ---- device text ---------------------------------------------------------------------------------------------------
// norm = sqrt(sum of squares of all gradients), out = g min(1, most / (norm + 1e-6)). The first launch adds up squares, each workgroup its chunks',
// the second adds up the workgroups' sums, in every workgroup again while its first chunk is on its way, and scales. Squares and their sums
// are f64: those of f32 values neither overflow nor vanish, and the order, which is fixed, leaves no trace in the norm's 24 bits.
//
// Bound by memory: everything is read twice and written once. The second launch goes through the chunks in the opposite order, so that it begins with
// what the first one read last; of more than the Infinity Cache (256 MB) holds, only the last 192 MB are read so that they stay there, and results never are
// written so. 24 x 4096 x 4096 bf16: squares 125 to 135 us (6.0 to 6.5 TB/s), scaling 268 (6.0 TB/s); in the same order 419 us together, without the distinction 408. The
// 65 tensors (47 MB) of a classifier 26.5 us; with 2048 workgroups 29.7, and results that stay in the caches cost another 1 (40 x 1000 x 1000 bf16: 42.8 and 51.3).
const char* kText = R"HIP(
typedef unsigned char u8;
typedef unsigned short u16;
typedef unsigned int u32;
typedef unsigned long long u64;
typedef u32 u32x4 __attribute__((ext_vector_type(4)));
// (a tensor begins at any whole value)
typedef u32 u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
#ifndef SHFL_XOR_F64
#define SHFL_XOR_F64(v, m) __shfl_xor(v, m, 64)
#define COUNT_LANES(p) __popcll(__ballot(p))
#endif
#define VECTORS (CHUNK / 256 / 16)   // of a thread
struct Tensor { u32 first, dtype; u64 bytes; };
struct Inputs { const u8* in[GROUP]; };
struct Both { const u8* in[GROUP]; u8* out[GROUP]; };
enum { F16_T = 0, BF16_T = 1, F32_T = 2 };

__device__ __forceinline__ float of_bits(u32 b) { return __builtin_bit_cast(float, b); }
__device__ __forceinline__ u32 bits_of(float f) { return __builtin_bit_cast(u32, f); }
__device__ __forceinline__ float f16_value(u32 b) { return (float)__builtin_bit_cast(_Float16, (u16)b); }
__device__ __forceinline__ u32 f16_bits(float f) { return __builtin_bit_cast(u16, (_Float16)f); }
__device__ __forceinline__ u32 bf16_bits(float f) { return __builtin_bit_cast(u16, (__bf16)f); }

// The tensors of a group: each lane knows where two of them begin, and a chunk's tensor is the last that begins no later.
struct Begins { u32 a, b; };
__device__ __forceinline__ Begins begins_of(const Tensor* tensors, u32 count) {
    const u32 lane = threadIdx.x & 63u;
    return {lane < count ? tensors[lane].first : ~0u, lane + 64 < count ? tensors[lane + 64].first : ~0u};
}
__device__ __forceinline__ u32 tensor_of(const Begins& begins, u32 chunk) {
    return __builtin_amdgcn_readfirstlane((u32)(COUNT_LANES(begins.a <= chunk) + COUNT_LANES(begins.b <= chunk)) - 1u);
}

struct Held { u32x4 v[VECTORS]; };
// A thread's vectors of a chunk: 256 threads side by side. What lies behind the tensor's end is zero.
template <bool PASSING> __device__ __forceinline__ void load(Held& h, const u8* from, u64 left) {
#pragma unroll
    for (int k = 0; k < VECTORS; k++) {
        const u32 at = (k * 256 + threadIdx.x) * 16;
        h.v[k] = u32x4{0, 0, 0, 0};
        if (at + 16 <= left) h.v[k] = PASSING ? __builtin_nontemporal_load((const u32x4_any*)(from + at)) : *(const u32x4_any*)(from + at);
        else if (at < left) {
            u32 part[4] = {0, 0, 0, 0};
#pragma unroll
            for (u32 e = 0; e < 8; e++)
                if (at + e * 2 < left) part[e / 2] |= (u32)*(const u16*)(from + at + e * 2) << (e % 2 * 16);
            h.v[k] = u32x4{part[0], part[1], part[2], part[3]};
        }
    }
}
__device__ __forceinline__ void store(const Held& h, u8* to, u64 left) {
#pragma unroll
    for (int k = 0; k < VECTORS; k++) {
        const u32 at = (k * 256 + threadIdx.x) * 16;
        if (at + 16 <= left) {
            __builtin_nontemporal_store(h.v[k], (u32x4_any*)(to + at));
        } else if (at < left)
#pragma unroll
            for (u32 e = 0; e < 8; e++)
                if (at + e * 2 < left) *(u16*)(to + at + e * 2) = (u16)(h.v[k][e / 2] >> (e % 2 * 16));
    }
}
__device__ __forceinline__ double squares(const Held& h, u32 dtype, double sum) {
    double other = 0.0;   // (two chains)
#pragma unroll
    for (int k = 0; k < VECTORS; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const u32 word = h.v[k][e];
            if (dtype == F32_T) {
                const double a = of_bits(word);
                if (e & 1) other += a * a;
                else sum += a * a;
            } else {
                const double a = dtype == BF16_T ? of_bits(word << 16) : f16_value(word), b = dtype == BF16_T ? of_bits(word & 0xffff0000u) : f16_value(word >> 16);
                sum += a * a;
                other += b * b;
            }
        }
    return sum + other;
}
template <class F> __device__ __forceinline__ void scale(Held& h, u32 dtype, F by) {
#pragma unroll
    for (int k = 0; k < VECTORS; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const u32 word = h.v[k][e];
            if (dtype == F32_T) h.v[k][e] = bits_of((float)(of_bits(word) * by));
            else if (dtype == BF16_T) h.v[k][e] = bf16_bits((float)(of_bits(word << 16) * by)) | bf16_bits((float)(of_bits(word & 0xffff0000u) * by)) << 16;
            else h.v[k][e] = f16_bits((float)(f16_value(word) * by)) | f16_bits((float)(f16_value(word >> 16) * by)) << 16;
        }
}
// (`passing`: chunks of the group that no later launch finds in a cache)
// The sum over a workgroup's 256 threads, in every one of them.
__device__ __forceinline__ double over_group(double s, double* waves) {
    for (int m = 32; m > 0; m /= 2) s += SHFL_XOR_F64(s, m);
    if ((threadIdx.x & 63u) == 0) waves[threadIdx.x >> 6] = s;
    __syncthreads();
    return waves[0] + waves[1] + waves[2] + waves[3];
}
__device__ __forceinline__ double norm_of(const double* __restrict__ sums, u32 count, double* waves) {
    double s = 0.0;
#pragma unroll 4
    for (u32 k = threadIdx.x; k < count; k += 256) s += sums[k];
    return sqrt(over_group(s, waves));
}

extern "C" __global__ __launch_bounds__(256) void clip_squares(Inputs o, const Tensor* __restrict__ tensors, u32 count, u32 chunks, u32 passing, double* __restrict__ sums) {
    __shared__ double waves[4];
    const Begins begins = begins_of(tensors, count);
    double sum = 0.0;
    for (u32 c = blockIdx.x; c < chunks; c += gridDim.x) {
        const u32 t = tensor_of(begins, c);
        const u64 at = (u64)(c - tensors[t].first) * CHUNK;
        Held h;
        if (c < passing) load<true>(h, o.in[t] + at, tensors[t].bytes - at);
        else load<false>(h, o.in[t] + at, tensors[t].bytes - at);
        sum = squares(h, tensors[t].dtype, sum);
    }
    sum = over_group(sum, waves);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

extern "C" __global__ __launch_bounds__(256) void clip_norm(const double* __restrict__ sums, u32 count, float* __restrict__ norm) {
    __shared__ double waves[4];
    const double n = norm_of(sums, count, waves);
    if (threadIdx.x == 0) *norm = (float)n;
}

extern "C" __global__ __launch_bounds__(256) void clip_scale(Both o, const Tensor* __restrict__ tensors, u32 count, u32 chunks, u32 passing, const double* __restrict__ sums,
                                                             u32 sum_count, float most, float* __restrict__ norm) {
    __shared__ double waves[4];
    const Begins begins = begins_of(tensors, count);
    float by = 1.0f;
    double exact_by = 1.0;
    for (u32 k = blockIdx.x; k < chunks; k += gridDim.x) {
        const u32 c = chunks - 1 - k, t = tensor_of(begins, c), dtype = tensors[t].dtype;
        const u64 at = (u64)(c - tensors[t].first) * CHUNK, left = tensors[t].bytes - at;
        Held h;
        if (passing) load<true>(h, o.in[t] + at, left);
        else load<false>(h, o.in[t] + at, left);
        if (k == blockIdx.x) {
            const double n = norm_of(sums, sum_count, waves), c = (double)most / (n + 1e-6);
            // (a norm that is NaN makes everything so, unless nothing is to be clipped)
            by = most == __builtin_inff() || c > 1.0 ? 1.0f : (float)c;
            exact_by = c;
            if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
        }
        // (nothing to do in place where nothing is clipped)
        if (by == 1.0f && o.in[t] == o.out[t]) continue;
        // (a factor near the end of f32's range, or beyond it, is taken in f64: of huge gradients there it leaves ordinary values)
        if (by < 0x1p-100f) scale(h, dtype, exact_by);
        else if (by != 1.0f) scale(h, dtype, by);
        store(h, o.out[t] + at, left);
    }
}
)HIP";

struct InputsArg {
    const void* in[kGroup];
};
struct BothArg {
    const void* in[kGroup];
    void* out[kGroup];
};

}  // namespace

GradientClip::GradientClip(const int64_t* sizes, const int* dtypes, int count) {
    HE_REQUIRE((size_t)count <= kMostTensors, HE_ERR_UNSUPPORTED, "gradient clip: %d tensors, at most %zu are taken", count, kMostTensors);
    uint64_t all = 0;  // chunks
    for (int k = 0; k < count; k++) {
        HE_REQUIRE(dtypes[k] == HE_F16 || dtypes[k] == HE_BF16 || dtypes[k] == HE_F32, HE_ERR_INVALID, "gradient clip does not take dtype %s", dtype_name(dtypes[k]));
        HE_REQUIRE(sizes[k] >= 0 && sizes[k] < (1ll << 40), HE_ERR_INVALID, "gradient clip: tensor %d has %lld values", k, (long long)sizes[k]);
        const uint64_t size = (uint64_t)sizes[k] * (dtype_bits(dtypes[k]) / 8), chunks = (size + kChunk - 1) / kChunk;
        if (k % kGroup == 0) groups_.push_back({(size_t)k, 0, 0, 0, 0, 0});
        ClipGroup& g = groups_.back();
        HE_REQUIRE(g.chunks + chunks < (1ull << 31), HE_ERR_UNSUPPORTED, "gradient clip: tensors up to %d are too large for one launch", k);
        tensors_.push_back({g.chunks, (uint32_t)dtypes[k], size});
        g.count++;
        g.chunks += (uint32_t)chunks;
        all += chunks;
    }
    const uint64_t total = all;
    for (ClipGroup& g : groups_) {
        // (a group's part of the workgroups is its part of the work)
        g.blocks = (uint32_t)std::min<uint64_t>(g.chunks, std::max<uint64_t>(1, (uint64_t)((double)kBlocks * g.chunks / std::max<uint64_t>(total, 1))));
        g.first_sum = sums_;
        sums_ += g.blocks;
        // (`all` is what is left from this group on)
        g.passing = (uint32_t)(all > kKept ? std::min<uint64_t>(g.chunks, all - kKept) : 0);
        all -= g.chunks;
    }
    std::ostringstream s;
    s << "#define GROUP " << kGroup << "\n#define CHUNK " << kChunk << "\n" << kText;
    source_ = s.str();
    squares_ = std::make_unique<JitKernel>(source_, "clip_squares");
    norm_ = std::make_unique<JitKernel>(source_, "clip_norm");
    scale_ = std::make_unique<JitKernel>(source_, "clip_scale");
    describe_ = strfmt("gradient_clip tensors=%d chunks=%llu groups=%zu sums=%u", count, (unsigned long long)total, groups_.size(), sums_);
    for (const ClipGroup& g : groups_) describe_ += strfmt("\ngroup first=%zu count=%zu chunks=%u blocks=%u first_sum=%u passing=%u", g.first, g.count, g.chunks, g.blocks, g.first_sum, g.passing);
}

GradientClip::~GradientClip() {
    for (auto& kv : per_stream_) {
        (void)hipFree(kv.second.tensors);
        (void)hipFree(kv.second.sums);
    }
}

GradientClip::Buffers GradientClip::buffers(hipStream_t stream) {
    auto it = per_stream_.find(stream);
    if (it != per_stream_.end()) return it->second;
    Buffers b;
    const size_t bytes = std::max<size_t>(1, tensors_.size()) * sizeof(ClipTensor);
    HE_HIP(hipMalloc((void**)&b.tensors, bytes));
    hipError_t e = hipMalloc((void**)&b.sums, std::max(1u, sums_) * sizeof(double));
    if (e == hipSuccess && !tensors_.empty()) e = hipMemcpy(b.tensors, tensors_.data(), bytes, hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        (void)hipFree(b.tensors);
        (void)hipFree(b.sums);
        fail(HE_ERR_HIP, strfmt("gradient clip: workspace: %s", hipGetErrorString(e)));
    }
    per_stream_[stream] = b;
    return b;
}

void GradientClip::check(const char* what, const void* const* addresses) const {
    HE_REQUIRE(addresses || tensors_.empty(), HE_ERR_INVALID, "gradient clip: the list of %s is null", what);
    for (size_t k = 0; k < tensors_.size(); k++)
        HE_REQUIRE(!tensors_[k].bytes || (addresses[k] && (uintptr_t)addresses[k] % (tensors_[k].dtype == HE_F32 ? 4 : 2) == 0), HE_ERR_INVALID,
                   "gradient clip: of the %s, tensor %zu is null or not aligned to its type", what, k);
}

void GradientClip::add_squares(const void* const* gradients, const Buffers& b, hipStream_t stream) {
    const uint32_t block[3] = {256, 1, 1};
    for (const ClipGroup& g : groups_) {
        if (!g.blocks) continue;
        InputsArg o{};
        std::copy(gradients + g.first, gradients + g.first + g.count, o.in);
        const ClipTensor* tensors = b.tensors + g.first;
        uint32_t count = (uint32_t)g.count, chunks = g.chunks, passing = g.passing;
        double* sums = b.sums + g.first_sum;
        const uint32_t grid[3] = {g.blocks, 1, 1};
        void* args[] = {&o, &tensors, &count, &chunks, &passing, &sums};
        squares_->launch(grid, block, 0, stream, args);
    }
}

void GradientClip::write_norm(const Buffers& b, float* norm, hipStream_t stream) {
    const uint32_t one[3] = {1, 1, 1}, block[3] = {256, 1, 1};
    const double* sums = b.sums;
    uint32_t count = sums_;
    void* args[] = {&sums, &count, &norm};
    norm_->launch(one, block, 0, stream, args, true);
}

void GradientClip::norm(const void* const* gradients, float* norm, hipStream_t stream) {
    check("gradients", gradients);
    HE_REQUIRE(norm && (uintptr_t)norm % 4 == 0, HE_ERR_INVALID, "gradient clip: the norm is null or not aligned to 4 bytes");
    std::lock_guard<std::mutex> lk(mu_);
    const Buffers b = buffers(stream);
    add_squares(gradients, b, stream);
    write_norm(b, norm, stream);
}

void GradientClip::clip(const void* const* gradients, void* const* out, float most, float* norm, hipStream_t stream) {
    check("gradients", gradients);
    check("results", out);
    HE_REQUIRE(most >= 0, HE_ERR_INVALID, "gradient clip: a largest norm of %g", (double)most);
    HE_REQUIRE((uintptr_t)norm % 4 == 0, HE_ERR_INVALID, "gradient clip: the norm is not aligned to 4 bytes");
    std::lock_guard<std::mutex> lk(mu_);
    const Buffers b = buffers(stream);
    add_squares(gradients, b, stream);
    if (!sums_ && norm) write_norm(b, norm, stream);
    const uint32_t block[3] = {256, 1, 1};
    for (size_t n = groups_.size(); n-- > 0;) {
        const ClipGroup& g = groups_[n];
        if (!g.blocks) continue;
        BothArg o{};
        std::copy(gradients + g.first, gradients + g.first + g.count, o.in);
        std::copy(out + g.first, out + g.first + g.count, o.out);
        const ClipTensor* tensors = b.tensors + g.first;
        uint32_t count = (uint32_t)g.count, chunks = g.chunks, passing = g.passing, sum_count = sums_;
        const double* sums = b.sums;
        const uint32_t grid[3] = {g.blocks, 1, 1};
        void* args[] = {&o, &tensors, &count, &chunks, &passing, &sums, &sum_count, &most, &norm};
        scale_->launch(grid, block, 0, stream, args, n == 0);
    }
}

}  // namespace he

// ---- C ABI ------------------------------------------------------------------------------------------------
struct he_gradient_clip_s {
    he::GradientClip impl;
    he_gradient_clip_s(const int64_t* sizes, const int* dtypes, int count) : impl(sizes, dtypes, count) {}
};

extern "C" {

int he_gradient_clip_create(he_gradient_clip_t* clip, const int64_t* sizes, const int* dtypes, int count) {
    return he::guard([&] {
        HE_REQUIRE(clip && count >= 0 && (count == 0 || (sizes && dtypes)), HE_ERR_INVALID, "bad argument");
        *clip = new he_gradient_clip_s(sizes, dtypes, count);
    });
}

int he_gradient_clip_destroy(he_gradient_clip_t clip) {
    return he::guard([&] { delete clip; });
}

int he_gradient_norm(he_gradient_clip_t clip, const void* const* gradients, int count, float* norm, he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(clip, HE_ERR_INVALID, "null gradient clip");
        HE_REQUIRE(count == (int)clip->impl.count(), HE_ERR_INVALID, "gradient clip takes %zu tensors, got %d", clip->impl.count(), count);
        clip->impl.norm(gradients, norm, stream ? stream->s : nullptr);
    });
}

int he_gradient_clip(he_gradient_clip_t clip, const void* const* gradients, void* const* out, int count, float most, float* norm, he_stream_t stream) {
    return he::guard([&] {
        HE_REQUIRE(clip, HE_ERR_INVALID, "null gradient clip");
        HE_REQUIRE(count == (int)clip->impl.count(), HE_ERR_INVALID, "gradient clip takes %zu tensors, got %d", clip->impl.count(), count);
        clip->impl.clip(gradients, out, most, norm, stream ? stream->s : nullptr);
    });
}

const char* he_gradient_clip_source(he_gradient_clip_t clip) { return clip ? clip->impl.source().c_str() : ""; }
const char* he_gradient_clip_describe(he_gradient_clip_t clip) { return clip ? clip->impl.describe().c_str() : ""; }

int he_gradient_clip_table(he_gradient_clip_t clip, void* data, size_t capacity, size_t* bytes) {
    return he::guard([&] {
        HE_REQUIRE(clip && bytes && (data || capacity == 0), HE_ERR_INVALID, "bad argument");
        *bytes = clip->impl.tensors().size() * sizeof(he::ClipTensor);
        if (capacity) memcpy(data, clip->impl.tensors().data(), std::min(capacity, *bytes));
    });
}

}  // extern "C"
