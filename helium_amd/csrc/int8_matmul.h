// Products of quantised matrices (8-bit whole numbers, a scale for each row of either operand), as generated kernels for gfx950.
#pragma once
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "common.h"
#include "kernels.h"
#include "rtc.h"

namespace he {

struct Int8Problem {
    int64_t inputs = 0, channels = 0;
    int dtype = HE_F32;  // of the result
};

// How one call is cut. Tiles: workgroups of waves_n x waves_m waves make tile_n channels of tile_m tokens each from operands in LDS, `shares`
// of them taking a part of the sum each. Streams (few tokens): the waves of a workgroup share the sum of 16 blocks_n channels of 16 blocks_m
// tokens and read their operands straight into registers.
struct Int8Shape {
    bool stream = false;
    int tile_n = 0, tile_m = 0, waves_n = 0, waves_m = 0, stages = 0, per_cu = 1;  // of tiles
    int blocks_n = 0, blocks_m = 0, waves = 0;                                      // of streams
    int channels() const { return stream ? 16 * blocks_n : tile_n; }
    int tokens() const { return stream ? 16 * blocks_m : tile_m; }
    static constexpr int kSharedTile = 128 * 128;  // the largest whose sum may be shared out
    bool can_share() const { return !stream && tile_n * tile_m <= kSharedTile; }
    int threads() const { return 64 * (stream ? waves : waves_n * waves_m); }
};
struct Int8Cut {
    int shape = 0;        // which of the shapes
    uint32_t shares = 1;
    uint64_t blocks = 0;  // of one share
    std::string describe(const Int8Problem& pr) const;
};
Int8Cut plan_int8(const Int8Problem& pr, int64_t tokens);

class Int8Matmul {
public:
    explicit Int8Matmul(const Int8Problem& pr);
    ~Int8Matmul();
    void multiply(int64_t tokens, const void* x, const float* x_scales, const void* weights, const float* weight_scales, const float* bias, void* y,
                  hipStream_t stream);
    const std::string& source() const { return source_; }
    std::string describe(int64_t tokens) const { return plan_int8(pr_, tokens).describe(pr_); }

private:
    struct Kernels {
        std::unique_ptr<JitKernel> product, join;
    };
    Int8Problem pr_;
    std::string source_;
    std::vector<Kernels> kernels_;
    std::mutex mu_;  // a call's launches follow each other on their stream: they share the stream's scratch
    ReduceScratch scratch_;
};

}  // namespace he
