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

// How one workgroup works. Tiles: waves_n x waves_m waves make tile_n channels of tile_m tokens from operands in LDS. Streams (few tokens): the waves
// of a workgroup share the sums of 16 blocks_n channels of 16 blocks_m tokens and read their operands straight into registers.
struct Int8Shape {
    int tile_n = 0, tile_m = 0, waves_n = 0, waves_m = 0, stages = 0, per_cu = 1;  // of tiles
    int ahead = 1;  // k-steps whose operands are read from LDS ahead of the matrix instructions: 1 or 2 (a k-tile has 4)
    double base = 0, alone = 0, full = 0, round = 0;  // microseconds: of a call; of a k-tile on a CU of its own, and on a full one; of another round of workgroups
    int blocks_n = 0, blocks_m = 0, waves = 0, steps = 0;  // of streams
    bool stream() const { return blocks_n > 0; }
    int channels() const { return stream() ? 16 * blocks_n : tile_n; }
    int tokens() const { return stream() ? 16 * blocks_m : tile_m; }
    int threads() const { return 64 * (stream() ? waves : waves_n * waves_m); }
};
// How one call is cut: which of the shapes, and into how many shares each sum, which a second launch adds up.
struct Int8Cut {
    int shape = 0;
    uint32_t shares = 1;
    uint64_t blocks = 0;  // of one share
    double estimate = 0;  // microseconds
    std::string describe() const;
};
Int8Cut plan_int8(const Int8Problem& pr, int64_t tokens);

// The kernels for one type of result: they know no sizes, and all products have them in common.
struct Int8Kernels;

class Int8Matmul {
public:
    explicit Int8Matmul(const Int8Problem& pr);
    void multiply(int64_t tokens, const void* x, const float* x_scales, const void* weights, const float* weight_scales, const float* bias, void* y,
                  hipStream_t stream);
    const std::string& source() const;
    std::string describe(int64_t tokens) const { return plan_int8(pr_, tokens).describe(); }

private:
    Int8Problem pr_;
    std::shared_ptr<Int8Kernels> kernels_;
};

}  // namespace he
