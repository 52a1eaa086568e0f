// Root-mean-square norm over rows with a residual's addition, forward (into its own type or 8 bits) and backward, and the quantisation of
// rows to 8 bits, as generated kernels for gfx950.
#pragma once
#include <memory>
#include <mutex>
#include <string>

#include "common.h"
#include "kernels.h"
#include "rtc.h"

namespace he {

struct RowProblem {
    int64_t columns = 0;
    int dtype = HE_F32;
    int residual_dtype = -1;  // -1: none, and what is normalised is the operand itself
    int param_dtype = HE_F32;
    bool to_i8 = false;
    bool norm = true;         // false: rows are only quantised
    float epsilon = 0;
    bool residual() const { return residual_dtype >= 0; }
    int stream_dtype() const { return residual() ? residual_dtype : dtype; }
};

// Bytes of a quantised row: its columns, and zeros up to whole vectors of 16.
inline int64_t quantized_pitch(int64_t columns) { return (columns + 15) / 16 * 16; }

// `lanes` neighbouring threads hold a row, each `vectors` vectors of `vec` values, `lanes` vectors apart.
struct RowTiling {
    int vec = 1, vectors = 1, lanes = 1, threads = 256;
    int rows() const { return threads / lanes; }
    std::string describe() const;
};
RowTiling plan_rows(const RowProblem& pr);

class RmsNorm {
public:
    explicit RmsNorm(const RowProblem& pr);
    ~RmsNorm();
    void forward(int64_t rows, const void* x, const void* gamma, const void* residual, void* new_residual, void* y, float* rstd, float* scales,
                 hipStream_t stream);
    void backward(int64_t rows, const void* dy, const void* h, const void* gamma, const float* rstd, const void* dh, void* dx, void* dresidual,
                  float* dgamma, hipStream_t stream);
    const std::string& source() const { return source_; }
    const std::string& describe() const { return describe_; }

private:
    RowProblem pr_;
    RowTiling tiling_;
    std::string source_, describe_;
    std::unique_ptr<JitKernel> forward_, forward_few_, backward_, backward_more_, fold_;
    std::mutex mu_;  // a backward pass's launches follow each other on their stream: they share the stream's scratch
    ReduceScratch scratch_;
};

}  // namespace he
