// Group norm with an activation over channels-last tensors, forward and backward, as generated kernels for gfx950.
#pragma once
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "common.h"
#include "kernels.h"
#include "rtc.h"

namespace he {

struct GroupNormProblem {
    int64_t batch = 0, pixels = 0, channels = 0, groups = 0;
    int dtype = HE_F32, param_dtype = HE_F32;
    int activation = HE_ACT_NONE;
    float epsilon = 0;
};

// How one pass over the tensor is cut: a workgroup takes `rows` pixels of `slice` channels (whole groups) of one sample and
// holds them in registers; `tx` threads stand side by side along the channels, `threads / tx` pixels below each other.
struct GroupNormTiling {
    bool whole = false;   // a workgroup holds all pixels of its groups
    bool merge = false;   // statistics of so many parts that a launch of their own joins them
    int mergers() const {  // threads of its workgroups
        int n = 64;
        while (n < 1024 && n < chunks) n *= 2;
        return n;
    }
    bool stream = false;  // results bypass the caches on their way to memory
    int vec = 1;          // elements per access
    int threads = 256;
    int slice_groups = 1; // groups per workgroup
    int64_t slice = 0;    // channels per workgroup
    int64_t tx = 1, ty = 1;
    int columns = 1;      // vectors of a pixel that one thread holds
    int rows_per_thread = 1;
    int64_t chunks = 1;   // workgroups along the pixels of a sample
    uint64_t grid = 0;
    int64_t rows() const { return ty * rows_per_thread; }
    std::string describe() const;
};
GroupNormTiling plan_group_norm(const GroupNormProblem& pr, bool backward);

class GroupNorm {
public:
    explicit GroupNorm(const GroupNormProblem& pr);
    ~GroupNorm();
    void forward(const void* x, const void* gamma, const void* beta, void* y, float* mean, float* rstd, hipStream_t stream);
    void backward(const void* dy, const void* x, const void* gamma, const void* beta, const float* mean, const float* rstd, void* dx,
                  float* dgamma, float* dbeta, hipStream_t stream);
    const std::string& source() const { return source_; }
    const std::string& describe() const { return describe_; }

private:
    void check(std::initializer_list<const void*> tensors, std::initializer_list<const void*> params, std::initializer_list<const void*> stats) const;
    void add_levels(float* samples, hipStream_t stream);
    GroupNormProblem pr_;
    std::vector<uint64_t> levels_;
    GroupNormTiling fwd_, bwd_;
    std::string source_, describe_;
    std::unique_ptr<JitKernel> whole_forward_, stats_, merge_, apply_, whole_backward_, parameters_, sums_, fold_, level_, gradient_;
    std::mutex mu_;  // a call's launches follow each other on their stream: they share the stream's scratch
    uint64_t scratch_floats_ = 0;
    ReduceScratch scratch_;
};

}  // namespace he
