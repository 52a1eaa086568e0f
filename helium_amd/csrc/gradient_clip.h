// The norm of all gradients of a model together, and the gradients scaled down to it, as generated kernels for gfx950.
#pragma once
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "common.h"
#include "kernels.h"
#include "rtc.h"

namespace he {

// What the kernels know of a tensor; the device holds an array of these.
struct ClipTensor {
    uint32_t first;  // chunk of its group
    uint32_t dtype;
    uint64_t bytes;
};
// Tensors whose addresses one launch takes: their chunks, of 16 KB each, are dealt to `blocks` workgroups, whose sums lie from `first_sum` on; the
// first `passing` chunks are read past the caches, which later ones fill.
struct ClipGroup {
    size_t first, count;
    uint32_t chunks, blocks, first_sum, passing;
};

class GradientClip {
public:
    GradientClip(const int64_t* sizes, const int* dtypes, int count);
    ~GradientClip();
    void norm(const void* const* gradients, float* norm, hipStream_t stream);
    void clip(const void* const* gradients, void* const* out, float most, float* norm, hipStream_t stream);
    size_t count() const { return tensors_.size(); }
    const std::string& source() const { return source_; }
    const std::string& describe() const { return describe_; }
    // The array of ClipTensor, as bytes.
    const std::vector<ClipTensor>& tensors() const { return tensors_; }

private:
    struct Buffers {
        ClipTensor* tensors = nullptr;
        double* sums = nullptr;
    };
    Buffers buffers(hipStream_t stream);
    void check(const char* what, const void* const* addresses) const;
    void add_squares(const void* const* gradients, const Buffers& b, hipStream_t stream);
    void write_norm(const Buffers& b, float* norm, hipStream_t stream);
    std::vector<ClipTensor> tensors_;
    std::vector<ClipGroup> groups_;
    uint32_t sums_ = 0;
    std::string source_, describe_;
    std::unique_ptr<JitKernel> squares_, norm_, scale_;
    std::mutex mu_;  // a call's launches follow each other on their stream: they share its sums
    std::map<hipStream_t, Buffers> per_stream_;
};

}  // namespace he
