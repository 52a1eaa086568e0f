// Orthogonalised updates of a group of matrices (Newton-Schulz products) and the optimizer step built on them.
#pragma once
#include <array>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "common.h"
#include "rtc.h"

namespace he {

struct MuonProblem {
    std::vector<std::array<int64_t, 2>> shapes;  // rows, columns
    int dtype = HE_F32;                          // of the matrices that come in (and of orthogonalised ones that go out)
    bool split = true;                           // f32_f32, and f16 matrices: f16 operands in two parts; otherwise in one
    int steps = 5;
};

// What the kernels know of a matrix; the device holds an array of these. The smaller extent is m, the larger n, both padded to whole
// blocks of 64 with zeros (which every product leaves zeros): X is [mp][np], XT its transpose. `at`: where its buffers lie in the workspace.
struct MuonMatrix {
    uint32_t rows, cols, mp, np;
    uint32_t tall, first_part, parts;  // parts: shares of the sum of squares
    float shape_scale;                 // sqrt(max(1, rows / cols))
    static constexpr int kBuffers = 9;
    uint64_t at[kBuffers];  // X, its transpose (twice, in turn), A, B, C, Q (twice), and what f16 drops of X where operands are of one part
};
// A workgroup's part of the conversions: a share of the sum of squares (i), or the 64 x 64 values at (i, j).
struct MuonBlock {
    uint32_t matrix, i, j;
};
// A workgroup's part of a product: k-tiles k_begin .. k_end - 1 of the tile (i, j), share `share` of `shares`; those of a tile that
// several work on are parked at `slot` onwards.
struct MuonTask {
    uint32_t matrix, i, j, k_begin, k_end, slot, share, shares;
};

// R = c1 E1 + c2 E2 + cs P Q^T + ci I of one matrix: operands and results by their offsets in the workspace; parked_at: where the
// product's shares wait, in floats.
struct MuonProduct {
    uint32_t mp, np;
    float c1, c2, cs, ci;
    uint64_t p, q, e1, e2, out, turned, low, parked_at;
};

struct MuonStep {
    float learning_rate, momentum, weight_decay;
    int32_t nesterov;
};

// Whether several steps may be taken at a time (HE_OPT_MUON_SEVERAL_STEPS).
void set_muon_several_steps(bool may);

class Muon {
public:
    explicit Muon(const MuonProblem& pr);
    ~Muon();
    void orthogonalize(const void* const* in, void* const* out, hipStream_t stream);
    void step(const void* const* grads, const float* const* momenta, const float* const* weights, float* const* new_momenta,
              float* const* new_weights, const MuonStep& how, hipStream_t stream);
    const std::string& source() const { return source_; }
    const std::string& describe() const { return describe_; }
    size_t count() const { return pr_.shapes.size(); }
    // The tables the kernels read, as bytes: 0 matrices, 1 to 3 tasks of the three products, 4 to 6 those of their tiles that several
    // workgroups share, 7 shares of the sums of squares, 8 blocks of the conversions, 9 what the launches compute
    // (a MuonProduct per matrix and product).
    static constexpr int kTables = 10;
    const std::vector<char>& table(int which) const { return tables_[which]; }

private:
    struct Buffers {
        char* tables = nullptr;
        char* workspace = nullptr;
    };
    Buffers buffers(hipStream_t stream);
    void step_or_not(const void* const* in, const float* const* momenta, const float* const* weights, float* const* new_momenta, void* const* out,
                     const MuonStep* how, hipStream_t stream);
    void products(char* ws, char* tables, hipStream_t stream);
    MuonProblem pr_;
    std::vector<MuonMatrix> matrices_;
    std::vector<char> tables_[kTables];
    size_t table_at_[kTables] = {}, table_bytes_ = 0, workspace_bytes_ = 0, shared_at_ = 0;
    uint32_t shares_ = 0;
    struct ProductKind {
        uint32_t grid = 0, threads = 0, join_grid = 0, parked = 0;
        double estimate = 0;
        std::string text;
        std::unique_ptr<JitKernel> kernel, join;
    } products_[3];
    struct Launch {
        int kind;
        uint32_t count;      // products
        size_t products_at;  // in table 9
    };
    std::vector<Launch> launches_;
    std::string launches_text_;
    std::vector<int> choose_runs() const;
    void plan_launches(const std::vector<int>& runs);
    std::vector<uint32_t> part_begin_, block_begin_;  // per matrix: first entry of tables 7 and 8
    std::string source_, describe_;
    std::unique_ptr<JitKernel> norm_, convert_, finish_, norm_step_, convert_step_, finish_step_;
    std::mutex mu_;
    std::map<hipStream_t, Buffers> per_stream_;
};

}  // namespace he
