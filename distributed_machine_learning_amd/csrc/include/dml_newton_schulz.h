// Orthogonalisation of matrices by Newton-Schulz products, and the Muon update built on it.
//
//   Y_0 = X / (||X||_F + eps);   per step:  A = Y Y^T,  B = b A + c A A,  Y <- a Y + B Y
//
// with Y the [m, n] matrix of the smaller dimension first (the map is odd in X, so working on the
// transpose gives the transposed result).  All matrices of one call share every launch: a plan
// holds their shapes, a kernel finds its matrix from its block number in a table passed by value,
// so nothing is uploaded, allocated or synchronised and a call can be captured into a hipGraph.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <memory>
#include <string>
#include <vector>

namespace dml {

// Element types of the matrices of `orthogonalize` (the update's are fp32).
enum NsType : int { NS_F32 = 0, NS_BF16 = 1, NS_F16 = 2 };

// One matrix, or a batch of equal ones, as it lies in memory: `rows` rows of `cols` contiguous
// elements, `ld` elements from row to row and `stride` from matrix to matrix.
struct NsShape {
    int rows = 0, cols = 0, batch = 1;
    long long offset = 0, ld = 0, stride = 0;                // source (and the update's weights)
    long long out_offset = 0, out_ld = 0, out_stride = 0;    // result of `orthogonalize`
    float lr = 0.f;                                          // the update's step for this matrix / lr
};

// Elements [offset, offset + count) of the flat buffers that SGD with momentum updates.
struct NsSegment {
    long long offset = 0, count = 0;
};

struct MuonArgs {
    float lr = 0.f, momentum = 0.f, weight_decay = 0.f;      // matrices
    bool nesterov = true;
    float sgd_lr = 0.f, sgd_momentum = 0.f, sgd_weight_decay = 0.f;      // segments
    float grad_scale = 1.f;
};

// A launch of a plan as it was chosen.
struct NsLaunchInfo {
    std::string kernel, tile;
    unsigned blocks = 0, threads = 0;
    unsigned whole = 0, joined = 0;      // tiles that one block makes; tiles joined from several blocks' parts
};

class NewtonSchulzPlan {
  public:
    // `coefficients`: one (a, b, c) per step.  `wide_products`: keep 22 bits of every factor of a
    // matrix product (two fp16 terms, three products) instead of 11.
    NewtonSchulzPlan(const std::vector<NsShape>& shapes, const std::vector<NsSegment>& segments,
                     const std::vector<float>& coefficients, double eps, bool wide_products);
    size_t workspace_bytes() const { return ws_bytes_; }
    // The preparing launches and those of one step, for every set of matrices that shares launches.
    std::vector<NsLaunchInfo> launches() const;
    // out = NewtonSchulz(x); the workspace (256-byte aligned) holds no state between calls.
    void orthogonalize(const void* x, void* out, NsType type, void* ws, size_t ws_bytes,
                       hipStream_t stream) const;
    // m <- mu m + g,  u = g + mu m (or m),  p <- (1 - lr wd) p - lr shape.lr NewtonSchulz(u)  for
    // the matrices;  g' = g + wd p, m <- mu m + g', p <- p - lr m  for the segments.
    void muon(float* p, const float* g, float* m, const MuonArgs& a, void* ws, size_t ws_bytes,
              hipStream_t stream) const;

  private:
    struct Group;                    // the launches of as many matrices as a launch takes
    struct Op;                       // one product of the chain
    void check_workspace(const void* ws, size_t ws_bytes) const;
    struct Solo;                     // one block per matrix
    template <typename T, bool MUON>
    void launch_solo(const Group& g, const void* x, const void* update, const void* result,
                     hipStream_t stream) const;
    template <typename T, bool MUON, int ROWS>
    void launch_solo_rows(const Group& g, const void* x, const void* update, const void* result,
                     hipStream_t stream) const;
    template <typename Prepare, typename SoloRun>
    void chain(char* ws, NsType type, const Prepare& prepare, const SoloRun& solo, void* out, float* p,
               float lr, float decay, hipStream_t stream) const;

    std::vector<NsSegment> segs_;
    std::vector<float> coef_;
    double eps_;
    bool wide_, fused_ = false;
    int x_exp_;                      // Y's planes hold value * 2^exp
    std::vector<std::shared_ptr<Op>> ops_;
    std::shared_ptr<Solo> solo_;
    std::vector<std::shared_ptr<Group>> groups_;
    size_t partials_ = 0, slab_ = 0, ws_bytes_ = 0;      // offsets in the workspace, its size
};

}  // namespace dml
