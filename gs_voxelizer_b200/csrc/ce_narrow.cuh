// Linear class loss of few channels (linear_ce_narrow.cu).
#pragma once

#include "ce_gemm.cuh"

namespace gsv {

constexpr int kNarrowD = 8;  // channels at most

struct NarrowArgs {
    long long N;
    int V, D;
    const void *features, *weight;
    const long long *labels;
    CeOpt opt;
    float2 *lse;   // by row
    float *count;  // labelled rows, at least 1
};

int narrow_class_splits(long long N, int V, int D);
long long narrow_fwd_blocks(long long N, int D);
int narrow_dw_splits(long long N, int V, int D);

// One class split: lse, per-block sums (several blocks) or the loss itself.
// Several: part [splits][N], psum, zt, to be merged.
template <typename T>
cudaError_t launch_narrow_fwd(const NarrowArgs &a, float *loss, float2 *sums, float2 *part,
                              float *psum, float *zt, cudaStream_t st);
// One class split: grad [N][D]. Several: acc [splits][N][D].
template <typename T>
cudaError_t launch_narrow_dx(const NarrowArgs &a, const CeUpstream &u, void *grad, float *acc,
                             cudaStream_t st);
// acc [narrow_dw_splits][V][D]
template <typename T>
cudaError_t launch_narrow_dw(const NarrowArgs &a, const CeUpstream &u, float *acc,
                             cudaStream_t st);

}  // namespace gsv
