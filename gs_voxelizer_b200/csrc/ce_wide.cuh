// Linear class loss of few classes and many float32 channels
// (linear_ce_wide.cu).
#pragma once

#include "ce_narrow.cuh"

namespace gsv {

constexpr int kWideV = 16;  // classes at most
// rows at least: blocks of 256 that walk all channels, 32 at a time, take 92 us
// forward for 1000 channels, however few they are
constexpr long long kWideRows = 16384;

struct WideShape {
    int row_blocks;            // forward: persistent blocks
    int dw_chunks, dx_blocks;  // channel chunks x row blocks
    int dw_blocks;             // those of dW: parts
};
WideShape wide_shape(long long N, int V, int D);
// of scores and of derivatives: [N][V rounded up to 4]
inline size_t wide_p_bytes(long long N, int V) {
    return sizeof(float) * (size_t)N * ((V + 3) / 4 * 4);
}

// loss (one block) or per-block sums; the (capped) scores, if z is not null
cudaError_t launch_wide_fwd(const NarrowArgs &a, float *z, float *loss, float2 *sums,
                            cudaStream_t st);
cudaError_t launch_wide_probs(const NarrowArgs &a, const CeUpstream &u, const float *z, float *p,
                              cudaStream_t st);
cudaError_t launch_wide_dx(const NarrowArgs &a, const float *p, float *grad, cudaStream_t st);
// acc [dw_blocks][V][D]
cudaError_t launch_wide_dw(const NarrowArgs &a, const float *p, float *acc, cudaStream_t st);

}  // namespace gsv
