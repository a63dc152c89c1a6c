// Linear class loss of a few rows, without a gradient (linear_ce_few.cu).
#pragma once

#include "ce.cuh"

namespace gsv {

constexpr int kFewRows = 8;  // rows at most (float32; 4 of 16 bits)

struct FewArgs {
    int N, V, D;
    const void *features, *weight;
    const long long *labels;
    CeOpt opt;
    float *count;
};

size_t few_workspace_bytes(int N, int V);
cudaError_t launch_few_forward(const FewArgs &a, int type, float *loss, void *workspace,
                               cudaStream_t st);

}  // namespace gsv
