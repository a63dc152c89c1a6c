// The three matrix products of the linear class loss (ce_gemm.cu), as
// linear_ce.cu asks for them. Operands are 16-bit matrices in "planes": one
// for bf16 / fp16 inputs; three bf16 planes whose sum is the float32 value
// for float32 inputs (8 + 8 + 8 significant bits), multiplied pair by pair.
#pragma once

#include "ce.cuh"

namespace gsv {

enum CeProduct {
    kCeScores = 0,  // X W^T, kept as (maximum, sum) pairs
    kCeProbs = 1,   // X W^T, stored as the loss's derivative in the scores
    kCeGradX = 2,   // P W
    kCeGradW = 3,   // P^T X
};

// rows x cols, cols contiguous; plane p starts at ptr + p * plane (elements).
// ptr, ld and plane keep 16-byte alignment.
struct CeMat {
    const void *ptr;
    long long rows, cols, ld, plane;
};

// Factor of the summed gradients. With reduction "none" each row's upstream
// gradient is in P already, over the largest finite one (gmax) in fp16.
struct CeUpstream {
    const float *g;      // [1]
    const float *count;  // labelled rows, at least 1
    const float *gmax;   // or null
    float inv_p;         // 1 / p_scale
    int reduction;
    const float *zmax = nullptr;  // largest factor of the z-loss
};

// The power of two from the largest factor of the z-loss on (up to 2^127), over
// which P is kept: another factor would round derivatives near 1 and 1/2, the
// most frequent ones, more coarsely (2.6e-4 of the gradients for 2.4e-4).
__device__ __forceinline__ float ce_z_scale(const CeUpstream &u) {
    if (!u.zmax) return 1.f;
    const int up = (__float_as_int(fmaxf(*u.zmax, 1.f)) + 0x7fffff) & 0x7f800000;
    return __int_as_float(min(up, 0x7f000000));
}

__device__ __forceinline__ float ce_grad_scale(const CeUpstream &u) {
    const float inv = u.inv_p * ce_z_scale(u);
    if (u.reduction == kCeNone) return (u.gmax && *u.gmax > 0.f ? *u.gmax : 1.f) * inv;
    return (u.reduction == kCeMean ? u.g[0] / u.count[0] : u.g[0]) * inv;
}

struct CeGemm {
    int product;
    bool bf16;
    int planes;         // 1 or 3
    CeMat X;            // [rows, D]
    CeMat W;            // [V, D]
    CeMat P;            // [rows of the piece, classes of the piece]
    long long row0;     // first row of the piece within X
    long long rows;     // rows of the piece
    int v0, nv;         // classes of the piece
    int V, D;
    const int *count;   // rows of X in use (device), or null: rows

    // a row's class: packed (lab), or from the caller's labels
    const int *lab;
    const long long *labels;
    const int *idx;     // packed row -> original row, or null
    CeOpt opt;

    // kCeScores: class tiles in `runs` runs
    int runs;
    float2 *part;       // [2 * runs][rows] (maximum, sum)
    float *psum;        // [2 * runs][rows] plain sums (label smoothing) or null
    float *zt;          // [rows] score of the row's class
    // kCeProbs: derivative * p_scale / z_scale * (row's upstream gradient / gmax)
    const float2 *lse;  // as X's rows
    void *p_out;        // P's storage (P describes it)
    float p_scale;
    const float *grow;  // upstream gradient by original row, or null
    const float *gmax;  // or null
    // kCeGradX, kCeGradW: acc[split][m][acc_ld] (+)= product, or, with dst set,
    // dst[row of m][D] = scale * product in the inputs' type
    float *acc;
    long long acc_ld;     // elements between rows: D in whole 16-byte words
    long long acc_split;  // elements between splits
    int splits;
    bool add;
    void *dst;
    CeUpstream up;
};

constexpr int kCeTileM = 256;     // rows a tile: packed rows come in whole tiles
constexpr int kCeTileN = 256;     // classes (or channels) a tile, at most
constexpr int kCePairs = kSMs / 2;  // tiles in flight: a pair of SMs each

// runs of class tiles for the forward: (rows of) partial sums and balance
int ce_runs(long long rows, int V, bool f32);
// columns of a gradient's tile
int ce_grad_tile(int cols, bool f32);

cudaError_t launch_ce_gemm(const CeGemm &g, cudaStream_t stream);

}  // namespace gsv
