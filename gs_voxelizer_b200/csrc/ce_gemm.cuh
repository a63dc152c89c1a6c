// The three matrix products of the linear class loss (ce_gemm.cu), as
// linear_ce.cu asks for them. Operands are 16-bit matrices in "planes": one
// for bf16 / fp16 inputs; three bf16 planes whose sum is the float32 value
// for float32 inputs (8 + 8 + 8 significant bits), multiplied pair by pair.
#pragma once

#include "ce.cuh"

namespace gsv {

enum CeProduct {
    kCeScores = 0,  // X W^T, kept as a (max, sum) pair per row and class tile
    kCeProbs = 1,   // X W^T, stored as the loss's derivative in the scores
    kCeGradX = 2,   // P W: accumulated for the features
    kCeGradW = 3,   // P^T X: accumulated for the table
};

// rows x cols, cols contiguous; plane p starts at ptr + p * plane (elements).
// ld, plane and ptr keep 16-byte alignment.
struct CeMat {
    const void *ptr;
    long long rows, cols, ld, plane;
};

struct CeGemm {
    int product;
    bool bf16;
    int planes;         // 1 or 3
    CeMat X;            // kCeScores, kCeProbs: [rows, D]; kCeGradW: [rows, D]
    CeMat W;            // [V, D]
    CeMat P;            // [rows of the piece, classes of the piece]
    long long row0;     // first row of the piece within the packed rows
    long long rows;     // rows of the piece
    int v0, nv;         // classes of the piece
    int V, D;
    const int *count;   // packed rows in use (device), or null: all of them

    // rows: packed class (>= 0, kCeInvalid, kCeIgnored), or raw labels
    const int *lab;
    const long long *labels;
    const int *idx;     // packed row -> original row (lse is by original row)
    CeOpt opt;

    // kCeScores
    float2 *part;       // [tiles][rows] (max, sum)
    float *psum;        // [tiles][rows] plain sums (label smoothing) or null
    float *zt;          // [rows] score of the row's class
    // kCeProbs
    const float *lse;
    void *p_out;        // P's storage (P describes it)
    float p_scale;      // stored = p_scale * derivative
    // kCeGradX, kCeGradW: out[split][m][D] (+)= product
    float *out;
    long long out_split;  // elements between splits
    int splits;
    bool add;
};

constexpr int kCeTileM = 128;    // packed rows come in whole tiles of these
constexpr int kCeScoreTile = 64; // classes behind one (max, sum) pair

cudaError_t launch_ce_gemm(const CeGemm &g, cudaStream_t stream);

}  // namespace gsv
