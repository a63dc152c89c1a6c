// Linear class loss of few channels on the CUDA cores (linear_ce_narrow.cu).
#pragma once

#include <type_traits>

#include "ce_gemm.cuh"

namespace gsv {

constexpr int kNarrowD = 32;  // channels at most
constexpr int kNarrowNT = 256;

struct NarrowArgs {
    long long N;
    int V, D;
    const void *features, *weight;
    const long long *labels;
    CeOpt opt;
    float2 *lse;   // by row
    float *count;  // labelled rows, at least 1

    // whether rows are whole wide words: D = 4, 8, 16 or 32 and every base
    // aligned to them (16 bytes at most)
    bool wide_rows(size_t size, const void *grad) const {
        const uintptr_t mask = std::min<size_t>(16, D * size) - 1;
        return (D == 4 || D == 8 || D == 16 || D == 32) &&
               ((reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(weight) |
                 reinterpret_cast<uintptr_t>(grad)) & mask) == 0;
    }
};

// Blocks of the kernels: rows x class splits (forward, dX), row blocks x
// class chunks (dW, whose parts are as many as its row blocks).
struct NarrowShape {
    int class_splits;
    long long row_blocks;
    int dw_lanes, dw_chunks, dw_blocks;
};
NarrowShape narrow_shape(long long N, int V, int D);

// One class split: lse, per-block sums (several blocks) or the loss itself.
// Several: part [splits][N], psum, zt, to be merged.
template <typename T>
cudaError_t launch_narrow_fwd(const NarrowArgs &a, float *loss, float2 *sums, float2 *part,
                              float *psum, float *zt, cudaStream_t st);
// One class split: grad [N][D]. Several: acc [splits][N][D].
template <typename T>
cudaError_t launch_narrow_dx(const NarrowArgs &a, const CeUpstream &u, void *grad, float *acc,
                             cudaStream_t st);
// acc [dw_blocks][V][D]
template <typename T>
cudaError_t launch_narrow_dw(const NarrowArgs &a, const CeUpstream &u, float *acc,
                             cudaStream_t st);
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

template <int DP>
struct alignas(16) Row {
    float v[DP];
};
// Row r of a [., D] matrix. VEC: D = DP and rows aligned to their size (or
// 16 bytes), so that a row is one or two wide accesses.
template <typename T, int DP, bool VEC>
__device__ __forceinline__ Row<DP> load_row(const T *p, long long r, int D) {
    constexpr int kBytes = DP * sizeof(T);
    Row<DP> x;
    if constexpr (VEC) {
        struct alignas(kBytes < 16 ? kBytes : 16) Raw { T t[DP]; };
        const Raw q = reinterpret_cast<const Raw *>(p)[r];
#pragma unroll
        for (int d = 0; d < DP; ++d) x.v[d] = ce_to_float(q.t[d]);
    } else {
        const T *q = p + r * D;
#pragma unroll
        for (int d = 0; d < DP; ++d) x.v[d] = d < D ? ce_to_float(q[d]) : 0.f;
    }
    return x;
}

template <typename T, int DP, bool VEC>
__device__ __forceinline__ void store_row(T *p, long long r, int D, const float (&v)[DP]) {
    constexpr int kBytes = DP * sizeof(T);
    if constexpr (VEC) {
        struct alignas(kBytes < 16 ? kBytes : 16) Raw { T t[DP]; };
        Raw q;
#pragma unroll
        for (int d = 0; d < DP; ++d) q.t[d] = ce_from_float<T>(v[d]);
        reinterpret_cast<Raw *>(p)[r] = q;
    } else {
#pragma unroll
        for (int d = 0; d < DP; ++d)
            if (d < D) p[r * D + d] = ce_from_float<T>(v[d]);
    }
}

struct Span {
    int v0, v1;
};
__device__ __forceinline__ Span class_span(int V) {
    return {(int)((long long)V * blockIdx.y / gridDim.y),
            (int)((long long)V * (blockIdx.y + 1) / gridDim.y)};
}

// Sum of a span of the table, by every thread the same, in shared memory.
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void table_sum(Row<DP> &out, Row<DP> *sh, const T *w, Span span, int D) {
    Row<DP> a;
#pragma unroll
    for (int d = 0; d < DP; ++d) a.v[d] = 0.f;
    for (int j = span.v0 + threadIdx.x; j < span.v1; j += kNarrowNT) {
        const Row<DP> r = load_row<T, DP, VEC>(w, j, D);
#pragma unroll
        for (int d = 0; d < DP; ++d) a.v[d] += r.v[d];
    }
#pragma unroll
    for (int d = 0; d < DP; ++d)
#pragma unroll
        for (int k = 16; k; k >>= 1) a.v[d] += __shfl_xor_sync(0xffffffffu, a.v[d], k);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
    __syncthreads();
    a = sh[0];
    for (int k = 1; k < kNarrowNT / 32; ++k)
#pragma unroll
        for (int d = 0; d < DP; ++d) a.v[d] += sh[k].v[d];
    out = a;
}

// Scores are exponents of two where there is no cap (the table times log2 e),
// and natural where there is one; so are the maxima that are kept.
template <bool CAP>
__device__ __forceinline__ float unit() { return CAP ? 1.f : kLog2e; }
template <bool CAP>
__device__ __forceinline__ float exp_of(float d) { return ex2(CAP ? d * kLog2e : d); }

// A row's part of the derivative: (kz prob - e - hit at its class), all with
// the row's upstream gradient in them.
struct RowGrad {
    float2 lse;
    float kz, e, hit;
};

// the upstream gradient that all rows share (a mean's divided by the count)
__device__ __forceinline__ float common_grad(const CeUpstream &u) {
    return u.reduction == kCeNone ? 0.f
           : u.reduction == kCeMean ? u.g[0] / u.count[0]
                                    : u.g[0];
}

template <bool CAP>
__device__ __forceinline__ RowGrad row_grad(long long r, int y, float2 lse, const CeOpt &o,
                                            const float *per_row, float common, float smooth) {
    RowGrad q{make_float2(0.f, 0.f), 0.f, 0.f, 0.f};
    if (y == kCeIgnored) return q;
    q.lse = lse;
    const float g = per_row ? per_row[r] : common;
    q.kz = g;
    if (o.zeta > 0.f)
        q.kz *= 1.f + 2.f * o.zeta * ce_lse(make_float2(CAP ? q.lse.x : q.lse.x * kCeLn2,
                                                       q.lse.y));
    q.e = smooth * g;
    q.hit = (1.f - o.eps) * g;
    return q;
}

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

}  // namespace gsv
