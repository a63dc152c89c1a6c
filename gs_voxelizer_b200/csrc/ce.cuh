// Shared pieces of the class losses (softmax_ce.cu, linear_ce*.cu, ce_gemm.cu).
//
// With z_ij the scores of row i (capped: z = c tanh(s / c) when c > 0),
//     lse_i  = log sum_j exp z_ij
//     loss_i = lse_i - (1 - eps) z_iy - eps / V sum_j z_ij + zeta lse_i^2
//     dloss_i / dz_ij = (1 + 2 zeta lse_i) exp(z_ij - lse_i)
//                       - (1 - eps) [j = y_i] - eps / V
// and, through the cap, ds = dz (1 - (z / c)^2). Scores, maxima, sums and
// losses are float32 whatever the type of the inputs.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace gsv {

enum CeType { kCeF32 = 0, kCeBf16 = 1, kCeF16 = 2 };
enum CeReduction { kCeNone = 0, kCeSum = 1, kCeMean = 2 };
// Directions of the linear loss: a forward without a backward to follow, one
// that leaves a state, the backward.
enum CeCall { kCeForwardOnly, kCeForward, kCeBackward };

// Options of a class loss, by value into the kernels.
struct CeOpt {
    long long ignore;
    float eps, cap, zeta;
    int reduction;
};

// What a row's label stands for: a class >= 0, or one of these.
constexpr int kCeInvalid = -1;  // outside [0, V): the row's loss is NaN
constexpr int kCeIgnored = -2;  // no label: the row takes no part

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kCeLn2 = 0.6931471805599453f;

__device__ __forceinline__ int ce_label(long long y, long long ignore, int V) {
    if (y == ignore) return kCeIgnored;
    return (unsigned long long)y < (unsigned long long)V ? (int)y : kCeInvalid;
}

__device__ __forceinline__ float ce_nan() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ float ce_neg_inf() { return __int_as_float(0xff800000); }

// tanh(s / cap). FAST (16-bit inputs): 1 - 2 / (1 + e^2x) on the
// special-function unit, off by at most 2^-22, and below 0.1, where that would
// be too much of a large cap's scores, the series to x^5 (off by 2^-24 x);
// float32 inputs take tanhf. The slope 1 - tanh^2 is off by twice as much: of
// scores beyond four caps it is below 2^-9 and keeps few digits of its own.
template <bool FAST>
__device__ __forceinline__ float ce_tanh(float s, float cap) {
    if (!FAST) return tanhf(s / cap);
    const float x = __fdividef(s, cap), x2 = x * x;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(fabsf(x) * (2.f * kLog2e))));
    const float far = copysignf(fmaf(-2.f, r, 1.f), x);
    const float near = x * fmaf(x2, fmaf(x2, 2.f / 15.f, -1.f / 3.f), 1.f);
    return fabsf(x) < 0.1f ? near : far;
}

// log2 of a sum of exponentials that holds its largest term, 1: s >= 1 (or 0 or
// NaN). The special-function unit's own is off by 2^-22 near 1, where a
// confident row's loss is smaller than that, and log2f takes 5 % of a pass over
// four classes. s = 2^e m, m in [0.75, 1.5); log2 m = 2 / ln 2 atanh(u) with
// u = (m - 1) / (m + 1), |u| <= 1/5, by its series to u^9 (2^-28 of it left);
// off by 2^-22 of log2 m and the last addition.
__device__ __forceinline__ float ce_log2(float s) {
    const int e = (__float_as_int(s) - 0x3f400000) >> 23;
    const float m = __int_as_float(__float_as_int(s) - (e << 23));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(m + 1.f));
    const float u = (m - 1.f) * r, u2 = u * u;
    float p = fmaf(u2, 2.f / 9.f * kLog2e, 2.f / 7.f * kLog2e);
    p = fmaf(p, u2, 2.f / 5.f * kLog2e);
    p = fmaf(p, u2, 2.f / 3.f * kLog2e);
    p = fmaf(p, u2, 2.f * kLog2e);
    return s >= 1.f ? fmaf(p, u, (float)e) : __log2f(s);
}

// Running maximum m, sum of exp(z - m) and plain sum of a row's scores. The
// difference is taken before the product with log2 e: a maximum that stays
// rescales by exactly 1, and rows of huge scores keep their digits.
struct CeAcc {
    float m, s, sz;
    __device__ __forceinline__ void init() {
        m = ce_neg_inf();
        s = 0.f;
        sz = 0.f;
    }
    // m stays -inf while every score is -inf: exponents are taken against 0
    // then, so that each term is exp(-inf) = 0 and not NaN
    __device__ __forceinline__ static float base(float m) {
        return m == ce_neg_inf() ? 0.f : m;
    }
    // LOG2: the scores are exponents of two already
    template <bool LOG2 = false>
    __device__ __forceinline__ void merge(float om, float os, float osz) {
        constexpr float k = LOG2 ? 1.f : kLog2e;
        const float nm = fmaxf(m, om), e = base(nm);
        s = s * ex2((m - e) * k) + os * ex2((om - e) * k);
        m = nm;
        sz += osz;
    }
    // A row's logsumexp, kept as (maximum, log2 of the sum): of scores at the
    // type's lowest value the one alone would lose the other.
    __device__ __forceinline__ float2 lse() const { return make_float2(base(m), log2f(s)); }
};

__device__ __forceinline__ float ce_lse(float2 l) { return fmaf(l.y, kCeLn2, l.x); }

// What the z-loss brings to a row's derivative; 0 where that is not finite.
__device__ __forceinline__ float ce_z_factor(float2 lse, const CeOpt &o) {
    const float f = 1.f + 2.f * o.zeta * fabsf(ce_lse(lse));
    return isfinite(f) ? f : 0.f;
}
// out[0] = max(out[0], v) over a warp's values; the bits of non-negative floats
// order as integers, and a maximum has no order
__device__ __forceinline__ void ce_warp_max(float v, float *out) {
#pragma unroll
    for (int k = 16; k; k >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, k));
    if ((threadIdx.x & 31) == 0 && v > 0.f)
        atomicMax(reinterpret_cast<int *>(out), __float_as_int(v));
}

// probability of score z in a row of logsumexp l
__device__ __forceinline__ float ce_prob(float z, float2 l) {
    return ex2(fmaf(z - l.x, kLog2e, -l.y));
}

// loss of a labelled row
__device__ __forceinline__ float ce_row_loss(float2 lse, float zy, float sz, int V,
                                             const CeOpt &o) {
    float l = fmaf(1.f - o.eps, lse.x - zy, lse.y * kCeLn2);
    if (o.eps > 0.f) l += o.eps * (lse.x - __fdividef(sz, (float)V));
    if (o.zeta > 0.f) l += o.zeta * ce_lse(lse) * ce_lse(lse);
    return l;
}

template <typename T> __device__ __forceinline__ float ce_to_float(T v);
template <> __device__ __forceinline__ float ce_to_float(float v) { return v; }
template <> __device__ __forceinline__ float ce_to_float(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <> __device__ __forceinline__ float ce_to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T ce_from_float(float v);
template <> __device__ __forceinline__ float ce_from_float(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 ce_from_float(float v) {
    return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half ce_from_float(float v) {
    return __float2half_rn(v);
}

// A thread's sum of the losses of its rows, thousands in a large volume, and
// what each addition has lost (exact while the sum is the larger one, as a sum
// of losses is).
struct CeSum {
    float s = 0.f, lost = 0.f;
    __device__ __forceinline__ void add(float v) {
        const float t = s + v;
        lost += v - (t - s);
        s = t;
    }
    __device__ __forceinline__ float value() const { return isfinite(s) ? s + lost : s; }
};

// Sums (loss, labelled rows) over a block of NT threads; valid in thread 0.
template <int NT>
__device__ __forceinline__ float2 ce_block_sum(float loss, float cnt, float2 *sh) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        loss += __shfl_xor_sync(0xffffffffu, loss, o);
        cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
    }
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = make_float2(loss, cnt);
    __syncthreads();
    float2 r = make_float2(0.f, 0.f);
    if (threadIdx.x == 0)
        for (int w = 0; w < NT / 32; ++w) {
            r.x += sh[w].x;
            r.y += sh[w].y;
        }
    return r;
}

// loss[0] from per-block (loss, rows) sums; count[0] = max(rows, 1), by which
// the mean and its gradient are divided (no labelled row: loss 0).
cudaError_t launch_ce_finish(const float2 *partials, int n, int reduction,
                             float *loss, float *count, cudaStream_t stream);

__device__ __forceinline__ void ce_finish(double loss, double rows, int reduction,
                                          float *out, float *count) {
    const double c = rows > 1.0 ? rows : 1.0;
    count[0] = (float)c;
    if (reduction != kCeNone)
        out[0] = (float)(reduction == kCeMean ? loss / c : loss);
}

}  // namespace gsv
