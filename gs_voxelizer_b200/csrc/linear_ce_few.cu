// Linear class loss of at most four rows, without a gradient: scoring one token,
// or the few that are decoded together.
//
// The table is read once and nothing else counts: 2 V D bytes (16 bits)
// against V D multiply-adds a row. A tile of the tensor cores would be 256
// rows deep whatever the rows, and takes as long as the read. Here a warp
// takes four classes at a time, its lanes 16 bytes of each, converts and
// multiplies in float32 and keeps a running maximum and sum per row; at five
// rows of 16 bits the multiply-adds would take longer than the read (22 of 45
// bytes a clock and SM at eight), so that more rows go to the tiles. float32,
// which the tiles would have to split into three planes first, comes here up
// to eight rows.
#include <type_traits>

#include "ce_few.cuh"

namespace gsv {
namespace {

constexpr int kNT = 256, kWarps = kNT / 32;
constexpr int kClasses = 4;                 // classes a warp takes at once
constexpr int kBlocks = 4 * kSMs;
constexpr int kMergeNT = 128;

// kW elements from p as float32
template <typename T, int kW>
__device__ __forceinline__ void fetch(const T *p, float (&v)[kW]) {
    if constexpr (kW == 1) {
        v[0] = ce_to_float(p[0]);
    } else {
        struct alignas(16) Vec { T t[kW]; };
        const Vec q = *reinterpret_cast<const Vec *>(p);
#pragma unroll
        for (int i = 0; i < kW; ++i) v[i] = ce_to_float(q.t[i]);
    }
}

// part[block][row] = (maximum, sum) of the block's classes, psum likewise
template <typename T, int R, bool CAP, bool VEC>
__global__ void __launch_bounds__(kNT, R == 8 ? 2 : 4)
few_fwd_kernel(int N, int V, int D, const T *__restrict__ features, const T *__restrict__ weight,
               const long long *__restrict__ labels, CeOpt o, float2 *__restrict__ part,
               float *__restrict__ psum, float *__restrict__ zt) {
    constexpr int kW = VEC ? 16 / sizeof(T) : 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    CeAcc a[R];
    int y[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        a[r].init();
        y[r] = r < N ? ce_label(labels[r], o.ignore, V) : kCeIgnored;
    }
    const int groups = (V + kClasses - 1) / kClasses;
    for (int q = blockIdx.x * kWarps + warp; q < groups; q += gridDim.x * kWarps) {
        const int j0 = q * kClasses;
        const T *w[kClasses];
#pragma unroll
        for (int c = 0; c < kClasses; ++c)
            w[c] = weight + (long long)min(j0 + c, V - 1) * D;
        float dot[R][kClasses] = {};
#pragma unroll 2
        for (int k = lane * kW; k < D; k += 32 * kW) {
            float wv[kClasses][kW];
#pragma unroll
            for (int c = 0; c < kClasses; ++c) fetch<T, kW>(w[c] + k, wv[c]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float xv[kW];
                fetch<T, kW>(features + (long long)min(r, N - 1) * D + k, xv);
#pragma unroll
                for (int c = 0; c < kClasses; ++c)
#pragma unroll
                    for (int i = 0; i < kW; ++i) dot[r][c] = fmaf(xv[i], wv[c][i], dot[r][c]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float z[kClasses], m = a[r].m;
#pragma unroll
            for (int c = 0; c < kClasses; ++c) {
                z[c] = dot[r][c];
#pragma unroll
                for (int s = 16; s; s >>= 1) z[c] += __shfl_xor_sync(0xffffffffu, z[c], s);
                if (CAP) z[c] = o.cap * ce_tanh<sizeof(T) == 2>(z[c], o.cap);
                if (j0 + c < V) {
                    a[r].sz += z[c];
                    if (y[r] == j0 + c && lane == 0) zt[r] = z[c];
                } else {
                    z[c] = ce_neg_inf();
                }
                m = fmaxf(m, z[c]);
            }
            const float b = CeAcc::base(m);
            float s = a[r].s * ex2((a[r].m - b) * kLog2e);
#pragma unroll
            for (int c = 0; c < kClasses; ++c) s += ex2((z[c] - b) * kLog2e);
            a[r].s = s;
            a[r].m = m;
        }
    }
    __shared__ float sh[kWarps][R][3];
    if (lane == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            sh[warp][r][0] = a[r].m;
            sh[warp][r][1] = a[r].s;
            sh[warp][r][2] = a[r].sz;
        }
    }
    __syncthreads();
    const int r = threadIdx.x;
    if (r >= N) return;
    CeAcc t;
    t.init();
    for (int k = 0; k < kWarps; ++k) t.merge(sh[k][r][0], sh[k][r][1], sh[k][r][2]);
    part[blockIdx.x * N + r] = make_float2(t.m, t.s);
    psum[blockIdx.x * N + r] = t.sz;
}

// All parts of all rows, 128 threads a row -> loss, count.
__global__ void __launch_bounds__(kMergeNT *kFewRows)
few_merge_kernel(int N, int V, int parts, const float2 *__restrict__ part,
                 const float *__restrict__ psum, const float *__restrict__ zt,
                 const long long *__restrict__ labels, CeOpt o, float *__restrict__ loss,
                 float *__restrict__ count) {
    __shared__ float sh[kFewRows][kMergeNT / 32][3];
    __shared__ float s_loss[kFewRows], s_count[kFewRows];
    const int r = threadIdx.x / kMergeNT, t = threadIdx.x % kMergeNT;
    CeAcc a;
    a.init();
    for (int i = t; i < parts; i += kMergeNT) {
        const float2 p = part[i * N + r];
        a.merge(p.x, p.y, psum[i * N + r]);
    }
#pragma unroll
    for (int k = 16; k; k >>= 1)
        a.merge(__shfl_xor_sync(0xffffffffu, a.m, k), __shfl_xor_sync(0xffffffffu, a.s, k),
                __shfl_xor_sync(0xffffffffu, a.sz, k));
    if ((t & 31) == 0) {
        sh[r][t >> 5][0] = a.m;
        sh[r][t >> 5][1] = a.s;
        sh[r][t >> 5][2] = a.sz;
    }
    __syncthreads();
    if (t == 0) {
        for (int k = 1; k < kMergeNT / 32; ++k) a.merge(sh[r][k][0], sh[r][k][1], sh[r][k][2]);
        const int y = ce_label(labels[r], o.ignore, V);
        float l = 0.f;
        if (y >= 0)
            l = ce_row_loss(a.lse(), zt[r], a.sz, V, o);
        else if (y == kCeInvalid)
            l = ce_nan();
        if (o.reduction == kCeNone) loss[r] = l;
        s_loss[r] = l;
        s_count[r] = y == kCeIgnored ? 0.f : 1.f;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double l = 0.0, c = 0.0;
        for (int k = 0; k < N; ++k) {
            l += s_loss[k];
            c += s_count[k];
        }
        ce_finish(l, c, o.reduction, loss, count);
    }
}

int few_blocks(int V) { return std::min(kBlocks, (V + kClasses * kWarps - 1) / (kClasses * kWarps)); }

size_t align16(size_t b) { return (b + 15) & ~(size_t)15; }

template <typename T, int R, bool CAP>
void launch_rows(const FewArgs &a, int blocks, float2 *part, float *psum, float *zt,
                 cudaStream_t st) {
    const T *x = static_cast<const T *>(a.features), *w = static_cast<const T *>(a.weight);
    const bool vec = a.D % (16 / sizeof(T)) == 0 &&
                     ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0;
    if (vec)
        few_fwd_kernel<T, R, CAP, true><<<blocks, kNT, 0, st>>>(a.N, a.V, a.D, x, w, a.labels,
                                                                a.opt, part, psum, zt);
    else
        few_fwd_kernel<T, R, CAP, false><<<blocks, kNT, 0, st>>>(a.N, a.V, a.D, x, w, a.labels,
                                                                 a.opt, part, psum, zt);
}

template <typename T, bool CAP>
cudaError_t few_forward(const FewArgs &a, float *loss, unsigned char *ws, cudaStream_t st) {
    const int blocks = few_blocks(a.V);
    float2 *part = reinterpret_cast<float2 *>(ws);
    float *psum = reinterpret_cast<float *>(ws + align16(sizeof(float2) * blocks * a.N));
    float *zt = psum + blocks * a.N;
    if (a.N == 1)
        launch_rows<T, 1, CAP>(a, blocks, part, psum, zt, st);
    else if (a.N == 2)
        launch_rows<T, 2, CAP>(a, blocks, part, psum, zt, st);
    else if (a.N <= 4 || sizeof(T) == 2)
        launch_rows<T, 4, CAP>(a, blocks, part, psum, zt, st);
    else
        launch_rows<T, 8, CAP>(a, blocks, part, psum, zt, st);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    few_merge_kernel<<<1, kMergeNT * a.N, 0, st>>>(a.N, a.V, blocks, part, psum, zt, a.labels,
                                                   a.opt, loss, a.count);
    count_launches(2);
    return cudaGetLastError();
}

}  // namespace

size_t few_workspace_bytes(int N, int V) {
    return align16(sizeof(float2) * few_blocks(V) * N) + sizeof(float) * (few_blocks(V) + 1) * N;
}

cudaError_t launch_few_forward(const FewArgs &a, int type, float *loss, void *ws,
                               cudaStream_t st) {
    unsigned char *w = static_cast<unsigned char *>(ws);
    const bool cap = a.opt.cap > 0.f;
    switch (type) {
        case kCeF32:
            return cap ? few_forward<float, true>(a, loss, w, st)
                       : few_forward<float, false>(a, loss, w, st);
        case kCeBf16:
            return cap ? few_forward<__nv_bfloat16, true>(a, loss, w, st)
                       : few_forward<__nv_bfloat16, false>(a, loss, w, st);
        default:
            return cap ? few_forward<__half, true>(a, loss, w, st)
                       : few_forward<__half, false>(a, loss, w, st);
    }
}

}  // namespace gsv
