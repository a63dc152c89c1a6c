// Softmax cross entropy of scores in memory, and its gradient.
//
// Both directions are bound by HBM: V b bytes a row are read forward, read
// and written backward (b bytes a score, V classes). Two layouts:
//  * V <= kStagedV: a block stages the contiguous scores of its rows in
//    shared memory with 16-byte accesses - rows of odd lengths have no
//    alignment of their own - and G lanes share a row;
//  * longer rows: one block a row, 16-byte accesses from the first aligned
//    element on, the running maximum and sum kept per thread and merged.
#include "ce.cuh"

namespace gsv {
namespace {

constexpr int kStagedV = 1024;
constexpr int kNT = 256;

template <typename T>
struct alignas(16) Vec16 {
    static constexpr int kN = 16 / sizeof(T);
    T v[kN];
};

// n contiguous elements, 16 bytes an access when `vec` (both sides aligned;
// n * sizeof(T) need not be a multiple of 16)
template <typename T>
__device__ __forceinline__ void copy_block(T *dst, const T *src, int n, bool vec) {
    if (vec) {
        constexpr int kN = Vec16<T>::kN;
        const int nv = n / kN;
        for (int i = threadIdx.x; i < nv; i += kNT)
            reinterpret_cast<Vec16<T> *>(dst)[i] =
                reinterpret_cast<const Vec16<T> *>(src)[i];
        for (int i = nv * kN + threadIdx.x; i < n; i += kNT) dst[i] = src[i];
    } else {
        for (int i = threadIdx.x; i < n; i += kNT) dst[i] = src[i];
    }
}

template <typename T, int G>
__global__ void __launch_bounds__(kNT)
staged_fwd_kernel(long long rows, int V, const T *__restrict__ scores,
                  const long long *__restrict__ labels, CeOpt o, bool vec,
                  float *__restrict__ loss, float2 *__restrict__ lse_out,
                  float *__restrict__ count, float2 *__restrict__ partials) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float2 sh[kNT / 32];
    T *tile = reinterpret_cast<T *>(smem_raw);
    constexpr int R = kNT / G;
    const long long row0 = (long long)blockIdx.x * R;
    const int nr = (int)min((long long)R, rows - row0);
    copy_block(tile, scores + row0 * V, nr * V, vec);
    __syncthreads();
    const int r = threadIdx.x / G, lane = threadIdx.x % G;
    float l = 0.f, cnt = 0.f;
    if (r < nr) {  // whole groups of G lanes take the same branch
        const unsigned mask = G == 32 ? 0xffffffffu
                                      : ((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) / G * G);
        const T *p = tile + r * V;
        const int y = ce_label(labels[row0 + r], o.ignore, V);
        CeAcc a;
        a.init();
        for (int j = lane; j < V; j += G) a.m = fmaxf(a.m, ce_cap(ce_to_float(p[j]), o.cap));
#pragma unroll
        for (int k = G / 2; k; k >>= 1) a.m = fmaxf(a.m, __shfl_xor_sync(mask, a.m, k));
        const float b = CeAcc::base(a.m);
        for (int j = lane; j < V; j += G) {
            const float z = ce_cap(ce_to_float(p[j]), o.cap);
            a.s += ex2((z - b) * kLog2e);
            a.sz += z;
        }
#pragma unroll
        for (int k = G / 2; k; k >>= 1) {
            a.s += __shfl_xor_sync(mask, a.s, k);
            a.sz += __shfl_xor_sync(mask, a.sz, k);
        }
        if (lane == 0) {
            float2 lse = a.lse();
            if (y >= 0) {
                l = ce_row_loss(lse, ce_cap(ce_to_float(p[y]), o.cap), a.sz, V, o);
            } else if (y == kCeInvalid) {
                l = lse.x = ce_nan();
            }
            cnt = y == kCeIgnored ? 0.f : 1.f;
            lse_out[row0 + r] = lse;
            if (o.reduction == kCeNone) loss[row0 + r] = l;
        }
    }
    const float2 t = ce_block_sum<kNT>(l, cnt, sh);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1)
            ce_finish(t.x, t.y, o.reduction, loss, count);
        else
            partials[blockIdx.x] = t;
    }
}

// gradient of one score: k = 1 + 2 zeta lse, e = eps / V
__device__ __forceinline__ float grad_of(float s, bool hit, float2 lse, float k, float e,
                                         float g, const CeOpt &o) {
    const float z = ce_cap(s, o.cap);
    float d = k * ce_prob(z, lse) - e;
    if (hit) d -= 1.f - o.eps;
    if (o.cap > 0.f) {
        const float t = z / o.cap;
        d *= 1.f - t * t;
    }
    return d * g;
}

__device__ __forceinline__ float upstream(const float *g, long long row,
                                          const float *count, const CeOpt &o) {
    if (o.reduction == kCeNone) return g[row];
    return o.reduction == kCeMean ? g[0] / count[0] : g[0];
}

template <typename T, int G>
__global__ void __launch_bounds__(kNT)
staged_bwd_kernel(long long rows, int V, const T *__restrict__ scores,
                  const long long *__restrict__ labels, CeOpt o, bool vec,
                  const float2 *__restrict__ lse_in, const float *__restrict__ count,
                  const float *__restrict__ grad_loss, T *__restrict__ grad) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T *tile = reinterpret_cast<T *>(smem_raw);
    constexpr int R = kNT / G;
    const long long row0 = (long long)blockIdx.x * R;
    const int nr = (int)min((long long)R, rows - row0);
    copy_block(tile, scores + row0 * V, nr * V, vec);
    __syncthreads();
    const int r = threadIdx.x / G, lane = threadIdx.x % G;
    if (r < nr) {
        T *p = tile + r * V;
        const int y = ce_label(labels[row0 + r], o.ignore, V);
        const float2 lse = lse_in[row0 + r];
        const float k = 1.f + 2.f * o.zeta * ce_lse(lse);
        const float e = o.eps / (float)V;
        const float g = upstream(grad_loss, row0 + r, count, o);
        for (int j = lane; j < V; j += G)
            p[j] = ce_from_float<T>(y == kCeIgnored ? 0.f
                                                    : grad_of(ce_to_float(p[j]), j == y, lse,
                                                              k, e, g, o));
    }
    __syncthreads();
    copy_block(grad + row0 * V, tile, nr * V, vec);
}

// One block a row. `head`: elements before the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int head_of(const T *p, int V) {
    const int mis = (int)(reinterpret_cast<uintptr_t>(p) & 15);
    return mis ? min(V, (16 - mis) / (int)sizeof(T)) : 0;
}

template <typename T>
__global__ void __launch_bounds__(kNT)
row_fwd_kernel(int V, const T *__restrict__ scores, const long long *__restrict__ labels,
               CeOpt o, float *__restrict__ loss, float2 *__restrict__ lse_out,
               float *__restrict__ count, float2 *__restrict__ partials) {
    constexpr int kN = Vec16<T>::kN;
    const long long row = blockIdx.x;
    const T *p = scores + row * (long long)V;
    const int head = head_of(p, V), nv = (V - head) / kN;
    CeAcc a;
    a.init();
    auto one = [&](float s) { const float z = ce_cap(s, o.cap); a.merge(z, 1.f, z); };
    for (int i = threadIdx.x; i < nv; i += kNT) {
        const Vec16<T> q = reinterpret_cast<const Vec16<T> *>(p + head)[i];
        float z[kN], m = a.m;
#pragma unroll
        for (int k = 0; k < kN; ++k) {
            z[k] = ce_cap(ce_to_float(q.v[k]), o.cap);
            m = fmaxf(m, z[k]);
            a.sz += z[k];
        }
        const float b = CeAcc::base(m);
        a.s *= ex2((a.m - b) * kLog2e);
        a.m = m;
#pragma unroll
        for (int k = 0; k < kN; ++k) a.s += ex2((z[k] - b) * kLog2e);
    }
    if ((int)threadIdx.x < head) one(ce_to_float(p[threadIdx.x]));
    const int tail = head + nv * kN + (int)threadIdx.x;
    if (tail < V) one(ce_to_float(p[tail]));
    __shared__ float sm[kNT / 32], ss[kNT / 32], sz[kNT / 32];
#pragma unroll
    for (int k = 16; k; k >>= 1)
        a.merge(__shfl_xor_sync(0xffffffffu, a.m, k), __shfl_xor_sync(0xffffffffu, a.s, k),
                __shfl_xor_sync(0xffffffffu, a.sz, k));
    if ((threadIdx.x & 31) == 0) {
        sm[threadIdx.x >> 5] = a.m;
        ss[threadIdx.x >> 5] = a.s;
        sz[threadIdx.x >> 5] = a.sz;
    }
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < kNT / 32; ++w) a.merge(sm[w], ss[w], sz[w]);
    const int y = ce_label(labels[row], o.ignore, V);
    float2 lse = a.lse();
    float l = 0.f;
    if (y >= 0)
        l = ce_row_loss(lse, ce_cap(ce_to_float(p[y]), o.cap), a.sz, V, o);
    else if (y == kCeInvalid)
        l = lse.x = ce_nan();
    lse_out[row] = lse;
    if (o.reduction == kCeNone) loss[row] = l;
    const float c = y == kCeIgnored ? 0.f : 1.f;
    if (gridDim.x == 1)
        ce_finish(l, c, o.reduction, loss, count);
    else
        partials[row] = make_float2(l, c);
}

template <typename T>
__global__ void __launch_bounds__(kNT)
row_bwd_kernel(int V, const T *__restrict__ scores, const long long *__restrict__ labels,
               CeOpt o, const float2 *__restrict__ lse_in, const float *__restrict__ count,
               const float *__restrict__ grad_loss, T *__restrict__ grad, bool same_head) {
    constexpr int kN = Vec16<T>::kN;
    const long long row = blockIdx.x;
    const T *p = scores + row * (long long)V;
    T *q = grad + row * (long long)V;
    const int head = same_head ? head_of(p, V) : V;
    const int nv = (V - head) / kN;
    const int y = ce_label(labels[row], o.ignore, V);
    const float2 lse = lse_in[row];
    const float k = 1.f + 2.f * o.zeta * ce_lse(lse), e = o.eps / (float)V;
    const float g = upstream(grad_loss, row, count, o);
    auto one = [&](int j) {
        q[j] = ce_from_float<T>(
            y == kCeIgnored ? 0.f : grad_of(ce_to_float(p[j]), j == y, lse, k, e, g, o));
    };
    for (int i = threadIdx.x; i < nv; i += kNT) {
        Vec16<T> v = reinterpret_cast<const Vec16<T> *>(p + head)[i];
#pragma unroll
        for (int t = 0; t < kN; ++t)
            v.v[t] = ce_from_float<T>(
                y == kCeIgnored ? 0.f
                                : grad_of(ce_to_float(v.v[t]), head + i * kN + t == y, lse,
                                          k, e, g, o));
        reinterpret_cast<Vec16<T> *>(q + head)[i] = v;
    }
    for (int j = threadIdx.x; j < head; j += kNT) one(j);
    for (int j = head + nv * kN + (int)threadIdx.x; j < V; j += kNT) one(j);
}

__global__ void __launch_bounds__(1024)
finish_kernel(const float2 *__restrict__ partials, int n, int reduction,
              float *__restrict__ loss, float *__restrict__ count) {
    __shared__ double sl[32], sc[32];
    double l = 0.0, c = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) {
        const float2 p = partials[i];
        l += p.x;
        c += p.y;
    }
#pragma unroll
    for (int k = 16; k; k >>= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, k);
        c += __shfl_xor_sync(0xffffffffu, c, k);
    }
    if ((threadIdx.x & 31) == 0) {
        sl[threadIdx.x >> 5] = l;
        sc[threadIdx.x >> 5] = c;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) {
            l += sl[w];
            c += sc[w];
        }
        ce_finish(l, c, reduction, loss, count);
    }
}

// lanes a row: about eight scores each
int lanes_of(int V) {
    int g = 1;
    while (g < 32 && g * 8 < V) g *= 2;
    return g;
}

template <typename T, int G>
cudaError_t staged(bool fwd, long long rows, int V, const void *scores,
                   const long long *labels, const CeOpt &o, float *loss, float2 *lse,
                   float *count, const float *grad_loss, void *grad, float2 *partials,
                   cudaStream_t st) {
    constexpr int R = kNT / G;
    const long long blocks = (rows + R - 1) / R;
    const size_t smem = (size_t)R * V * sizeof(T);  // <= 32 KB
    const bool vec = ((reinterpret_cast<uintptr_t>(scores) |
                       reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
    if (fwd)
        staged_fwd_kernel<T, G><<<(unsigned)blocks, kNT, smem, st>>>(
            rows, V, static_cast<const T *>(scores), labels, o, vec, loss, lse, count, partials);
    else
        staged_bwd_kernel<T, G><<<(unsigned)blocks, kNT, smem, st>>>(
            rows, V, static_cast<const T *>(scores), labels, o, vec, lse, count, grad_loss,
            static_cast<T *>(grad));
    count_launches(1);
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess && fwd && blocks > 1)
        err = launch_ce_finish(partials, (int)blocks, o.reduction, loss, count, st);
    return err;
}

template <typename T>
cudaError_t run(bool fwd, long long rows, int V, const void *scores, const long long *labels,
                const CeOpt &o, float *loss, float2 *lse, float *count,
                const float *grad_loss, void *grad, float2 *partials, cudaStream_t st) {
    if (V <= kStagedV) {
        switch (lanes_of(V)) {
#define GSV_CE_G(G)                                                                     \
    case G:                                                                             \
        return staged<T, G>(fwd, rows, V, scores, labels, o, loss, lse, count, grad_loss, \
                            grad, partials, st)
            GSV_CE_G(1);
            GSV_CE_G(2);
            GSV_CE_G(4);
            GSV_CE_G(8);
            GSV_CE_G(16);
            default:
            GSV_CE_G(32);
#undef GSV_CE_G
        }
    }
    if (fwd) {
        row_fwd_kernel<T><<<(unsigned)rows, kNT, 0, st>>>(V, static_cast<const T *>(scores),
                                                          labels, o, loss, lse, count, partials);
    } else {
        const bool same = ((reinterpret_cast<uintptr_t>(scores) ^
                            reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
        row_bwd_kernel<T><<<(unsigned)rows, kNT, 0, st>>>(V, static_cast<const T *>(scores),
                                                          labels, o, lse, count, grad_loss,
                                                          static_cast<T *>(grad), same);
    }
    count_launches(1);
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess && fwd && rows > 1)
        err = launch_ce_finish(partials, (int)rows, o.reduction, loss, count, st);
    return err;
}

}  // namespace

cudaError_t launch_ce_finish(const float2 *partials, int n, int reduction, float *loss,
                             float *count, cudaStream_t stream) {
    finish_kernel<<<1, 1024, 0, stream>>>(partials, n, reduction, loss, count);
    count_launches(1);
    return cudaGetLastError();
}

size_t softmax_ce_workspace_bytes(long long rows, int V) {
    const long long r = V <= kStagedV ? kNT / lanes_of(V) : 1;
    return sizeof(float2) * (size_t)((rows + r - 1) / r);
}

cudaError_t launch_softmax_ce(bool fwd, int type, long long rows, int V, const void *scores,
                              const long long *labels, const CeOpt &o, float *loss,
                              float2 *lse, float *count, const float *grad_loss, void *grad,
                              void *ws, cudaStream_t st) {
    float2 *partials = static_cast<float2 *>(ws);
    switch (type) {
        case kCeF32:
            return run<float>(fwd, rows, V, scores, labels, o, loss, lse, count, grad_loss,
                              grad, partials, st);
        case kCeBf16:
            return run<__nv_bfloat16>(fwd, rows, V, scores, labels, o, loss, lse, count,
                                      grad_loss, grad, partials, st);
        default:
            return run<__half>(fwd, rows, V, scores, labels, o, loss, lse, count, grad_loss,
                               grad, partials, st);
    }
}

}  // namespace gsv
