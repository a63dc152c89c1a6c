// Softmax cross entropy of scores in memory, and its gradient.
//
// Both directions are bound by HBM: V b bytes a row are read forward, read
// and written backward (b bytes a score, V classes). Two layouts:
//  * V <= kStagedV: a block stages the contiguous scores of its rows in
//    shared memory with asynchronous 16-byte copies - rows of odd lengths
//    have no alignment of their own - about 32 KB at once, which is what
//    keeps enough loads in flight, and G lanes share a row;
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

// n contiguous elements into shared memory, 16 bytes a copy when `vec`
// (src aligned; n * sizeof(T) need not be a multiple of 16)
template <typename T>
__device__ __forceinline__ void stage(T *dst, const T *src, int n, bool vec) {
    int done = 0;
    if (vec) {
        constexpr int kN = Vec16<T>::kN;
        const int nv = n / kN;
        const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
        for (int i = threadIdx.x; i < nv; i += kNT)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + 16 * i),
                         "l"(src + i * kN)
                         : "memory");
        done = nv * kN;
    }
    for (int i = done + threadIdx.x; i < n; i += kNT) dst[i] = src[i];
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename T>
__device__ __forceinline__ void unstage(T *dst, const T *src, int n, bool vec) {
    int done = 0;
    if (vec) {
        constexpr int kN = Vec16<T>::kN;
        const int nv = n / kN;
        for (int i = threadIdx.x; i < nv; i += kNT)
            __stcs(reinterpret_cast<int4 *>(dst) + i, reinterpret_cast<const int4 *>(src)[i]);
        done = nv * kN;
    }
    for (int i = done + threadIdx.x; i < n; i += kNT) dst[i] = src[i];
}

// Elements of a row that a lane of its group takes: lane, lane + G, ... from
// a start that differs between the groups of a warp, as rows of V = 2^k
// would otherwise all begin in the same bank.
template <int G, typename F>
__device__ __forceinline__ void each_of_row(int V, F f) {
    const int lane = threadIdx.x % G, n = (V + G - 1) / G;
    int k = G == 32 ? 0 : ((threadIdx.x & 31) / G) % n;
    for (int i = 0; i < n; ++i) {
        const int j = k * G + lane;
        if (G == 1 || j < V) f(j);
        if (++k == n) k = 0;
    }
}

template <int G>
__device__ __forceinline__ unsigned group_mask() {
    return G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) / G * G);
}

// kPass rows at once (one a group of G lanes), `passes` times
template <typename T, int G, bool CAP>
__global__ void __launch_bounds__(kNT)
staged_fwd_kernel(long long rows, int V, int passes, const T *__restrict__ scores,
                  const long long *__restrict__ labels, CeOpt o, bool vec,
                  float *__restrict__ loss, float2 *__restrict__ lse_out,
                  float *__restrict__ count, float2 *__restrict__ partials) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float2 sh[kNT / 32];
    T *tile = reinterpret_cast<T *>(smem_raw);
    constexpr int kPass = kNT / G;
    const long long row0 = (long long)blockIdx.x * kPass * passes;
    const int nr = (int)min((long long)kPass * passes, rows - row0);
    const int r0 = threadIdx.x / G, lane = threadIdx.x % G;
    long long y_next = r0 < nr ? labels[row0 + r0] : o.ignore;
    stage(tile, scores + row0 * V, nr * V, vec);
    __syncthreads();
    const unsigned mask = group_mask<G>();
    auto score = [&](T v) {
        const float s = ce_to_float(v);
        return CAP ? o.cap * ce_tanh<sizeof(T) == 2>(s, o.cap) : s;
    };
    float lsum = 0.f, cnt = 0.f;
    for (int r = r0; r < nr; r += kPass) {  // whole groups take the same path
        const T *p = tile + r * V;
        const int y = ce_label(y_next, o.ignore, V);
        if (r + kPass < nr) y_next = labels[row0 + r + kPass];
        CeAcc a;
        a.init();
        each_of_row<G>(V, [&](int j) { a.m = fmaxf(a.m, score(p[j])); });
#pragma unroll
        for (int k = G / 2; k; k >>= 1) a.m = fmaxf(a.m, __shfl_xor_sync(mask, a.m, k));
        const float b = CeAcc::base(a.m);
        each_of_row<G>(V, [&](int j) {
            const float z = score(p[j]);
            a.s += ex2((z - b) * kLog2e);
            a.sz += z;
        });
#pragma unroll
        for (int k = G / 2; k; k >>= 1) {
            a.s += __shfl_xor_sync(mask, a.s, k);
            a.sz += __shfl_xor_sync(mask, a.sz, k);
        }
        if (lane == 0) {
            float2 lse = a.lse();
            float l = 0.f;
            if (y >= 0)
                l = ce_row_loss(lse, score(p[y]), a.sz, V, o);
            else if (y == kCeInvalid)
                l = lse.x = ce_nan();
            cnt += y == kCeIgnored ? 0.f : 1.f;
            lsum += l;
            lse_out[row0 + r] = lse;
            if (o.reduction == kCeNone) loss[row0 + r] = l;
        }
    }
    const float2 t = ce_block_sum<kNT>(lsum, cnt, sh);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1)
            ce_finish(t.x, t.y, o.reduction, loss, count);
        else
            partials[blockIdx.x] = t;
    }
}

// A row's share of the gradient of its scores: kz prob - e (- hit at its
// class), the upstream gradient in all three.
struct RowGrad {
    float2 lse;
    float kz, e, hit;
};

__device__ __forceinline__ RowGrad row_grad(long long row, float2 lse, int V, const float *g,
                                            const float *count, const CeOpt &o) {
    const float f = o.reduction == kCeNone ? g[row]
                    : o.reduction == kCeMean ? g[0] / count[0]
                                             : g[0];
    return {lse, (1.f + 2.f * o.zeta * ce_lse(lse)) * f, o.eps / (float)V * f,
            (1.f - o.eps) * f};
}

template <typename T, bool CAP>
__device__ __forceinline__ float grad_of(T v, bool is_class, const RowGrad &q, float cap) {
    const float s = ce_to_float(v);
    const float t = CAP ? ce_tanh<sizeof(T) == 2>(s, cap) : 0.f;
    float d = fmaf(q.kz, ce_prob(CAP ? cap * t : s, q.lse), -q.e);
    if (is_class) d -= q.hit;
    if (CAP) d *= fmaf(-t, t, 1.f);
    return d;
}

template <typename T, int G, bool CAP>
__global__ void __launch_bounds__(kNT)
staged_bwd_kernel(long long rows, int V, int passes, const T *__restrict__ scores,
                  const long long *__restrict__ labels, CeOpt o, bool vec,
                  const float2 *__restrict__ lse_in, const float *__restrict__ count,
                  const float *__restrict__ grad_loss, T *__restrict__ grad) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T *tile = reinterpret_cast<T *>(smem_raw);
    constexpr int kPass = kNT / G;
    const long long row0 = (long long)blockIdx.x * kPass * passes;
    const int nr = (int)min((long long)kPass * passes, rows - row0);
    const int r0 = threadIdx.x / G;
    long long y_next = o.ignore;
    float2 lse_next = make_float2(0.f, 0.f);
    if (r0 < nr) {
        y_next = labels[row0 + r0];
        lse_next = lse_in[row0 + r0];
    }
    stage(tile, scores + row0 * V, nr * V, vec);
    __syncthreads();
    for (int r = r0; r < nr; r += kPass) {
        T *p = tile + r * V;
        const int y = ce_label(y_next, o.ignore, V);
        const RowGrad q = row_grad(row0 + r, lse_next, V, grad_loss, count, o);
        if (r + kPass < nr) {
            y_next = labels[row0 + r + kPass];
            lse_next = lse_in[row0 + r + kPass];
        }
        each_of_row<G>(V, [&](int j) {
            const float d = grad_of<T, CAP>(p[j], j == y, q, o.cap);
            p[j] = ce_from_float<T>(y == kCeIgnored ? 0.f : d);
        });
    }
    __syncthreads();
    unstage(grad + row0 * V, tile, nr * V, vec);
}

// One block a row. `head`: elements before the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int head_of(const T *p, int V) {
    const int mis = (int)(reinterpret_cast<uintptr_t>(p) & 15);
    return mis ? min(V, (16 - mis) / (int)sizeof(T)) : 0;
}

template <typename T, bool CAP>
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
    auto score = [&](T v) {
        const float s = ce_to_float(v);
        return CAP ? o.cap * ce_tanh<sizeof(T) == 2>(s, o.cap) : s;
    };
    auto one = [&](T v) {
        const float z = score(v);
        a.merge(z, 1.f, z);
    };
    for (int i = threadIdx.x; i < nv; i += kNT) {
        const Vec16<T> q = reinterpret_cast<const Vec16<T> *>(p + head)[i];
        float z[kN], m = a.m;
#pragma unroll
        for (int k = 0; k < kN; ++k) {
            z[k] = score(q.v[k]);
            m = fmaxf(m, z[k]);
            a.sz += z[k];
        }
        const float b = CeAcc::base(m);
        a.s *= ex2((a.m - b) * kLog2e);
        a.m = m;
#pragma unroll
        for (int k = 0; k < kN; ++k) a.s += ex2((z[k] - b) * kLog2e);
    }
    if ((int)threadIdx.x < head) one(p[threadIdx.x]);
    const int tail = head + nv * kN + (int)threadIdx.x;
    if (tail < V) one(p[tail]);
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
        l = ce_row_loss(lse, score(p[y]), a.sz, V, o);
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

template <typename T, bool CAP>
__global__ void __launch_bounds__(kNT)
row_bwd_kernel(int V, const T *__restrict__ scores, const long long *__restrict__ labels,
               CeOpt o, const float2 *__restrict__ lse_in, const float *__restrict__ count,
               const float *__restrict__ grad_loss, T *__restrict__ grad, bool same_head) {
    constexpr int kN = Vec16<T>::kN;
    const long long row = blockIdx.x;
    const T *p = scores + row * (long long)V;
    T *out = grad + row * (long long)V;
    const int head = same_head ? head_of(p, V) : V;
    const int nv = (V - head) / kN;
    const int y = ce_label(labels[row], o.ignore, V);
    const RowGrad q = row_grad(row, lse_in[row], V, grad_loss, count, o);
    auto one = [&](int j) {
        const float d = grad_of<T, CAP>(p[j], j == y, q, o.cap);
        out[j] = ce_from_float<T>(y == kCeIgnored ? 0.f : d);
    };
    int4 *o16 = reinterpret_cast<int4 *>(out + head);
    if (y == kCeIgnored) {  // nothing of the row is read
        for (int i = threadIdx.x; i < nv; i += kNT) __stcs(o16 + i, make_int4(0, 0, 0, 0));
    } else {
#pragma unroll 2
        for (int i = threadIdx.x; i < nv; i += kNT) {
            Vec16<T> v = reinterpret_cast<const Vec16<T> *>(p + head)[i];
            const int at = y - (head + i * kN);
#pragma unroll
            for (int t = 0; t < kN; ++t)
                v.v[t] = ce_from_float<T>(grad_of<T, CAP>(v.v[t], t == at, q, o.cap));
            __stcs(o16 + i, reinterpret_cast<const int4 &>(v));
        }
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

// lanes a row: at most 32 scores each
int lanes_of(int V) {
    int g = 1;
    while (g < 32 && g * 32 < V) g *= 2;
    return g;
}

// Times that a block's groups go over its rows: as many as 32 KB of scores
// hold (at most 8), while the blocks still fill the device twice.
int passes_of(long long rows, int V, size_t bytes) {
    const long long pass = kNT / lanes_of(V);
    const long long fit = (32 << 10) / (pass * V * (long long)bytes);
    return (int)std::max(1LL, std::min({8LL, fit, rows / (pass * 2 * kSMs)}));
}

// Every argument of both directions.
struct Args {
    long long rows;
    int V;
    const void *scores;
    const long long *labels;
    CeOpt o;
    float *loss;
    float2 *lse;
    float *count;
    const float *grad_loss;
    void *grad;
    float2 *partials;
    cudaStream_t st;
};

template <typename T, int G, bool CAP>
cudaError_t staged(bool fwd, const Args &a) {
    const int passes = passes_of(a.rows, a.V, sizeof(T));
    const long long per = (long long)(kNT / G) * passes, blocks = (a.rows + per - 1) / per;
    const size_t smem = (size_t)per * a.V * sizeof(T);  // <= 32 KB
    const bool vec = ((reinterpret_cast<uintptr_t>(a.scores) |
                       reinterpret_cast<uintptr_t>(a.grad)) & 15) == 0;
    if (fwd)
        staged_fwd_kernel<T, G, CAP><<<(unsigned)blocks, kNT, smem, a.st>>>(
            a.rows, a.V, passes, static_cast<const T *>(a.scores), a.labels, a.o, vec, a.loss,
            a.lse, a.count, a.partials);
    else
        staged_bwd_kernel<T, G, CAP><<<(unsigned)blocks, kNT, smem, a.st>>>(
            a.rows, a.V, passes, static_cast<const T *>(a.scores), a.labels, a.o, vec, a.lse,
            a.count, a.grad_loss, static_cast<T *>(a.grad));
    count_launches(1);
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess && fwd && blocks > 1)
        err = launch_ce_finish(a.partials, (int)blocks, a.o.reduction, a.loss, a.count, a.st);
    return err;
}

template <typename T, bool CAP>
cudaError_t run(bool fwd, const Args &a) {
    if (a.V <= kStagedV) {
        switch (lanes_of(a.V)) {
            case 1: return staged<T, 1, CAP>(fwd, a);
            case 2: return staged<T, 2, CAP>(fwd, a);
            case 4: return staged<T, 4, CAP>(fwd, a);
            case 8: return staged<T, 8, CAP>(fwd, a);
            case 16: return staged<T, 16, CAP>(fwd, a);
            default: return staged<T, 32, CAP>(fwd, a);
        }
    }
    const T *scores = static_cast<const T *>(a.scores);
    if (fwd) {
        row_fwd_kernel<T, CAP><<<(unsigned)a.rows, kNT, 0, a.st>>>(
            a.V, scores, a.labels, a.o, a.loss, a.lse, a.count, a.partials);
    } else {
        const bool same = ((reinterpret_cast<uintptr_t>(a.scores) ^
                            reinterpret_cast<uintptr_t>(a.grad)) & 15) == 0;
        row_bwd_kernel<T, CAP><<<(unsigned)a.rows, kNT, 0, a.st>>>(
            a.V, scores, a.labels, a.o, a.lse, a.count, a.grad_loss,
            static_cast<T *>(a.grad), same);
    }
    count_launches(1);
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess && fwd && a.rows > 1)
        err = launch_ce_finish(a.partials, (int)a.rows, a.o.reduction, a.loss, a.count, a.st);
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
    // with one pass a block, the most blocks there can be
    const long long r = V <= kStagedV ? kNT / lanes_of(V) : 1;
    return sizeof(float2) * (size_t)((rows + r - 1) / r);
}

cudaError_t launch_softmax_ce(bool fwd, int type, long long rows, int V, const void *scores,
                              const long long *labels, const CeOpt &o, float *loss,
                              float2 *lse, float *count, const float *grad_loss, void *grad,
                              void *ws, cudaStream_t st) {
    const Args a{rows, V,     scores,    labels, o,
                 loss, lse,   count,     grad_loss, grad,
                 static_cast<float2 *>(ws), st};
    const bool cap = o.cap > 0.f;
    switch (type) {
        case kCeF32: return cap ? run<float, true>(fwd, a) : run<float, false>(fwd, a);
        case kCeBf16:
            return cap ? run<__nv_bfloat16, true>(fwd, a) : run<__nv_bfloat16, false>(fwd, a);
        default: return cap ? run<__half, true>(fwd, a) : run<__half, false>(fwd, a);
    }
}

}  // namespace gsv
