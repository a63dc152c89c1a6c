// Softmax cross entropy of scores in memory, and its gradient.
//
// Both directions are bound by HBM: V b bytes a row are read forward, read
// and written backward (b bytes a score, V classes). Two layouts:
//  * V <= kStagedV: a block stages the contiguous scores of its rows in
//    shared memory with asynchronous 16-byte copies - rows of odd lengths
//    have no alignment of their own - about 32 KB at once, which is what
//    keeps enough loads in flight. G lanes share a row and hold it in
//    registers, E scores each. The backward forms the row's maximum and sum
//    again, which costs less than the 16 bytes a row of keeping them;
//  * longer rows: one block a row, 16-byte accesses from the first aligned
//    element on, the running maximum and sum kept per thread and merged.
#include <type_traits>

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

template <int G>
__device__ __forceinline__ unsigned group_mask() {
    return G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) / G * G);
}

// A staged row in the registers of its G lanes, at most E scores each; slots
// past the row hold -inf. WORDS: rows of whole 16-byte words, of which a lane
// takes every G-th, in an order that starts elsewhere in each group of a warp
// (rows of V = 2^k would all begin in the same bank). Else a lane takes every
// G-th score: rows that are no whole words conflict twofold at most, and the
// addresses are one register and constants. Slots go in fours, skipped
// together past the row.
template <typename T, int G, int E, bool CAP, bool WORDS>
struct RowRegs {
    static constexpr int kN = WORDS ? Vec16<T>::kN : 1;  // scores a slot word
    static constexpr int kWords = E / kN;
    float z[E], t[CAP ? E : 1];
    int lane, n, rot, limit;

    __device__ __forceinline__ RowRegs(int V) {
        lane = threadIdx.x % G;
        n = (V / kN + G - 1) / G;  // words a lane
        rot = WORDS && G < 32 ? ((threadIdx.x & 31) / G) % n : 0;
        limit = V / kN - lane;     // word k of the lane exists if k G < limit
    }
    // word of slot word k, in units of words; false past the row
    __device__ __forceinline__ bool at(int k, int &w) const {
        if (!WORDS) {
            w = k * G + lane;
            return k * G < limit;
        }
        int s = k + rot;
        if (s >= n) s -= n;
        w = s * G + lane;
        return k < n && s * G < limit;
    }
    __device__ __forceinline__ void load(const T *p, float cap) {
        constexpr int kStep = WORDS ? 1 : 4;
#pragma unroll
        for (int k0 = 0; k0 < kWords; k0 += kStep) {
            if (k0 >= n) {
#pragma unroll
                for (int k = k0 * kN; k < (k0 + kStep) * kN; ++k) z[k] = ce_neg_inf();
                continue;
            }
#pragma unroll
            for (int k = k0; k < k0 + kStep; ++k) {
                int w;
                const bool ok = at(k, w);
                float s[kN];
#pragma unroll
                for (int i = 0; i < kN; ++i) s[i] = ce_neg_inf();
                if (ok) {
                    if constexpr (WORDS) {
                        const Vec16<T> v = reinterpret_cast<const Vec16<T> *>(p)[w];
#pragma unroll
                        for (int i = 0; i < kN; ++i) s[i] = ce_to_float(v.v[i]);
                    } else {
                        s[0] = ce_to_float(p[w]);
                    }
                }
#pragma unroll
                for (int i = 0; i < kN; ++i) {
                    const int e = k * kN + i;
                    if (CAP) {
                        t[CAP ? e : 0] = ce_tanh<sizeof(T) == 2>(s[i], cap);
                        s[i] = ok ? cap * t[CAP ? e : 0] : ce_neg_inf();
                    }
                    z[e] = s[i];
                }
            }
        }
    }
    // f(slot, element) -> the element's new value
    template <typename F>
    __device__ __forceinline__ void store(T *p, F f) {
        constexpr int kStep = WORDS ? 1 : 4;
#pragma unroll
        for (int k0 = 0; k0 < kWords; k0 += kStep) {
            if (k0 >= n) break;
#pragma unroll
            for (int k = k0; k < k0 + kStep; ++k) {
                int w;
                const bool ok = at(k, w);
                if constexpr (WORDS) {
                    Vec16<T> v;
#pragma unroll
                    for (int i = 0; i < kN; ++i)
                        v.v[i] = ce_from_float<T>(f(k * kN + i, w * kN + i));
                    if (ok) reinterpret_cast<Vec16<T> *>(p)[w] = v;
                } else if (ok) {
                    p[w] = ce_from_float<T>(f(k, w));
                }
            }
        }
    }
    // maximum and sum over the group
    __device__ __forceinline__ CeAcc reduce() const {
        const unsigned mask = group_mask<G>();
        CeAcc a;
        a.init();
#pragma unroll
        for (int k = 0; k < E; ++k) a.m = fmaxf(a.m, z[k]);
#pragma unroll
        for (int k = G / 2; k; k >>= 1) a.m = fmaxf(a.m, __shfl_xor_sync(mask, a.m, k));
        const float b = CeAcc::base(a.m);
#pragma unroll
        for (int k0 = 0; k0 < E; k0 += 4) {
            if (k0 >= n * kN) break;
#pragma unroll
            for (int k = k0; k < k0 + 4; ++k) a.s += ex2((z[k] - b) * kLog2e);
        }
#pragma unroll
        for (int k = G / 2; k; k >>= 1) a.s += __shfl_xor_sync(mask, a.s, k);
        return a;
    }
    __device__ __forceinline__ float plain_sum() const {
        const unsigned mask = group_mask<G>();
        float sz = 0.f;
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
            int w;
            if (k >= n) break;
            if (at(k, w)) {
#pragma unroll
                for (int i = 0; i < kN; ++i) sz += z[k * kN + i];
            }
        }
#pragma unroll
        for (int k = G / 2; k; k >>= 1) sz += __shfl_xor_sync(mask, sz, k);
        return sz;
    }
};

// kPass rows at once (one a group of G lanes), `passes` times
template <typename T, int G, int E, bool CAP, bool WORDS>
__global__ void __launch_bounds__(kNT)
staged_fwd_kernel(long long rows, int V, int passes, const T *__restrict__ scores,
                  const long long *__restrict__ labels, CeOpt o, bool vec,
                  float *__restrict__ loss, float *__restrict__ count,
                  float2 *__restrict__ partials) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float2 sh[kNT / 32];
    T *tile = reinterpret_cast<T *>(smem_raw);
    constexpr int kPass = kNT / G;
    const long long row0 = (long long)blockIdx.x * kPass * passes;
    const int nr = (int)min((long long)kPass * passes, rows - row0);
    const int r0 = threadIdx.x / G;
    long long y_next = r0 < nr ? labels[row0 + r0] : o.ignore;
    stage(tile, scores + row0 * V, nr * V, vec);
    __syncthreads();
    RowRegs<T, G, E, CAP, WORDS> row(V);
    float lsum = 0.f, cnt = 0.f;
    for (int r = r0; r < nr; r += kPass) {  // whole groups take the same path
        const T *p = tile + r * V;
        const int y = ce_label(y_next, o.ignore, V);
        if (r + kPass < nr) y_next = labels[row0 + r + kPass];
        row.load(p, o.cap);
        const CeAcc a = row.reduce();
        const float sz = o.eps > 0.f ? row.plain_sum() : 0.f;
        if (row.lane == 0) {
            float l = 0.f;
            if (y >= 0) {
                const float s = ce_to_float(p[y]);
                l = ce_row_loss(make_float2(CeAcc::base(a.m), ce_log2(a.s)),
                                CAP ? o.cap * ce_tanh<sizeof(T) == 2>(s, o.cap) : s, sz,
                                V, o);
            } else if (y == kCeInvalid) {
                l = ce_nan();
            }
            cnt += y == kCeIgnored ? 0.f : 1.f;
            lsum += l;
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

// f: the row's upstream gradient
__device__ __forceinline__ RowGrad row_grad(float2 lse, int V, float f, const CeOpt &o) {
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

template <typename T, int G, int E, bool CAP, bool WORDS>
__global__ void __launch_bounds__(kNT)
staged_bwd_kernel(long long rows, int V, int passes, const T *__restrict__ scores,
                  const long long *__restrict__ labels, CeOpt o, bool vec,
                  const float *__restrict__ count, const float *__restrict__ grad_loss,
                  T *__restrict__ grad) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T *tile = reinterpret_cast<T *>(smem_raw);
    constexpr int kPass = kNT / G;
    const long long row0 = (long long)blockIdx.x * kPass * passes;
    const int nr = (int)min((long long)kPass * passes, rows - row0);
    const int r0 = threadIdx.x / G;
    long long y_next = r0 < nr ? labels[row0 + r0] : o.ignore;
    const float common = o.reduction == kCeNone ? 0.f
                         : o.reduction == kCeMean ? grad_loss[0] / count[0]
                                                  : grad_loss[0];
    stage(tile, scores + row0 * V, nr * V, vec);
    __syncthreads();
    RowRegs<T, G, E, CAP, WORDS> row(V);
    for (int r = r0; r < nr; r += kPass) {
        T *p = tile + r * V;
        const int y = ce_label(y_next, o.ignore, V);
        if (r + kPass < nr) y_next = labels[row0 + r + kPass];
        row.load(p, o.cap);
        const CeAcc a = row.reduce();
        // probabilities are exp(z - max) over their sum: no logarithm, unless
        // the z-loss asks for the logsumexp itself
        const float base = CeAcc::base(a.m);
        float lse = 0.f;
        if (o.zeta > 0.f) lse = ce_lse(make_float2(base, ce_log2(a.s)));
        RowGrad q = row_grad(make_float2(lse, 0.f), V,
                             o.reduction == kCeNone ? grad_loss[row0 + r] : common, o);
        q.kz = y == kCeInvalid ? ce_nan() : __fdividef(q.kz, a.s);
        row.store(p, [&](int k, int j) {
            float d = fmaf(q.kz, ex2((row.z[k] - base) * kLog2e), -q.e);
            if (j == y) d -= q.hit;
            if (CAP) d *= fmaf(-row.t[CAP ? k : 0], row.t[CAP ? k : 0], 1.f);
            return y == kCeIgnored ? 0.f : d;
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

// Eight (16 bits) or four scores of a 16-byte word, in pairs for the paired
// FP32 instructions, before the cap.
__device__ __forceinline__ void pairs_of(const Vec16<float> &q, float2 (&s)[2]) {
    s[0] = make_float2(q.v[0], q.v[1]);
    s[1] = make_float2(q.v[2], q.v[3]);
}
__device__ __forceinline__ void pairs_of(const Vec16<__nv_bfloat16> &q, float2 (&s)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        s[k] = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162 *>(q.v)[k]);
}
__device__ __forceinline__ void pairs_of(const Vec16<__half> &q, float2 (&s)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = __half22float2(reinterpret_cast<const __half2 *>(q.v)[k]);
}
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

template <typename T, bool CAP>
__global__ void __launch_bounds__(kNT)
row_fwd_kernel(int V, const T *__restrict__ scores, const long long *__restrict__ labels,
               CeOpt o, float *__restrict__ loss, float2 *__restrict__ lse_out,
               float *__restrict__ count, float2 *__restrict__ partials) {
    constexpr int kN = Vec16<T>::kN, kP = kN / 2;
    const long long row = blockIdx.x;
    const T *p = scores + row * (long long)V;
    const int y = ce_label(labels[row], o.ignore, V);
    if (y == kCeIgnored) {  // nothing of the row is read, here or backward
        if (threadIdx.x) return;
        if (o.reduction == kCeNone) loss[row] = 0.f;
        if (gridDim.x == 1)
            ce_finish(0.0, 0.0, o.reduction, loss, count);
        else
            partials[row] = make_float2(0.f, 0.f);
        return;
    }
    auto score = [&](T v) {
        const float s = ce_to_float(v);
        return CAP ? o.cap * ce_tanh<sizeof(T) == 2>(s, o.cap) : s;
    };
    const float zy = y >= 0 ? score(p[y]) : 0.f;
    const int head = head_of(p, V), nv = (V - head) / kN;
    const bool smooth = o.eps > 0.f;
    CeAcc a;
    a.init();
    auto one = [&](T v) {
        const float z = score(v);
        a.merge(z, 1.f, z);
    };
    float2 s2 = f2(0.f), sz2 = f2(0.f);
    // two words at a time, both loads in flight
    auto absorb = [&](const Vec16<T> *q, auto words) {
        constexpr int kW = decltype(words)::value;
        float2 z[kW][kP];
        float m = a.m;
#pragma unroll
        for (int w = 0; w < kW; ++w) {
            pairs_of(q[w], z[w]);
#pragma unroll
            for (int k = 0; k < kP; ++k) {
                if (CAP)
                    z[w][k] = make_float2(o.cap * ce_tanh<sizeof(T) == 2>(z[w][k].x, o.cap),
                                          o.cap * ce_tanh<sizeof(T) == 2>(z[w][k].y, o.cap));
                m = fmaxf(m, fmaxf(z[w][k].x, z[w][k].y));
                if (smooth) sz2 = __fadd2_rn(sz2, z[w][k]);
            }
        }
        const float b = CeAcc::base(m);
        s2 = __fmul2_rn(s2, f2(ex2((a.m - b) * kLog2e)));
        a.m = m;
#pragma unroll
        for (int w = 0; w < kW; ++w)
#pragma unroll
            for (int k = 0; k < kP; ++k) {
                const float2 d = __fmul2_rn(__fadd2_rn(z[w][k], f2(-b)), f2(kLog2e));
                s2 = __fadd2_rn(s2, make_float2(ex2(d.x), ex2(d.y)));
            }
    };
    const Vec16<T> *words = reinterpret_cast<const Vec16<T> *>(p + head);
    int i = threadIdx.x;
    for (; i + kNT < nv; i += 2 * kNT) {
        const Vec16<T> q[2] = {words[i], words[i + kNT]};
        absorb(q, std::integral_constant<int, 2>{});
    }
    if (i < nv) absorb(words + i, std::integral_constant<int, 1>{});
    a.s = s2.x + s2.y;
    a.sz = sz2.x + sz2.y;
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
    float2 lse = a.lse();
    float l;
    if (y >= 0)
        l = ce_row_loss(lse, zy, a.sz, V, o);
    else
        l = lse.x = ce_nan();
    lse_out[row] = lse;
    if (o.reduction == kCeNone) loss[row] = l;
    if (gridDim.x == 1)
        ce_finish(l, 1.0, o.reduction, loss, count);
    else
        partials[row] = make_float2(l, 1.f);
}

template <typename T, bool CAP>
__global__ void __launch_bounds__(kNT)
row_bwd_kernel(int V, const T *__restrict__ scores, const long long *__restrict__ labels,
               CeOpt o, const float2 *__restrict__ lse_in, const float *__restrict__ count,
               const float *__restrict__ grad_loss, T *__restrict__ grad, bool same_head) {
    constexpr int kN = Vec16<T>::kN, kP = kN / 2;
    const long long row = blockIdx.x;
    const T *p = scores + row * (long long)V;
    T *out = grad + row * (long long)V;
    const int head = same_head ? head_of(p, V) : V;
    const int nv = (V - head) / kN, rest = head + nv * kN;
    const int y = ce_label(labels[row], o.ignore, V);
    int4 *o16 = reinterpret_cast<int4 *>(out + head);
    if (y == kCeIgnored) {
        for (int i = threadIdx.x; i < nv; i += kNT) __stcs(o16 + i, make_int4(0, 0, 0, 0));
        for (int j = threadIdx.x; j < head; j += kNT) out[j] = ce_from_float<T>(0.f);
        for (int j = rest + (int)threadIdx.x; j < V; j += kNT) out[j] = ce_from_float<T>(0.f);
        return;
    }
    const float f = o.reduction == kCeNone ? grad_loss[row]
                    : o.reduction == kCeMean ? grad_loss[0] / count[0]
                                             : grad_loss[0];
    const RowGrad q = row_grad(lse_in[row], V, f, o);
    const Vec16<T> *words = reinterpret_cast<const Vec16<T> *>(p + head);
#pragma unroll 2
    for (int i = threadIdx.x; i < nv; i += kNT) {
        float2 z[kP];
        pairs_of(words[i], z);
        const int at = y - (head + i * kN);
        Vec16<T> v;
#pragma unroll
        for (int k = 0; k < kP; ++k) {
            float2 t;
            if (CAP) {
                t = make_float2(ce_tanh<sizeof(T) == 2>(z[k].x, o.cap),
                                ce_tanh<sizeof(T) == 2>(z[k].y, o.cap));
                z[k] = __fmul2_rn(t, f2(o.cap));
            }
            float2 d = __ffma2_rn(__fadd2_rn(z[k], f2(-q.lse.x)), f2(kLog2e), f2(-q.lse.y));
            d = __ffma2_rn(f2(q.kz), make_float2(ex2(d.x), ex2(d.y)), f2(-q.e));
            if (at == 2 * k) d.x -= q.hit;
            if (at == 2 * k + 1) d.y -= q.hit;
            if (CAP) d = __fmul2_rn(d, __ffma2_rn(make_float2(-t.x, -t.y), t, f2(1.f)));
            v.v[2 * k] = ce_from_float<T>(d.x);
            v.v[2 * k + 1] = ce_from_float<T>(d.y);
        }
        __stcs(o16 + i, reinterpret_cast<const int4 &>(v));
    }
    auto one = [&](int j) {
        out[j] = ce_from_float<T>(grad_of<T, CAP>(p[j], j == y, q, o.cap));
    };
    for (int j = threadIdx.x; j < head; j += kNT) one(j);
    for (int j = rest + (int)threadIdx.x; j < V; j += kNT) one(j);
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

// lanes a row: up to 32 scores each. What a row costs besides its scores (its
// label, the shuffles, its loss) is paid by every lane, so few lanes are best:
// 37 classes took 66 us with eight lanes and 40 with two (786k rows).
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

template <typename T, int G, int E, bool CAP, bool WORDS>
cudaError_t staged(bool fwd, const Args &a) {
    const int passes = passes_of(a.rows, a.V, sizeof(T));
    const long long per = (long long)(kNT / G) * passes, blocks = (a.rows + per - 1) / per;
    const size_t smem = (size_t)per * a.V * sizeof(T);  // <= 32 KB
    const bool vec = ((reinterpret_cast<uintptr_t>(a.scores) |
                       reinterpret_cast<uintptr_t>(a.grad)) & 15) == 0;
    if (fwd)
        staged_fwd_kernel<T, G, E, CAP, WORDS><<<(unsigned)blocks, kNT, smem, a.st>>>(
            a.rows, a.V, passes, static_cast<const T *>(a.scores), a.labels, a.o, vec, a.loss,
            a.count, a.partials);
    else
        staged_bwd_kernel<T, G, E, CAP, WORDS><<<(unsigned)blocks, kNT, smem, a.st>>>(
            a.rows, a.V, passes, static_cast<const T *>(a.scores), a.labels, a.o, vec, a.count,
            a.grad_loss, static_cast<T *>(a.grad));
    count_launches(1);
    cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess && fwd && blocks > 1)
        err = launch_ce_finish(a.partials, (int)blocks, a.o.reduction, a.loss, a.count, a.st);
    return err;
}

template <typename T, bool CAP, bool WORDS>
cudaError_t staged_any(bool fwd, const Args &a) {
    switch (lanes_of(a.V)) {
        case 1:
            return a.V <= 4    ? staged<T, 1, (WORDS && sizeof(T) == 2 ? 8 : 4), CAP, WORDS>(fwd, a)
                   : a.V <= 8  ? staged<T, 1, 8, CAP, WORDS>(fwd, a)
                   : a.V <= 16 ? staged<T, 1, 16, CAP, WORDS>(fwd, a)
                               : staged<T, 1, 32, CAP, WORDS>(fwd, a);
        case 2: return staged<T, 2, 32, CAP, WORDS>(fwd, a);
        case 4: return staged<T, 4, 32, CAP, WORDS>(fwd, a);
        case 8: return staged<T, 8, 32, CAP, WORDS>(fwd, a);
        case 16: return staged<T, 16, 32, CAP, WORDS>(fwd, a);
        default: return staged<T, 32, 32, CAP, WORDS>(fwd, a);
    }
}

template <typename T, bool CAP>
cudaError_t run(bool fwd, const Args &a) {
    if (a.V <= kStagedV)
        return a.V * sizeof(T) % 16 == 0 ? staged_any<T, CAP, true>(fwd, a)
                                         : staged_any<T, CAP, false>(fwd, a);
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

bool softmax_ce_keeps_lse(int V) { return V > kStagedV; }

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
