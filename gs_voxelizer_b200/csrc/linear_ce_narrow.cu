// Linear class loss of few channels (D <= 8: the channels of a voxelized
// volume) on the CUDA cores, float32 throughout.
//
// A score is D multiply-adds here, and the loss's exponential (16 a clock and
// SM) costs as much as eight of them, so that the tensor cores have nothing to
// give: they pad D to 16 and, for float32, take six products. The table goes
// through shared memory in float32, each value twice, and rows go in pairs
// through the paired FP32 instructions, which leaves the exponentials (two a
// pair of scores, against 12 to 14 other instructions) as the bound. Forward
// and dX: a thread owns two rows and walks the classes with the running
// maximum and sum, or the gradient, in registers. dW: a thread owns a class
// and walks the rows, so that neither gradient needs atomics. Without a cap
// the table is held times log2 e, so that a score is an exponent of two, and
// what is linear stays out of the loops: the label's own term, the sum of all
// scores (x . sum of the table) and the smoothing's share of dX.
// Few rows or many classes: the classes (for dW the rows) are split over
// blocks and the parts are joined in a fixed order.
#include <type_traits>

#include "ce_narrow.cuh"

namespace gsv {
namespace {

constexpr int kNT = 256;
constexpr int kPairs = 1;                // pairs of rows a thread
// blocks an SM, as many as registers hold without spills
constexpr int per_sm(int dp) { return dp == 4 ? 3 : 2; }
constexpr int kBlockRows = kNT * 2 * kPairs;
constexpr int kChunk = 256;              // classes staged at once
constexpr int kTile = 256;               // rows staged at once (dW)

__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

template <int DP>
struct alignas(16) Row {
    float v[DP];
};
// every value twice, for the paired instructions
template <int DP>
struct alignas(16) Row2 {
    float2 v[DP];
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

// classes [v0, v0 + n) of the table into shared memory, times scale
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void stage_table(Row2<DP> *sw, const T *w, long long v0, int n, int D,
                                            float scale) {
    for (int j = threadIdx.x; j < n; j += kNT) {
        const Row<DP> r = load_row<T, DP, VEC>(w, v0 + j, D);
#pragma unroll
        for (int d = 0; d < DP; ++d) sw[j].v[d] = f2(r.v[d] * scale);
    }
}

template <int DP>
__device__ __forceinline__ float dot(const Row<DP> &a, const Row<DP> &b) {
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < DP; ++d) s = fmaf(a.v[d], b.v[d], s);
    return s;
}
template <int DP>
__device__ __forceinline__ float2 dot2(const Row2<DP> &a, const Row2<DP> &b) {
    float2 s = __fmul2_rn(a.v[0], b.v[0]);
#pragma unroll
    for (int d = 1; d < DP; ++d) s = __ffma2_rn(a.v[d], b.v[d], s);
    return s;
}
// What a thread reads of its rows, one tile ahead of their use: the loads of
// a tile cost as long as its classes otherwise.
template <int DP, int R>
struct Ahead {
    Row<DP> x[R];
    long long label[R];
    float2 lse[R];
};

template <typename T, int DP, bool VEC, int R>
__device__ __forceinline__ void read_ahead(Ahead<DP, R> &a, long long t0, long long N, int D,
                                           const T *features, const long long *labels,
                                           long long ignore, const float2 *lse) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const long long r = t0 + k * kNT + threadIdx.x;
        a.label[k] = ignore;
        a.lse[k] = make_float2(0.f, 0.f);
#pragma unroll
        for (int d = 0; d < DP; ++d) a.x[k].v[d] = 0.f;
        if (r < N) {
            a.x[k] = load_row<T, DP, VEC>(features, r, D);
            a.label[k] = labels[r];
            if (lse) a.lse[k] = lse[r];
        }
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
    for (int j = span.v0 + threadIdx.x; j < span.v1; j += kNT) {
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
    for (int k = 1; k < kNT / 32; ++k)
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

template <typename T, int DP, bool CAP, bool VEC>
__global__ void __launch_bounds__(kNT, per_sm(DP))
narrow_fwd_kernel(long long N, int V, int D, const T *__restrict__ features,
                  const T *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                  float *__restrict__ loss, float2 *__restrict__ lse_out,
                  float *__restrict__ count, float2 *__restrict__ sums,
                  float2 *__restrict__ part, float *__restrict__ psum,
                  float *__restrict__ zt) {
    __shared__ Row2<DP> sw[kChunk];
    __shared__ Row<DP> sh_sum[kNT / 32];
    __shared__ float2 sh[kNT / 32];
    const Span span = class_span(V);
    const bool smooth = o.eps > 0.f;
    Row<DP> wsum;
    if (smooth && !CAP) table_sum<T, DP, VEC>(wsum, sh_sum, weight, span, D);
    float lsum = 0.f, cnt = 0.f;
    bool staged = false;
    const long long stride = (long long)gridDim.x * kBlockRows;
    Ahead<DP, 2 * kPairs> next;
    read_ahead<T, DP, VEC>(next, (long long)blockIdx.x * kBlockRows, N, D, features, labels,
                           o.ignore, nullptr);
    for (long long t0 = (long long)blockIdx.x * kBlockRows; t0 < N; t0 += stride) {
        Row2<DP> x[kPairs];
        float2 m[kPairs], s[kPairs], sz[kPairs];
        int label[2 * kPairs];
#pragma unroll
        for (int k = 0; k < 2 * kPairs; ++k) {
            label[k] = ce_label(next.label[k], o.ignore, V);
#pragma unroll
            for (int d = 0; d < DP; ++d)
                (k & 1 ? x[k / 2].v[d].y : x[k / 2].v[d].x) = next.x[k].v[d];
            m[k / 2] = f2(ce_neg_inf());
            s[k / 2] = sz[k / 2] = f2(0.f);
        }
        read_ahead<T, DP, VEC>(next, t0 + stride, N, D, features, labels, o.ignore, nullptr);
        for (int v0 = span.v0; v0 < span.v1; v0 += kChunk) {
            const int n = min(kChunk, span.v1 - v0);
            if (!staged) {
                __syncthreads();
                stage_table<T, DP, VEC>(sw, weight, v0, n, D, unit<CAP>());
                __syncthreads();
                staged = span.v1 - span.v0 <= kChunk;
            }
            auto group = [&](int j0, auto size) {
                constexpr int kG = decltype(size)::value;
                float2 z[kPairs][kG];
#pragma unroll
                for (int j = 0; j < kG; ++j) {
                    const Row2<DP> w = sw[j0 + j];
#pragma unroll
                    for (int k = 0; k < kPairs; ++k) {
                        z[k][j] = dot2<DP>(x[k], w);
                        if (CAP) {
                            z[k][j].x = o.cap * ce_tanh<sizeof(T) == 2>(z[k][j].x, o.cap);
                            z[k][j].y = o.cap * ce_tanh<sizeof(T) == 2>(z[k][j].y, o.cap);
                            sz[k] = __fadd2_rn(sz[k], z[k][j]);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < kPairs; ++k) {
                    float2 top = m[k];
#pragma unroll
                    for (int j = 0; j < kG; ++j) {
                        top.x = fmaxf(top.x, z[k][j].x);
                        top.y = fmaxf(top.y, z[k][j].y);
                    }
                    // (all scores at -inf: not a distribution, NaN like theirs)
                    s[k].x *= exp_of<CAP>(m[k].x - top.x);
                    s[k].y *= exp_of<CAP>(m[k].y - top.y);
                    m[k] = top;
                    const float2 nb = make_float2(-top.x, -top.y);
                    float2 e = f2(0.f);
#pragma unroll
                    for (int j = 0; j < kG; ++j) {
                        const float2 d = __fadd2_rn(z[k][j], nb);
                        e = __fadd2_rn(e, make_float2(exp_of<CAP>(d.x), exp_of<CAP>(d.y)));
                    }
                    s[k] = __fadd2_rn(s[k], e);
                }
            };
            int j0 = 0;
            for (; j0 + 8 <= n; j0 += 8) group(j0, std::integral_constant<int, 8>{});
            if (j0 + 4 <= n) {
                group(j0, std::integral_constant<int, 4>{});
                j0 += 4;
            }
            for (; j0 < n; ++j0) group(j0, std::integral_constant<int, 1>{});
        }
#pragma unroll
        for (int k = 0; k < 2 * kPairs; ++k) {
            const long long r = t0 + k * kNT + threadIdx.x;
            if (r >= N) continue;
            const int y = label[k];
            Row<DP> q;
#pragma unroll
            for (int d = 0; d < DP; ++d) q.v[d] = k & 1 ? x[k / 2].v[d].y : x[k / 2].v[d].x;
            CeAcc a;
            a.m = k & 1 ? m[k / 2].y : m[k / 2].x;
            a.s = k & 1 ? s[k / 2].y : s[k / 2].x;
            a.sz = k & 1 ? sz[k / 2].y : sz[k / 2].x;
            if (smooth && !CAP) a.sz = dot<DP>(q, wsum);
            float zy = 0.f;
            if (y >= 0) {
                zy = dot<DP>(q, load_row<T, DP, VEC>(weight, y, D));
                if (CAP) zy = o.cap * ce_tanh<sizeof(T) == 2>(zy, o.cap);
            }
            if (gridDim.y > 1) {
                part[blockIdx.y * N + r] = make_float2(a.m, a.s);
                if (psum) psum[blockIdx.y * N + r] = a.sz;
                if (blockIdx.y == 0) zt[r] = zy;
                continue;
            }
            float l = 0.f;
            float2 lse = make_float2(CeAcc::base(a.m), __log2f(a.s));
            if (y >= 0)
                l = ce_row_loss(make_float2(CAP ? lse.x : lse.x * kCeLn2, lse.y), zy, a.sz, V, o);
            else if (y == kCeInvalid)
                l = lse.x = ce_nan();
            lse_out[r] = lse;
            if (o.reduction == kCeNone) loss[r] = l;
            lsum += l;
            cnt += y == kCeIgnored ? 0.f : 1.f;
        }
    }
    if (gridDim.y > 1) return;
    const float2 t = ce_block_sum<kNT>(lsum, cnt, sh);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1)
            ce_finish(t.x, t.y, o.reduction, loss, count);
        else
            sums[blockIdx.x] = t;
    }
}

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

template <typename T, int DP, bool CAP, bool VEC>
__global__ void __launch_bounds__(kNT, per_sm(DP))
narrow_dx_kernel(long long N, int V, int D, const T *__restrict__ features,
                 const T *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                 const float2 *__restrict__ lse, CeUpstream u, T *__restrict__ grad,
                 float *__restrict__ acc) {
    __shared__ Row2<DP> sw[kChunk];
    __shared__ Row<DP> sh_sum[kNT / 32];
    const Span span = class_span(V);
    const bool smooth = o.eps > 0.f;
    Row<DP> wsum;
    if (smooth && !CAP) table_sum<T, DP, VEC>(wsum, sh_sum, weight, span, D);
    bool staged = false;
    const float common = common_grad(u), ev = o.eps / (float)V;
    const float *per_row = u.reduction == kCeNone ? u.g : nullptr;
    const long long stride = (long long)gridDim.x * kBlockRows;
    Ahead<DP, 2 * kPairs> next;
    read_ahead<T, DP, VEC>(next, (long long)blockIdx.x * kBlockRows, N, D, features, labels,
                           o.ignore, lse);
    for (long long t0 = (long long)blockIdx.x * kBlockRows; t0 < N; t0 += stride) {
        Row2<DP> x[kPairs], dx[kPairs];
        float2 nm[kPairs], nl[kPairs], kz[kPairs], e[kPairs];
        RowGrad q[2 * kPairs];
        int y[2 * kPairs];
#pragma unroll
        for (int k = 0; k < 2 * kPairs; ++k) {
            const long long r = t0 + k * kNT + threadIdx.x;
            y[k] = ce_label(next.label[k], o.ignore, V);
            q[k] = row_grad<CAP>(r, y[k], next.lse[k], o, per_row, common, ev);
            auto put = [&](float2 &a, float b) { (k & 1 ? a.y : a.x) = b; };
#pragma unroll
            for (int d = 0; d < DP; ++d) {
                put(x[k / 2].v[d], next.x[k].v[d]);
                dx[k / 2].v[d] = f2(0.f);
            }
            put(nm[k / 2], -q[k].lse.x);
            put(nl[k / 2], -q[k].lse.y);
            put(kz[k / 2], q[k].kz);
            put(e[k / 2], -q[k].e);
        }
        read_ahead<T, DP, VEC>(next, t0 + stride, N, D, features, labels, o.ignore, lse);
        for (int v0 = span.v0; v0 < span.v1; v0 += kChunk) {
            const int n = min(kChunk, span.v1 - v0);
            if (!staged) {
                __syncthreads();
                stage_table<T, DP, VEC>(sw, weight, v0, n, D, unit<CAP>());
                __syncthreads();
                staged = span.v1 - span.v0 <= kChunk;
            }
#pragma unroll 4
            for (int j = 0; j < n; ++j) {
                const Row2<DP> w = sw[j];
#pragma unroll
                for (int k = 0; k < kPairs; ++k) {
                    float2 z = dot2<DP>(x[k], w), t;
                    if (CAP) {
                        t = make_float2(ce_tanh<sizeof(T) == 2>(z.x, o.cap),
                                        ce_tanh<sizeof(T) == 2>(z.y, o.cap));
                        z = __fmul2_rn(t, f2(o.cap));
                    }
                    z = __fadd2_rn(z, nm[k]);
                    z = CAP ? __ffma2_rn(z, f2(kLog2e), nl[k]) : __fadd2_rn(z, nl[k]);
                    float2 d = make_float2(ex2(z.x), ex2(z.y));
                    if (CAP) {  // the whole derivative goes through the slope
                        d = __ffma2_rn(kz[k], d, e[k]);
                        if (y[2 * k] == v0 + j) d.x -= q[2 * k].hit;
                        if (y[2 * k + 1] == v0 + j) d.y -= q[2 * k + 1].hit;
                        d = __fmul2_rn(d, __ffma2_rn(make_float2(-t.x, -t.y), t, f2(1.f)));
                    }
#pragma unroll
                    for (int i = 0; i < DP; ++i) dx[k].v[i] = __ffma2_rn(d, w.v[i], dx[k].v[i]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2 * kPairs; ++k) {
            const long long r = t0 + k * kNT + threadIdx.x;
            if (r >= N) continue;
            float out[DP];
#pragma unroll
            for (int d = 0; d < DP; ++d) out[d] = k & 1 ? dx[k / 2].v[d].y : dx[k / 2].v[d].x;
            if (!CAP) {
                const float f = q[k].kz * kCeLn2;  // the table is times log2 e
#pragma unroll
                for (int d = 0; d < DP; ++d) {
                    out[d] *= f;
                    if (smooth) out[d] = fmaf(-q[k].e, wsum.v[d], out[d]);
                }
                if (y[k] >= span.v0 && y[k] < span.v1) {
                    const Row<DP> w = load_row<T, DP, VEC>(weight, y[k], D);
#pragma unroll
                    for (int d = 0; d < DP; ++d) out[d] = fmaf(-q[k].hit, w.v[d], out[d]);
                }
            }
            if (y[k] == kCeIgnored) {
#pragma unroll
                for (int d = 0; d < DP; ++d) out[d] = 0.f;
            }
            if (gridDim.y > 1)
                store_row<float, DP, false>(acc + blockIdx.y * N * D, r, D, out);
            else
                store_row<T, DP, VEC>(grad, r, D, out);
        }
    }
}

// Two staged rows for dW, value by value. `more` is read where smoothing or
// z-loss make it differ from what kz gives.
template <int DP>
struct alignas(16) DwPair {
    Row2<DP> x;
    float2 nm, nl;
    float2 kz;
    int2 y;
    float2 e, hit;
};

// acc[blockIdx.x][V][D]: the block's rows' part of its classes' gradients.
// Threads: `lanes` pairs of classes (j, j + lanes) x (kNT / lanes) slices of
// the staged rows; two classes a thread halve the shared-memory reads, which
// bound it with one.
template <typename T, int DP, bool CAP, bool VEC>
__global__ void __launch_bounds__(kNT, per_sm(DP))
narrow_dw_kernel(long long N, int V, int D, int lanes, const T *__restrict__ features,
                 const T *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                 const float2 *__restrict__ lse, CeUpstream u, float *__restrict__ acc) {
    // two buffers: a tile is staged while others still read the last one
    __shared__ DwPair<DP> buffers[2][kTile / 2];
    __shared__ float red[kNT][DP + 1];
    const int slices = kNT / lanes, slice = threadIdx.x / lanes;
    const int j0 = blockIdx.y * 2 * lanes + threadIdx.x % lanes;
    const bool active = slice < slices && j0 < V;
    Row2<DP> w[2], dw[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        Row<DP> q;
#pragma unroll
        for (int d = 0; d < DP; ++d) q.v[d] = 0.f;
        if (active && j0 + c * lanes < V) q = load_row<T, DP, VEC>(weight, j0 + c * lanes, D);
#pragma unroll
        for (int d = 0; d < DP; ++d) {
            w[c].v[d] = f2(q.v[d] * unit<CAP>());
            dw[c].v[d] = f2(0.f);
        }
    }
    const bool plain = o.eps == 0.f && o.zeta == 0.f;
    const float common = common_grad(u), ev = o.eps / (float)V;
    const float *per_row = u.reduction == kCeNone ? u.g : nullptr;
    const long long stride = (long long)gridDim.x * kTile;
    int buffer = 0;
    Ahead<DP, 1> next;
    read_ahead<T, DP, VEC>(next, (long long)blockIdx.x * kTile, N, D, features, labels, o.ignore,
                           lse);
    for (long long t0 = (long long)blockIdx.x * kTile; t0 < N; t0 += stride) {
        const long long r = t0 + threadIdx.x;
        // an unlabelled row is all zeros
        const int y = ce_label(next.label[0], o.ignore, V);
        const RowGrad q = row_grad<CAP>(r, y, next.lse[0], o, per_row, common, ev);
        DwPair<DP> *rows = buffers[buffer];
        buffer ^= 1;
        {
            const int h = threadIdx.x & 1;
            DwPair<DP> &p = rows[threadIdx.x / 2];
            auto put = [&](float2 &a, float b) { (&a.x)[h] = b; };
#pragma unroll
            for (int d = 0; d < DP; ++d) put(p.x.v[d], y == kCeIgnored ? 0.f : next.x[0].v[d]);
            put(p.nm, -q.lse.x);
            put(p.nl, -q.lse.y);
            put(p.kz, q.kz);
            (&p.y.x)[h] = y;
            put(p.e, -q.e);
            put(p.hit, q.hit);
        }
        read_ahead<T, DP, VEC>(next, t0 + stride, N, D, features, labels, o.ignore, lse);
        __syncthreads();
        if (!active) continue;
        for (int i = slice; i < kTile / 2; i += slices) {
            const DwPair<DP> &p = rows[i];
            const Row2<DP> xv = p.x;
            const float2 nm = p.nm, nl = p.nl, kz = p.kz;
            const int2 yy = p.y;
            float2 hit = kz, e = f2(0.f);
            if (!plain) {
                hit = p.hit;
                e = p.e;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float2 z = dot2<DP>(xv, w[c]), t;
                if (CAP) {
                    t = make_float2(ce_tanh<sizeof(T) == 2>(z.x, o.cap),
                                    ce_tanh<sizeof(T) == 2>(z.y, o.cap));
                    z = __fmul2_rn(t, f2(o.cap));
                }
                z = __fadd2_rn(z, nm);
                z = CAP ? __ffma2_rn(z, f2(kLog2e), nl) : __fadd2_rn(z, nl);
                float2 d = make_float2(ex2(z.x), ex2(z.y));
                d = __ffma2_rn(kz, d, e);
                if (yy.x == j0 + c * lanes) d.x -= hit.x;
                if (yy.y == j0 + c * lanes) d.y -= hit.y;
                if (CAP) d = __fmul2_rn(d, __ffma2_rn(make_float2(-t.x, -t.y), t, f2(1.f)));
#pragma unroll
                for (int k = 0; k < DP; ++k) dw[c].v[k] = __ffma2_rn(d, xv.v[k], dw[c].v[k]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        float out[DP];
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DP; ++d)
            red[threadIdx.x][d] = out[d] = dw[c].v[d].x + dw[c].v[d].y;
        __syncthreads();
        const int j = j0 + c * lanes;
        if (slice == 0 && j < V) {
            for (int s = 1; s < slices; ++s)
#pragma unroll
                for (int d = 0; d < DP; ++d) out[d] += red[s * lanes + threadIdx.x][d];
            store_row<float, DP, false>(acc + (long long)blockIdx.x * V * D, j, D, out);
        }
    }
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// blocks over the rows, each taking every gridDim.x-th tile of them: a
// block stages its table once
long long row_blocks(long long N, int D) {
    return std::min(ceil_div(N, kBlockRows), (long long)per_sm(D <= 4 ? 4 : 8) * kSMs);
}
// classes split over blocks until these fill the device, 64 classes a part
// at least
int class_splits(long long N, int V, int D) {
    return (int)std::max(
        1LL, std::min({ceil_div(V, 64),
                       (long long)per_sm(D <= 4 ? 4 : 8) * kSMs / row_blocks(N, D), 1024LL}));
}

struct DwShape {
    int lanes, chunks, blocks;
};
DwShape dw_shape(long long N, int V, int D) {
    DwShape s;
    s.lanes = (int)std::min<long long>(ceil_div(V, 2), kNT);
    s.chunks = (int)ceil_div(V, 2 * s.lanes);
    s.blocks = (int)std::max(1LL, std::min(ceil_div(N, kTile), (long long)per_sm(D <= 4 ? 4 : 8) * kSMs / s.chunks));
    return s;
}

template <typename T, typename F>
cudaError_t by_form(const NarrowArgs &a, const void *grad, F f) {
    const int dp = a.D <= 4 ? 4 : 8;
    const uintptr_t mask = std::min<size_t>(16, dp * sizeof(T)) - 1;
    const bool vec = a.D == dp && ((reinterpret_cast<uintptr_t>(a.features) |
                                    reinterpret_cast<uintptr_t>(a.weight) |
                                    reinterpret_cast<uintptr_t>(grad)) & mask) == 0;
    std::integral_constant<int, 4> d4;
    std::integral_constant<int, 8> d8;
    std::true_type yes;
    std::false_type no;
    if (a.opt.cap > 0.f) {
        if (vec) return dp == 4 ? f(d4, yes, yes) : f(d8, yes, yes);
        return dp == 4 ? f(d4, yes, no) : f(d8, yes, no);
    }
    if (vec) return dp == 4 ? f(d4, no, yes) : f(d8, no, yes);
    return dp == 4 ? f(d4, no, no) : f(d8, no, no);
}

}  // namespace

int narrow_class_splits(long long N, int V, int D) { return class_splits(N, V, D); }
long long narrow_fwd_blocks(long long N, int D) { return row_blocks(N, D); }
int narrow_dw_splits(long long N, int V, int D) { return dw_shape(N, V, D).blocks; }

template <typename T>
cudaError_t launch_narrow_fwd(const NarrowArgs &a, float *loss, float2 *sums, float2 *part,
                              float *psum, float *zt, cudaStream_t st) {
    return by_form<T>(a, nullptr, [&](auto dp, auto cap, auto vec) {
        const dim3 grid((unsigned)narrow_fwd_blocks(a.N, a.D), class_splits(a.N, a.V, a.D));
        narrow_fwd_kernel<T, decltype(dp)::value, decltype(cap)::value, decltype(vec)::value><<<grid, kNT, 0, st>>>(
            a.N, a.V, a.D, static_cast<const T *>(a.features), static_cast<const T *>(a.weight),
            a.labels, a.opt, loss, a.lse, a.count, sums, part, psum, zt);
        count_launches(1);
        return cudaGetLastError();
    });
}

template <typename T>
cudaError_t launch_narrow_dx(const NarrowArgs &a, const CeUpstream &u, void *grad, float *acc,
                             cudaStream_t st) {
    return by_form<T>(a, grad, [&](auto dp, auto cap, auto vec) {
        const dim3 grid((unsigned)narrow_fwd_blocks(a.N, a.D), class_splits(a.N, a.V, a.D));
        narrow_dx_kernel<T, decltype(dp)::value, decltype(cap)::value, decltype(vec)::value><<<grid, kNT, 0, st>>>(
            a.N, a.V, a.D, static_cast<const T *>(a.features), static_cast<const T *>(a.weight),
            a.labels, a.opt, a.lse, u, static_cast<T *>(grad), acc);
        count_launches(1);
        return cudaGetLastError();
    });
}

template <typename T>
cudaError_t launch_narrow_dw(const NarrowArgs &a, const CeUpstream &u, float *acc,
                             cudaStream_t st) {
    return by_form<T>(a, nullptr, [&](auto dp, auto cap, auto vec) {
        const DwShape s = dw_shape(a.N, a.V, a.D);
        narrow_dw_kernel<T, decltype(dp)::value, decltype(cap)::value, decltype(vec)::value>
            <<<dim3(s.blocks, s.chunks), kNT, 0, st>>>(
                a.N, a.V, a.D, s.lanes, static_cast<const T *>(a.features),
                static_cast<const T *>(a.weight), a.labels, a.opt, a.lse, u, acc);
        count_launches(1);
        return cudaGetLastError();
    });
}

#define GSV_NARROW(T)                                                                         \
    template cudaError_t launch_narrow_fwd<T>(const NarrowArgs &, float *, float2 *, float2 *, \
                                              float *, float *, cudaStream_t);                \
    template cudaError_t launch_narrow_dx<T>(const NarrowArgs &, const CeUpstream &, void *,  \
                                             float *, cudaStream_t);                          \
    template cudaError_t launch_narrow_dw<T>(const NarrowArgs &, const CeUpstream &, float *, \
                                             cudaStream_t);
GSV_NARROW(float)
GSV_NARROW(__nv_bfloat16)
GSV_NARROW(__half)

}  // namespace gsv
