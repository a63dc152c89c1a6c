// Linear class loss of few channels (D <= 8: the channels of a voxelized
// volume) on the CUDA cores, float32 throughout.
//
// A score is D multiply-adds here, and the loss's exponential (16 a clock and
// SM) costs as much as eight of them, so that the tensor cores have nothing to
// give: they pad D to 16 and, for float32, take six products. The table goes
// through shared memory in float32 and every value read there serves all rows
// of a warp. Forward and dX: a thread owns rows and walks the classes with
// the running maximum and sum (or the derivative) in registers. dW: a thread
// owns a class and walks the rows, so that neither gradient needs atomics.
// Few rows or many classes: the classes (dX: the rows, for dW) are split over
// blocks and the parts are joined in a fixed order.
#include <type_traits>

#include "ce_narrow.cuh"

namespace gsv {
namespace {

constexpr int kNT = 256;
constexpr int kRows = 2;            // rows a thread
constexpr int kChunk = 256;         // classes staged at once
constexpr int kTile = 256;          // rows staged at once (dW)

template <int DP>
struct alignas(16) Row {
    float v[DP];
};

template <typename T, int DP>
__device__ __forceinline__ Row<DP> load_row(const T *p, long long r, int D) {
    Row<DP> x;
    const T *q = p + r * D;
    if (DP == 4 && D == 4 && sizeof(T) == 4 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        const float4 f = *reinterpret_cast<const float4 *>(q);
        x.v[0] = f.x;
        x.v[1] = f.y;
        x.v[2] = f.z;
        x.v[3] = f.w;
        return x;
    }
#pragma unroll
    for (int d = 0; d < DP; ++d) x.v[d] = d < D ? ce_to_float(q[d]) : 0.f;
    return x;
}

// classes [v0, v0 + n) of the table into shared memory
template <typename T, int DP>
__device__ __forceinline__ void stage_table(Row<DP> *sw, const T *w, long long v0, int n, int D) {
    for (int j = threadIdx.x; j < n; j += kNT) sw[j] = load_row<T, DP>(w, v0 + j, D);
}

template <int DP>
__device__ __forceinline__ float dot(const Row<DP> &a, const Row<DP> &b) {
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < DP; ++d) s = fmaf(a.v[d], b.v[d], s);
    return s;
}

struct Span {
    int v0, v1;
};
__device__ __forceinline__ Span class_span(int V) {
    return {(int)((long long)V * blockIdx.y / gridDim.y),
            (int)((long long)V * (blockIdx.y + 1) / gridDim.y)};
}

template <typename T, int DP, bool CAP>
__global__ void __launch_bounds__(kNT)
narrow_fwd_kernel(long long N, int V, int D, const T *__restrict__ features,
                  const T *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                  float *__restrict__ loss, float2 *__restrict__ lse_out,
                  float *__restrict__ count, float2 *__restrict__ sums,
                  float2 *__restrict__ part, float *__restrict__ psum,
                  float *__restrict__ zt) {
    __shared__ Row<DP> sw[kChunk];
    __shared__ float2 sh[kNT / 32];
    const Span span = class_span(V);
    Row<DP> x[kRows];
    CeAcc a[kRows];
    float zy[kRows];
    int y[kRows];
    const long long r0 = (long long)blockIdx.x * kNT * kRows + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
        const long long r = r0 + k * kNT;
        a[k].init();
        zy[k] = 0.f;
        y[k] = kCeIgnored;
#pragma unroll
        for (int d = 0; d < DP; ++d) x[k].v[d] = 0.f;
        if (r < N) {
            x[k] = load_row<T, DP>(features, r, D);
            y[k] = ce_label(labels[r], o.ignore, V);
        }
    }
    for (int v0 = span.v0; v0 < span.v1; v0 += kChunk) {
        const int n = min(kChunk, span.v1 - v0);
        __syncthreads();
        stage_table<T, DP>(sw, weight, v0, n, D);
        __syncthreads();
        auto group = [&](int j0, auto full) {
            constexpr bool kFull = decltype(full)::value;
            float z[kRows][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (kFull || j0 + j < n) {
                    const Row<DP> w = sw[j0 + j];
#pragma unroll
                    for (int k = 0; k < kRows; ++k) {
                        z[k][j] = dot<DP>(x[k], w);
                        if (CAP) z[k][j] = ce_cap<sizeof(T) == 2>(z[k][j], o.cap);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < kRows; ++k) z[k][j] = ce_neg_inf();
                }
            }
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const int at = y[k] - v0 - j0;
                if (at >= 0 && at < 8) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) zy[k] = at == j ? z[k][j] : zy[k];
                }
                if (o.eps > 0.f) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (kFull || j0 + j < n) a[k].sz += z[k][j];
                }
                float m = a[k].m;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, z[k][j]);
                const float b = CeAcc::base(m);
                if (m != a[k].m) a[k].s *= ex2((a[k].m - b) * kLog2e);
                a[k].m = m;
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) s += ex2((z[k][j] - b) * kLog2e);
                a[k].s += s;
            }
        };
        int j0 = 0;
        for (; j0 + 8 <= n; j0 += 8) group(j0, std::true_type{});
        if (j0 < n) group(j0, std::false_type{});
    }
    if (gridDim.y > 1) {
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const long long r = r0 + k * kNT;
            if (r >= N) continue;
            part[blockIdx.y * N + r] = make_float2(a[k].m, a[k].s);
            if (psum) psum[blockIdx.y * N + r] = a[k].sz;
            if (y[k] >= span.v0 && y[k] < span.v1) zt[r] = zy[k];
        }
        return;
    }
    float lsum = 0.f, cnt = 0.f;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
        const long long r = r0 + k * kNT;
        if (r >= N) continue;
        float l = 0.f;
        float2 lse = a[k].lse();
        if (y[k] >= 0)
            l = ce_row_loss(lse, zy[k], a[k].sz, V, o);
        else if (y[k] == kCeInvalid)
            l = lse.x = ce_nan();
        lse_out[r] = lse;
        if (o.reduction == kCeNone) loss[r] = l;
        lsum += l;
        cnt += y[k] == kCeIgnored ? 0.f : 1.f;
    }
    const float2 t = ce_block_sum<kNT>(lsum, cnt, sh);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1)
            ce_finish(t.x, t.y, o.reduction, loss, count);
        else
            sums[blockIdx.x] = t;
    }
}

// A row's part of the derivative: kz prob - e (- hit at its class), all with
// the row's upstream gradient in them.
struct RowGrad {
    float2 lse;
    float g, kz, e, hit;
};

__device__ __forceinline__ RowGrad row_grad(long long r, int y, const float2 *lse, CeOpt o,
                                            int V, const CeUpstream &u) {
    RowGrad q{make_float2(0.f, 0.f), 0.f, 0.f, 0.f, 0.f};
    if (y == kCeIgnored) return q;
    q.lse = lse[r];
    const float g = u.reduction == kCeNone ? u.g[r]
                    : u.reduction == kCeMean ? u.g[0] / u.count[0]
                                             : u.g[0];
    q.g = g;
    q.kz = (1.f + 2.f * o.zeta * ce_lse(q.lse)) * g;
    q.e = o.eps / (float)V * g;
    q.hit = (1.f - o.eps) * g;
    return q;
}

template <bool CAP, bool FAST>
__device__ __forceinline__ float derivative(float s, bool is_class, const RowGrad &q,
                                            float cap) {
    const float t = CAP ? ce_tanh<FAST>(s, cap) : 0.f;
    float d = fmaf(q.kz, ce_prob(CAP ? cap * t : s, q.lse), -q.e);
    if (is_class) d -= q.hit;
    if (CAP) d *= fmaf(-t, t, 1.f);
    return d;
}

template <typename T, int DP, bool CAP>
__global__ void __launch_bounds__(kNT)
narrow_dx_kernel(long long N, int V, int D, const T *__restrict__ features,
                 const T *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                 const float2 *__restrict__ lse, CeUpstream u, T *__restrict__ grad,
                 float *__restrict__ acc) {
    __shared__ Row<DP> sw[kChunk];
    const Span span = class_span(V);
    Row<DP> x[kRows], dx[kRows];
    RowGrad q[kRows];
    int y[kRows];
    const long long r0 = (long long)blockIdx.x * kNT * kRows + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
        const long long r = r0 + k * kNT;
        y[k] = r < N ? ce_label(labels[r], o.ignore, V) : kCeIgnored;
        q[k] = row_grad(r, y[k], lse, o, V, u);
#pragma unroll
        for (int d = 0; d < DP; ++d) x[k].v[d] = dx[k].v[d] = 0.f;
        // an unlabelled row keeps x = 0: nothing of it is read
        if (y[k] != kCeIgnored) x[k] = load_row<T, DP>(features, r, D);
    }
    for (int v0 = span.v0; v0 < span.v1; v0 += kChunk) {
        const int n = min(kChunk, span.v1 - v0);
        __syncthreads();
        stage_table<T, DP>(sw, weight, v0, n, D);
        __syncthreads();
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const Row<DP> w = sw[j];
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const float d = derivative<CAP, sizeof(T) == 2>(dot<DP>(x[k], w), y[k] == v0 + j, q[k], o.cap);
#pragma unroll
                for (int i = 0; i < DP; ++i) dx[k].v[i] = fmaf(d, w.v[i], dx[k].v[i]);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
        const long long r = r0 + k * kNT;
        if (r >= N) continue;
        const bool zero = y[k] == kCeIgnored;
        if (gridDim.y > 1) {
            float *p = acc + (blockIdx.y * N + r) * D;
            for (int d = 0; d < DP; ++d)
                if (d < D) p[d] = zero ? 0.f : dx[k].v[d];
        } else if (DP == 4 && D == 4 && sizeof(T) == 4 &&
                   (reinterpret_cast<uintptr_t>(grad) & 15) == 0) {
            reinterpret_cast<float4 *>(grad)[r] =
                zero ? make_float4(0.f, 0.f, 0.f, 0.f)
                     : make_float4(dx[k].v[0], dx[k].v[1], dx[k].v[2], dx[k].v[3]);
        } else {
#pragma unroll
            for (int d = 0; d < DP; ++d)
                if (d < D) grad[r * D + d] = ce_from_float<T>(zero ? 0.f : dx[k].v[d]);
        }
    }
}

// What a staged row holds for dW.
template <int DP>
struct alignas(16) DwRow {
    Row<DP> x;
    float m, l2, g;
    int y;
};

// acc[blockIdx.x][V][D]: the block's rows' part of its classes' gradients.
// Threads: `lanes` classes x (kNT / lanes) slices of the staged rows.
template <typename T, int DP, bool CAP>
__global__ void __launch_bounds__(kNT)
narrow_dw_kernel(long long N, int V, int D, int lanes, const T *__restrict__ features,
                 const T *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                 const float2 *__restrict__ lse, CeUpstream u, float *__restrict__ acc) {
    __shared__ DwRow<DP> rows[kTile];
    __shared__ float red[kNT][DP + 1];
    const int slices = kNT / lanes, slice = threadIdx.x / lanes;
    const int j = blockIdx.y * lanes + threadIdx.x % lanes;
    const bool active = slice < slices && j < V;
    Row<DP> w, dw;
#pragma unroll
    for (int d = 0; d < DP; ++d) w.v[d] = dw.v[d] = 0.f;
    if (active) w = load_row<T, DP>(weight, j, D);
    const float ev = o.eps / (float)V, hv = 1.f - o.eps;
    const bool plain = o.eps == 0.f && o.zeta == 0.f;
    for (long long t0 = (long long)blockIdx.x * kTile; t0 < N; t0 += (long long)gridDim.x * kTile) {
        const long long r = t0 + threadIdx.x;
        __syncthreads();
        // rows are packed without the unlabelled ones
        const int y = r < N ? ce_label(labels[r], o.ignore, V) : kCeIgnored;
        const bool keep = y != kCeIgnored;
        __shared__ int s_warp[kNT / 32];
        const unsigned ballot = __ballot_sync(0xffffffffu, keep);
        if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = __popc(ballot);
        __syncthreads();
        int before = __popc(ballot & ((1u << (threadIdx.x & 31)) - 1u)), n = 0;
#pragma unroll
        for (int k = 0; k < kNT / 32; ++k) {
            if (k < (int)(threadIdx.x >> 5)) before += s_warp[k];
            n += s_warp[k];
        }
        if (keep) {
            const RowGrad q = row_grad(r, y, lse, o, V, u);
            DwRow<DP> s;
            s.x = load_row<T, DP>(features, r, D);
            s.m = q.lse.x;
            s.l2 = q.lse.y;
            s.g = q.g;
            s.y = y;
            rows[before] = s;
        }
        __syncthreads();
        if (!active) continue;
#pragma unroll 2
        for (int i = slice; i < n; i += slices) {
            const DwRow<DP> s = rows[i];
            const float2 l = make_float2(s.m, s.l2);
            float z = dot<DP>(s.x, w), t = 0.f;
            if (CAP) {
                t = ce_tanh<sizeof(T) == 2>(z, o.cap);
                z = o.cap * t;
            }
            float d = ce_prob(z, l);
            if (!plain) d = fmaf(1.f + 2.f * o.zeta * ce_lse(l), d, -ev);
            if (s.y == j) d -= hv;
            d *= s.g;
            if (CAP) d *= fmaf(-t, t, 1.f);
#pragma unroll
            for (int k = 0; k < DP; ++k) dw.v[k] = fmaf(d, s.x.v[k], dw.v[k]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DP; ++d) red[threadIdx.x][d] = dw.v[d];
    __syncthreads();
    if (slice == 0 && j < V) {
        for (int s = 1; s < slices; ++s)
#pragma unroll
            for (int d = 0; d < DP; ++d) dw.v[d] += red[s * lanes + threadIdx.x][d];
        float *p = acc + ((long long)blockIdx.x * V + j) * D;
        for (int d = 0; d < DP; ++d)
            if (d < D) p[d] = dw.v[d];
    }
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// classes split over blocks until the rows' blocks fill the device twice,
// 64 classes a part at least
int class_splits(long long N, int V) {
    const long long blocks = ceil_div(N, kNT * kRows);
    return (int)std::max(1LL, std::min({ceil_div(V, 64), 4LL * kSMs / blocks, 1024LL}));
}

struct DwShape {
    int lanes, chunks, blocks;
};
DwShape dw_shape(long long N, int V) {
    DwShape s;
    s.lanes = std::min(V, kNT);
    s.chunks = (int)ceil_div(V, s.lanes);
    s.blocks = (int)std::max(1LL, std::min(ceil_div(N, kTile), 6LL * kSMs / s.chunks));
    return s;
}

template <typename F>
cudaError_t by_width(int D, bool cap, F f) {
    std::integral_constant<int, 4> d4;
    std::integral_constant<int, 8> d8;
    if (D <= 4) return cap ? f(d4, std::true_type{}) : f(d4, std::false_type{});
    return cap ? f(d8, std::true_type{}) : f(d8, std::false_type{});
}

}  // namespace

int narrow_class_splits(long long N, int V) { return class_splits(N, V); }
long long narrow_fwd_blocks(long long N) { return ceil_div(N, kNT * kRows); }
int narrow_dw_splits(long long N, int V) { return dw_shape(N, V).blocks; }

template <typename T>
cudaError_t launch_narrow_fwd(const NarrowArgs &a, float *loss, float2 *sums, float2 *part,
                              float *psum, float *zt, cudaStream_t st) {
    return by_width(a.D, a.opt.cap > 0.f, [&](auto dp, auto cap) {
        const dim3 grid((unsigned)narrow_fwd_blocks(a.N), class_splits(a.N, a.V));
        narrow_fwd_kernel<T, decltype(dp)::value, decltype(cap)::value><<<grid, kNT, 0, st>>>(
            a.N, a.V, a.D, static_cast<const T *>(a.features), static_cast<const T *>(a.weight),
            a.labels, a.opt, loss, a.lse, a.count, sums, part, psum, zt);
        count_launches(1);
        return cudaGetLastError();
    });
}

template <typename T>
cudaError_t launch_narrow_dx(const NarrowArgs &a, const CeUpstream &u, void *grad, float *acc,
                             cudaStream_t st) {
    return by_width(a.D, a.opt.cap > 0.f, [&](auto dp, auto cap) {
        const dim3 grid((unsigned)narrow_fwd_blocks(a.N), class_splits(a.N, a.V));
        narrow_dx_kernel<T, decltype(dp)::value, decltype(cap)::value><<<grid, kNT, 0, st>>>(
            a.N, a.V, a.D, static_cast<const T *>(a.features), static_cast<const T *>(a.weight),
            a.labels, a.opt, a.lse, u, static_cast<T *>(grad), acc);
        count_launches(1);
        return cudaGetLastError();
    });
}

template <typename T>
cudaError_t launch_narrow_dw(const NarrowArgs &a, const CeUpstream &u, float *acc,
                             cudaStream_t st) {
    return by_width(a.D, a.opt.cap > 0.f, [&](auto dp, auto cap) {
        const DwShape s = dw_shape(a.N, a.V);
        narrow_dw_kernel<T, decltype(dp)::value, decltype(cap)::value>
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
