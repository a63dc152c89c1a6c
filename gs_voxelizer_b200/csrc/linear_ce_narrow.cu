// Linear class loss of few channels (D <= 32: the channels of a voxelized
// volume, and small feature volumes) on the CUDA cores, float32 throughout.
//
// Tiles of the tensor cores would be mostly padding here: they take 9 ps a
// score of float32 (six products of padded planes) and 3 to 25 of 16 bits, the
// more the fewer the classes, against about (2 + 0.3 D) ps for all of a
// training step here. A score is D multiply-adds and an exponential (16 a
// clock and SM, as long as eight multiply-adds). A thread takes two rows
// (forward, dX) against the classes of the table in shared memory, or one to
// four classes (dW) against the staged rows, so that each value read serves
// them all; the paired FP32 instructions run along the channels; the running
// maximum and sum, or the gradient, stay in registers, and neither gradient
// needs atomics.
//
// What bounds it: issue and latency at the occupancy that the registers leave
// (256^3 rows x 4 channels, 20 classes, float32: forward 193 us, dX 209 us,
// dW 258 us; 0.6 instructions a clock and scheduler, 12 to 20 a score, the
// exponentials alone would take 75 us each). One, two or four rows a thread,
// three to five blocks an SM and pairs of rows instead of channels came to
// 636 to 770 us for the three.
//
// Without a cap the table is held times log2 e, so that a score is an exponent
// of two, and what is linear stays out of the loops: the label's own term, the
// sum of all scores (x . sum of the table) and the smoothing's share of dX.
// Few rows or many classes: the classes (for dW the rows) are split over
// blocks and the parts are joined in a fixed order.
#include <cfloat>

#include "ce_narrow.cuh"

namespace gsv {
namespace {

constexpr int kNT = kNarrowNT;
// rows staged at once (dW), in two buffers of 48 KB at most
constexpr int dw_rows_of(int dp) { return dp <= 8 ? 256 : 128; }
constexpr int chunk_of(int dp) { return 4096 / dp; }  // classes staged at once
constexpr int kRows = 2;                              // rows a thread
// classes a thread (dW): the registers hold 2 DP each
constexpr int classes_of(int dp) { return dp == 4 ? 4 : 2; }
// Rows that a thread of dW adds up in a launch, after which its sum joins the
// block's so far: a sum of all of a block's rows, hundreds of thousands with
// many classes, was off by 1e-3 where all were alike. (Joined within the kernel,
// a loop around the tiles, 256^3 x 20 x 4 took 264 to 284 us for 258.)
constexpr int kDwChain = 1024;
// blocks an SM, as many as registers hold without spills
constexpr int per_sm(int dp) { return dp <= 8 ? 3 : dp == 16 ? 2 : 1; }
constexpr int width_of(int D) { return D <= 4 ? 4 : D <= 8 ? 8 : D <= 16 ? 16 : 32; }

template <int DP>
struct alignas(16) Pairs {
    float2 v[DP / 2];
};

template <int DP>
__device__ __forceinline__ Pairs<DP> to_pairs(const Row<DP> &r) {
    Pairs<DP> p;
#pragma unroll
    for (int d = 0; d < DP / 2; ++d) p.v[d] = make_float2(r.v[2 * d], r.v[2 * d + 1]);
    return p;
}

// A row of the table times unit<CAP>(). What was finite stays so: rows at the
// type's lowest value mask classes, and 0 times infinity would be NaN. For dW
// (FINITE) infinities become the largest numbers: rows without a label are
// staged as zeros, and of the others a probability is 0 either way (but against
// features below 2^-100, which add nothing).
template <int DP, bool CAP, bool FINITE = false>
__device__ __forceinline__ Pairs<DP> table_pairs(Row<DP> r) {
    if (!CAP || FINITE) {
#pragma unroll
        for (int d = 0; d < DP; ++d) {
            const float v = r.v[d];
            if (isnan(v) || (!FINITE && isinf(v))) continue;
            r.v[d] = fminf(fmaxf(v * unit<CAP>(), -FLT_MAX), FLT_MAX);
        }
    }
    return to_pairs<DP>(r);
}

// four chains of multiply-adds, two to a register pair
template <int DP>
__device__ __forceinline__ float dot_pairs(const Pairs<DP> &a, const Pairs<DP> &b) {
    float2 s = __fmul2_rn(a.v[0], b.v[0]), t = __fmul2_rn(a.v[1], b.v[1]);
#pragma unroll
    for (int d = 2; d < DP / 2; d += 2) {
        s = __ffma2_rn(a.v[d], b.v[d], s);
        t = __ffma2_rn(a.v[d + 1], b.v[d + 1], t);
    }
    s = __fadd2_rn(s, t);
    return s.x + s.y;
}

template <typename T, int DP, bool CAP, bool VEC>
__device__ __forceinline__ void stage_pairs(Pairs<DP> *sw, const T *w, long long v0, int n, int D) {
    for (int j = threadIdx.x; j < n; j += kNT)
        sw[j] = table_pairs<DP, CAP>(load_row<T, DP, VEC>(w, v0 + j, D));
}

// What a thread reads of its rows, one tile ahead of their use: the loads of a
// tile take as long as its classes otherwise. LSE: with the rows' statistics.
template <int DP, int R>
struct Ahead {
    Row<DP> x[R];
    long long label[R];
    float2 lse[R];
};
template <typename T, int DP, bool VEC, int R, bool LSE>
__device__ __forceinline__ void read_ahead(Ahead<DP, R> &a, long long t0, int stride, long long N,
                                           int D, const T *features, const long long *labels,
                                           long long ignore, const float2 *lse) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const long long r = t0 + k * stride + threadIdx.x;
        a.label[k] = ignore;
        a.lse[k] = make_float2(0.f, 0.f);
#pragma unroll
        for (int d = 0; d < DP; ++d) a.x[k].v[d] = 0.f;
        if (r < N) {
            a.x[k] = load_row<T, DP, VEC>(features, r, D);
            a.label[k] = labels[r];
            if (LSE) a.lse[k] = lse[r];
        }
    }
}

template <typename T, int DP, bool CAP, bool VEC>
__global__ void __launch_bounds__(kNT, per_sm(DP))
narrow_fwd_kernel(long long N, int V, int D, const T *__restrict__ features,
                  const T *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                  float *__restrict__ loss, float2 *__restrict__ lse_out,
                  float *__restrict__ count, float2 *__restrict__ sums,
                  float2 *__restrict__ part, float *__restrict__ psum,
                  float *__restrict__ zt) {
    constexpr int kChunk = chunk_of(DP), R = kRows;
    __shared__ Pairs<DP> sw[kChunk];
    __shared__ Row<DP> sh_sum[kNT / 32], s_wsum;
    __shared__ float2 sh[kNT / 32];
    const Span span = class_span(V);
    const bool smooth = o.eps > 0.f;
    if (smooth && !CAP) {
        Row<DP> wsum;
        table_sum<T, DP, VEC>(wsum, sh_sum, weight, span, D);
        if (threadIdx.x == 0) s_wsum = wsum;
        __syncthreads();
    }
    CeSum lsum;
    float cnt = 0.f;
    bool staged = false;
    const bool whole = gridDim.y == 1 && V <= kChunk;  // the table is staged, and stays
    const long long stride = (long long)gridDim.x * kNT * R;
    long long t0 = (long long)blockIdx.x * kNT * R;
    Ahead<DP, R> next;
    read_ahead<T, DP, VEC, R, false>(next, t0, kNT, N, D, features, labels, o.ignore, nullptr);
    for (; t0 < N; t0 += stride) {
        Pairs<DP> x[R];
        float m[R], s[R], sz[R];
        int y[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            x[k] = to_pairs<DP>(next.x[k]);
            y[k] = ce_label(next.label[k], o.ignore, V);
            // finite, so that classes at -inf add e^-inf = 0 wherever they come
            m[k] = -FLT_MAX;
            s[k] = sz[k] = 0.f;
        }
        // (of more channels there are no registers to read ahead into)
        if (DP == 4)
            read_ahead<T, DP, VEC, R, false>(next, t0 + stride, kNT, N, D, features, labels,
                                             o.ignore, nullptr);
        for (int v0 = span.v0; v0 < span.v1; v0 += kChunk) {
            const int n = min(kChunk, span.v1 - v0);
            if (!staged) {
                __syncthreads();
                stage_pairs<T, DP, CAP, VEC>(sw, weight, v0, n, D);
                __syncthreads();
                staged = span.v1 - span.v0 <= kChunk;
            }
            auto group = [&](int j0, auto size) {
                constexpr int kG = decltype(size)::value;
                float z[R][kG];
#pragma unroll
                for (int j = 0; j < kG; ++j) {
                    const Pairs<DP> w = sw[j0 + j];
#pragma unroll
                    for (int k = 0; k < R; ++k) {
                        z[k][j] = dot_pairs<DP>(x[k], w);
                        if (CAP) {
                            z[k][j] = o.cap * ce_tanh<sizeof(T) == 2>(z[k][j], o.cap);
                            sz[k] += z[k][j];
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    float top = m[k];
#pragma unroll
                    for (int j = 0; j < kG; ++j) top = fmaxf(top, z[k][j]);
                    s[k] *= exp_of<CAP>(m[k] - top);
                    m[k] = top;
                    float e = 0.f;
#pragma unroll
                    for (int j = 0; j < kG; ++j) e += exp_of<CAP>(z[k][j] - top);
                    s[k] += e;
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
        for (int k = 0; k < R; ++k) {
            const long long r = t0 + k * kNT + threadIdx.x;
            if (r >= N) continue;
            if (smooth && !CAP) sz[k] = dot_pairs<DP>(x[k], to_pairs<DP>(s_wsum));
            float zy = 0.f;
            if (y[k] >= 0) {
                // the same products as among all classes: where the label's
                // score is the maximum, their difference is 0
                zy = dot_pairs<DP>(x[k], whole ? sw[y[k]]
                                               : table_pairs<DP, CAP>(load_row<T, DP, VEC>(
                                                     weight, y[k], D)));
                zy = CAP ? o.cap * ce_tanh<sizeof(T) == 2>(zy, o.cap) : zy * kCeLn2;
            }
            if (gridDim.y > 1) {
                part[blockIdx.y * N + r] = make_float2(m[k], s[k]);
                if (psum) psum[blockIdx.y * N + r] = sz[k];
                if (blockIdx.y == 0) zt[r] = zy;
                continue;
            }
            float l = 0.f;
            float2 lse = make_float2(m[k], ce_log2(s[k]));
            if (y[k] >= 0)
                l = ce_row_loss(make_float2(CAP ? lse.x : lse.x * kCeLn2, lse.y), zy, sz[k], V,
                                o);
            else if (y[k] == kCeInvalid)
                l = lse.x = ce_nan();
            lse_out[r] = lse;
            if (o.reduction == kCeNone) loss[r] = l;
            lsum.add(l);
            cnt += y[k] == kCeIgnored ? 0.f : 1.f;
        }
        if (DP > 4)
            read_ahead<T, DP, VEC, R, false>(next, t0 + stride, kNT, N, D, features, labels,
                                             o.ignore, nullptr);
    }
    if (gridDim.y > 1) return;
    const float2 t = ce_block_sum<kNT>(lsum.value(), cnt, sh);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1)
            ce_finish(t.x, t.y, o.reduction, loss, count);
        else
            sums[blockIdx.x] = t;
    }
}

// 2^(score - logsumexp) of a score before the cap, and the cap's slope
template <bool CAP, bool FAST>
__device__ __forceinline__ float prob(float z, float2 lse, float cap, float &slope) {
    if (CAP) {
        const float t = ce_tanh<FAST>(z, cap);
        slope = fmaf(-t, t, 1.f);
        return ex2(fmaf(cap * t - lse.x, kLog2e, -lse.y));
    }
    return ex2((z - lse.x) - lse.y);
}

template <typename T, int DP, bool CAP, bool VEC>
__global__ void __launch_bounds__(kNT, per_sm(DP))
narrow_dx_kernel(long long N, int V, int D, const T *__restrict__ features,
                 const T *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                 const float2 *__restrict__ lse, CeUpstream u, T *__restrict__ grad,
                 float *__restrict__ acc) {
    constexpr int kChunk = chunk_of(DP), R = kRows;
    __shared__ Pairs<DP> sw[kChunk];
    __shared__ Row<DP> sh_sum[kNT / 32], s_wsum;
    const Span span = class_span(V);
    const bool smooth = o.eps > 0.f;
    if (smooth && !CAP) {
        Row<DP> wsum;
        table_sum<T, DP, VEC>(wsum, sh_sum, weight, span, D);
        if (threadIdx.x == 0) s_wsum = wsum;
        __syncthreads();
    }
    bool staged = false;
    const float common = common_grad(u), ev = o.eps / (float)V;
    const float *per_row = u.reduction == kCeNone ? u.g : nullptr;
    const long long stride = (long long)gridDim.x * kNT * R;
    long long t0 = (long long)blockIdx.x * kNT * R;
    Ahead<DP, R> next;
    read_ahead<T, DP, VEC, R, true>(next, t0, kNT, N, D, features, labels, o.ignore, lse);
    for (; t0 < N; t0 += stride) {
        Pairs<DP> x[R], dx[R];
        RowGrad q[R];
        int y[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const long long r = t0 + k * kNT + threadIdx.x;
            y[k] = ce_label(next.label[k], o.ignore, V);
            q[k] = row_grad<CAP>(r, y[k], next.lse[k], o, per_row, common, ev);
            x[k] = to_pairs<DP>(next.x[k]);
#pragma unroll
            for (int d = 0; d < DP / 2; ++d) dx[k].v[d] = f2(0.f);
        }
        if (DP == 4)
            read_ahead<T, DP, VEC, R, true>(next, t0 + stride, kNT, N, D, features, labels,
                                            o.ignore, lse);
        for (int v0 = span.v0; v0 < span.v1; v0 += kChunk) {
            const int n = min(kChunk, span.v1 - v0);
            if (!staged) {
                __syncthreads();
                stage_pairs<T, DP, CAP, VEC>(sw, weight, v0, n, D);
                __syncthreads();
                staged = span.v1 - span.v0 <= kChunk;
            }
#pragma unroll 2
            for (int j = 0; j < n; ++j) {
                const Pairs<DP> w = sw[j];
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    float slope = 1.f;
                    float d = prob<CAP, sizeof(T) == 2>(dot_pairs<DP>(x[k], w), q[k].lse, o.cap,
                                                        slope);
                    if (CAP) {  // the whole derivative goes through the slope
                        d = fmaf(q[k].kz, d, -q[k].e);
                        if (y[k] == v0 + j) d -= q[k].hit;
                        d *= slope;
                    }
#pragma unroll
                    for (int i = 0; i < DP / 2; ++i)
                        dx[k].v[i] = __ffma2_rn(f2(d), w.v[i], dx[k].v[i]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const long long r = t0 + k * kNT + threadIdx.x;
            if (r >= N) continue;
            float out[DP];
            // the table is times log2 e where there is no cap
            const float f = CAP ? 1.f : q[k].kz * kCeLn2;
#pragma unroll
            for (int d = 0; d < DP / 2; ++d) {
                out[2 * d] = dx[k].v[d].x * f;
                out[2 * d + 1] = dx[k].v[d].y * f;
            }
            if (!CAP) {
                if (smooth) {
#pragma unroll
                    for (int d = 0; d < DP; ++d) out[d] = fmaf(-q[k].e, s_wsum.v[d], out[d]);
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
        if (DP > 4)
            read_ahead<T, DP, VEC, R, true>(next, t0 + stride, kNT, N, D, features, labels,
                                            o.ignore, lse);
    }
}

// A staged row for dW; e and hit are read where smoothing or z-loss make them
// differ from what kz gives.
template <int DP>
struct alignas(16) DwRow {
    Pairs<DP> x;
    float2 lse;
    float kz;
    int y;
    float e, hit, unused[2];
};

// acc[blockIdx.x][V][D] (+)= the part of its classes' gradients of the block's
// rows among [row0, N).
// Threads: `lanes` groups of classes (j, j + lanes, ...) x (kNT / lanes)
// slices of the staged rows.
template <typename T, int DP, bool CAP, bool VEC>
__global__ void __launch_bounds__(kNT, per_sm(DP))
narrow_dw_kernel(long long row0, long long N, int V, int D, int lanes,
                 const T *__restrict__ features,
                 const T *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                 const float2 *__restrict__ lse, CeUpstream u, float *__restrict__ acc, bool add) {
    constexpr int C = classes_of(DP), kDwRows = dw_rows_of(DP);
    constexpr size_t kRowBytes = sizeof(DwRow<DP>) * kDwRows * 2;
    constexpr size_t kRedBytes = sizeof(float) * kNT * (DP + 1);
    // two buffers of rows: a tile is staged while others still read the last
    // one; and in the end the slices' sums
    __shared__ __align__(16) unsigned char raw[kRowBytes > kRedBytes ? kRowBytes : kRedBytes];
    DwRow<DP> *buffers = reinterpret_cast<DwRow<DP> *>(raw);
    float *red = reinterpret_cast<float *>(raw);
    const int slices = kNT / lanes, slice = threadIdx.x / lanes;
    const int j0 = blockIdx.y * C * lanes + threadIdx.x % lanes;
    const bool active = slice < slices && j0 < V;
    Pairs<DP> w[C], dw[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int d = 0; d < DP / 2; ++d) w[c].v[d] = dw[c].v[d] = f2(0.f);
        if (active && j0 + c * lanes < V)
            w[c] = table_pairs<DP, CAP, true>(
                load_row<T, DP, VEC>(weight, j0 + c * lanes, D));
    }
    const bool plain = o.eps == 0.f && o.zeta == 0.f;
    const float common = common_grad(u), ev = o.eps / (float)V;
    const float *per_row = u.reduction == kCeNone ? u.g : nullptr;
    const long long stride = (long long)gridDim.x * kDwRows;
    long long t0 = row0 + (long long)blockIdx.x * kDwRows;
    int buffer = 0;
    const bool stager = threadIdx.x < kDwRows;
    Ahead<DP, 1> next;
    read_ahead<T, DP, VEC, 1, true>(next, stager ? t0 : N, 0, N, D, features, labels, o.ignore,
                                    lse);
    for (; t0 < N; t0 += stride) {
        DwRow<DP> *rows = buffers + buffer * kDwRows;
        buffer ^= 1;
        if (stager) {
            // an unlabelled row is all zeros
            DwRow<DP> s{};
            s.y = ce_label(next.label[0], o.ignore, V);
            if (s.y != kCeIgnored) {
                const RowGrad q = row_grad<CAP>(t0 + threadIdx.x, s.y, next.lse[0], o, per_row,
                                                common, ev);
                s.x = to_pairs<DP>(next.x[0]);
                s.lse = q.lse;
                s.kz = q.kz;
                s.e = q.e;
                s.hit = q.hit;
            }
            rows[threadIdx.x] = s;
            read_ahead<T, DP, VEC, 1, true>(next, t0 + stride, 0, N, D, features, labels,
                                            o.ignore, lse);
        }
        __syncthreads();
        if (!active) continue;
#pragma unroll(DP == 8 || DP == 32 ? 2 : 1)
        for (int i = slice; i < kDwRows; i += slices) {
            const Pairs<DP> x = rows[i].x;
            const float2 l = rows[i].lse;
            const float kz = rows[i].kz;
            const int y = rows[i].y;
            float hit = kz, e = 0.f;
            if (!plain) {
                hit = rows[i].hit;
                e = rows[i].e;
            }
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float slope = 1.f;
                const float p =
                    prob<CAP, sizeof(T) == 2>(dot_pairs<DP>(x, w[c]), l, o.cap, slope);
                float d = fmaf(kz, p, -e);
                if (y == j0 + c * lanes) d -= hit;
                if (CAP) d *= slope;
#pragma unroll
                for (int k = 0; k < DP / 2; ++k)
                    dw[c].v[k] = __ffma2_rn(f2(d), x.v[k], dw[c].v[k]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float out[DP];
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DP / 2; ++d) {
            out[2 * d] = dw[c].v[d].x;
            out[2 * d + 1] = dw[c].v[d].y;
        }
#pragma unroll
        for (int d = 0; d < DP; ++d) red[threadIdx.x * (DP + 1) + d] = out[d];
        __syncthreads();
        const int j = j0 + c * lanes;
        if (slice == 0 && j < V) {
            for (int s = 1; s < slices; ++s)
#pragma unroll
                for (int d = 0; d < DP; ++d)
                    out[d] += red[(s * lanes + threadIdx.x) * (DP + 1) + d];
            float *sum = acc + (long long)blockIdx.x * V * D;
            if (add) {
                const Row<DP> old = load_row<float, DP, false>(sum, j, D);
#pragma unroll
                for (int d = 0; d < DP; ++d) out[d] += old.v[d];
            }
            store_row<float, DP, false>(sum, j, D, out);
        }
    }
}

template <typename F>
cudaError_t by_width(int D, F f) {
    switch (width_of(D)) {
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        case 16: return f(std::integral_constant<int, 16>{});
        default: return f(std::integral_constant<int, 32>{});
    }
}
template <typename F>
cudaError_t by_form(int D, bool cap, bool vec, F f) {
    return by_width(D, [&](auto dp) {
        std::true_type yes;
        std::false_type no;
        if (cap) return vec ? f(dp, yes, yes) : f(dp, yes, no);
        return vec ? f(dp, no, yes) : f(dp, no, no);
    });
}

}  // namespace

NarrowShape narrow_shape(long long N, int V, int D) {
    NarrowShape s;
    const int dp = width_of(D);
    const long long blocks = (long long)per_sm(dp) * kSMs;
    // blocks over the rows, each taking every gridDim.x-th tile of them: a
    // block stages its table once
    s.row_blocks = std::min(ceil_div(N, kNT * kRows), blocks);
    // classes split over blocks until these fill the device, 64 a part at
    // least
    s.class_splits =
        (int)std::max(1LL, std::min({ceil_div(V, 64), blocks / s.row_blocks, 1024LL}));
    s.dw_lanes = (int)std::min<long long>(ceil_div(V, classes_of(dp)), kNT);
    s.dw_chunks = (int)ceil_div(V, (long long)classes_of(dp) * s.dw_lanes);
    s.dw_blocks =
        (int)std::max(1LL, std::min(ceil_div(N, dw_rows_of(dp)), blocks / s.dw_chunks));
    return s;
}

template <typename T>
cudaError_t launch_narrow_fwd(const NarrowArgs &a, float *loss, float2 *sums, float2 *part,
                              float *psum, float *zt, cudaStream_t st) {
    return by_form(a.D, a.opt.cap > 0.f, a.wide_rows(sizeof(T), nullptr),
                   [&](auto dp, auto cap, auto vec) {
        const NarrowShape s = narrow_shape(a.N, a.V, a.D);
        narrow_fwd_kernel<T, decltype(dp)::value, decltype(cap)::value, decltype(vec)::value>
            <<<dim3((unsigned)s.row_blocks, s.class_splits), kNT, 0, st>>>(
                a.N, a.V, a.D, static_cast<const T *>(a.features),
                static_cast<const T *>(a.weight), a.labels, a.opt, loss, a.lse, a.count, sums,
                part, psum, zt);
        count_launches(1);
        return cudaGetLastError();
    });
}

template <typename T>
cudaError_t launch_narrow_dx(const NarrowArgs &a, const CeUpstream &u, void *grad, float *acc,
                             cudaStream_t st) {
    return by_form(a.D, a.opt.cap > 0.f, a.wide_rows(sizeof(T), grad),
                   [&](auto dp, auto cap, auto vec) {
        const NarrowShape s = narrow_shape(a.N, a.V, a.D);
        narrow_dx_kernel<T, decltype(dp)::value, decltype(cap)::value, decltype(vec)::value>
            <<<dim3((unsigned)s.row_blocks, s.class_splits), kNT, 0, st>>>(
                a.N, a.V, a.D, static_cast<const T *>(a.features),
                static_cast<const T *>(a.weight), a.labels, a.opt, a.lse, u,
                static_cast<T *>(grad), acc);
        count_launches(1);
        return cudaGetLastError();
    });
}

template <typename T>
cudaError_t launch_narrow_dw(const NarrowArgs &a, const CeUpstream &u, float *acc,
                             cudaStream_t st) {
    return by_form(a.D, a.opt.cap > 0.f, a.wide_rows(sizeof(T), nullptr),
                   [&](auto dp, auto cap, auto vec) {
        const NarrowShape s = narrow_shape(a.N, a.V, a.D);
        const long long rows = (long long)s.dw_blocks * (kNT / s.dw_lanes) * kDwChain;
        for (long long row0 = 0; row0 < a.N; row0 += rows) {
            narrow_dw_kernel<T, decltype(dp)::value, decltype(cap)::value, decltype(vec)::value>
                <<<dim3(s.dw_blocks, s.dw_chunks), kNT, 0, st>>>(
                    row0, std::min(a.N, row0 + rows), a.V, a.D, s.dw_lanes,
                    static_cast<const T *>(a.features), static_cast<const T *>(a.weight),
                    a.labels, a.opt, a.lse, u, acc, row0 > 0);
            count_launches(1);
        }
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
