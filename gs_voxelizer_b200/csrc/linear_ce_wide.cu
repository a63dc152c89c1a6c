// Linear class loss of at most 16 classes and more than 32 float32 channels,
// on the CUDA cores: a feature volume against a handful of classes.
//
// The features are all there is to move - read forward, for dX and for dW, dX
// written: 4 passes of 4 N D bytes. The tensor cores' tiles would first split
// them into three bf16 planes (10 bytes moved for 4, twice) and read those
// three times. Here a warp takes four rows, its lanes four channels each, the
// table in shared memory; the V sums of a row are joined by shuffles and the
// softmax is formed by every lane. V multiply-adds a channel against the 11
// floats a clock and SM that HBM delivers: bound by HBM up to about ten classes
// and by the multiply-adds above. dW sums rows, the other axis: it reads the
// derivatives P (V floats a row, left by dX's kernel) beside the features, each
// lane keeping V x 4 sums.
#include <atomic>

#include "ce_wide.cuh"

namespace gsv {
namespace {

constexpr int kNT = 256, kWarps = kNT / 32;
constexpr int kR = 4;        // rows a warp takes at once
constexpr int kChunk = 128;  // channels of a dW block

template <bool VEC>
__device__ __forceinline__ float4 load4(const float *p, int c, int D) {
    if (VEC) return *reinterpret_cast<const float4 *>(p + c);
    return make_float4(p[c], c + 1 < D ? p[c + 1] : 0.f, c + 2 < D ? p[c + 2] : 0.f,
                       c + 3 < D ? p[c + 3] : 0.f);
}

// the table as [V][Dp], channels past D zero
template <bool VEC>
__device__ __forceinline__ void stage(float *sw, const float *w, int V, int D, int Dp) {
    for (int i = threadIdx.x; i < V * (Dp / 4); i += kNT) {
        const int j = i / (Dp / 4), c = i % (Dp / 4) * 4;
        *reinterpret_cast<float4 *>(sw + j * Dp + c) = load4<VEC>(w + (long long)j * D, c, D);
    }
    __syncthreads();
}

// scores of rows r0 .. r0 + 3 (clamped to N - 1), in every lane
template <int VP, bool VEC, bool CAP>
__device__ __forceinline__ void scores_of(float (&z)[kR][VP], float (&t)[CAP ? kR : 1][VP],
                                          const float *sw, const float *x, long long r0,
                                          long long N, int V, int D, int Dp, float cap) {
    const int lane = threadIdx.x & 31;
    const float *row[kR];
#pragma unroll
    for (int k = 0; k < kR; ++k) row[k] = x + min(r0 + k, N - 1) * D;
#pragma unroll
    for (int k = 0; k < kR; ++k)
#pragma unroll
        for (int j = 0; j < VP; ++j) z[k][j] = 0.f;
    for (int c = 4 * lane; c < D; c += 128) {
        float4 v[kR];
#pragma unroll
        for (int k = 0; k < kR; ++k) v[k] = load4<VEC>(row[k], c, D);
#pragma unroll
        for (int j = 0; j < VP; ++j) {
            if (j >= V) break;
            const float4 w = *reinterpret_cast<const float4 *>(sw + j * Dp + c);
#pragma unroll
            for (int k = 0; k < kR; ++k)
                z[k][j] = fmaf(v[k].x, w.x, fmaf(v[k].y, w.y, fmaf(v[k].z, w.z,
                                                                  fmaf(v[k].w, w.w, z[k][j]))));
        }
    }
#pragma unroll
    for (int k = 0; k < kR; ++k)
#pragma unroll
        for (int j = 0; j < VP; ++j) {
            if (j >= V) break;
#pragma unroll
            for (int s = 16; s; s >>= 1) z[k][j] += __shfl_xor_sync(0xffffffffu, z[k][j], s);
            if (CAP) {
                t[CAP ? k : 0][j] = ce_tanh<false>(z[k][j], cap);
                z[k][j] = cap * t[CAP ? k : 0][j];
            }
        }
}

template <int VP, bool VEC, bool CAP>
__global__ void __launch_bounds__(kNT, 2)
wide_fwd_kernel(long long N, int V, int D, int Dp, const float *__restrict__ features,
                const float *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                float *__restrict__ loss, float2 *__restrict__ lse_out,
                float *__restrict__ count, float2 *__restrict__ sums) {
    extern __shared__ __align__(16) float wide_smem[];
    __shared__ float2 sh[kWarps];
    stage<VEC>(wide_smem, weight, V, D, Dp);
    const int lane = threadIdx.x & 31;
    float lsum = 0.f, cnt = 0.f;
    const long long stride = (long long)gridDim.x * kWarps * kR;
    for (long long r0 = ((long long)blockIdx.x * kWarps + threadIdx.x / 32) * kR; r0 < N;
         r0 += stride) {
        float z[kR][VP], t[CAP ? kR : 1][VP];
        scores_of<VP, VEC, CAP>(z, t, wide_smem, features, r0, N, V, D, Dp, o.cap);
#pragma unroll
        for (int k = 0; k < kR; ++k) {
            const long long r = r0 + k;
            if (r >= N) break;
            const int y = ce_label(labels[r], o.ignore, V);
            CeAcc a;
            a.init();
            float zy = 0.f;
#pragma unroll
            for (int j = 0; j < VP; ++j)
                if (j < V) a.m = fmaxf(a.m, z[k][j]);
            const float b = CeAcc::base(a.m);
#pragma unroll
            for (int j = 0; j < VP; ++j)
                if (j < V) {
                    a.s += ex2((z[k][j] - b) * kLog2e);
                    a.sz += z[k][j];
                    zy = y == j ? z[k][j] : zy;
                }
            if (lane != k) continue;
            float2 lse = a.lse();
            float l = 0.f;
            if (y >= 0)
                l = ce_row_loss(lse, zy, a.sz, V, o);
            else if (y == kCeInvalid)
                l = lse.x = ce_nan();
            lse_out[r] = lse;
            if (o.reduction == kCeNone) loss[r] = l;
            lsum += l;
            cnt += y == kCeIgnored ? 0.f : 1.f;
        }
    }
    const float2 s = ce_block_sum<kNT>(lsum, cnt, sh);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1)
            ce_finish(s.x, s.y, o.reduction, loss, count);
        else
            sums[blockIdx.x] = s;
    }
}

template <int VP, bool VEC, bool CAP>
__global__ void __launch_bounds__(kNT, 2)
wide_dx_kernel(long long N, int V, int D, int Dp, const float *__restrict__ features,
               const float *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
               const float2 *__restrict__ lse, CeUpstream u, float *__restrict__ grad,
               float *__restrict__ p_out) {
    extern __shared__ __align__(16) float wide_smem[];
    stage<VEC>(wide_smem, weight, V, D, Dp);
    const int lane = threadIdx.x & 31, ldp = (V + 3) / 4 * 4;
    const float common = common_grad(u), ev = o.eps / (float)V;
    const float *per_row = u.reduction == kCeNone ? u.g : nullptr;
    const long long stride = (long long)gridDim.x * kWarps * kR;
    for (long long r0 = ((long long)blockIdx.x * kWarps + threadIdx.x / 32) * kR; r0 < N;
         r0 += stride) {
        float z[kR][VP], t[CAP ? kR : 1][VP];
        scores_of<VP, VEC, CAP>(z, t, wide_smem, features, r0, N, V, D, Dp, o.cap);
        // scores to derivatives, the same in every lane
        unsigned unlabelled = 0;
#pragma unroll
        for (int k = 0; k < kR; ++k) {
            const long long r = r0 + k;
            if (r >= N) break;
            const int y = ce_label(labels[r], o.ignore, V);
            if (y == kCeIgnored) unlabelled |= 1u << k;
            const RowGrad q = row_grad<true>(r, y, lse[r], o, per_row, common, ev);
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                if (j >= V) break;
                float d = fmaf(q.kz, ce_prob(z[k][j], q.lse), -q.e);
                if (y == j) d -= q.hit;
                if (CAP) d *= fmaf(-t[CAP ? k : 0][j], t[CAP ? k : 0][j], 1.f);
                z[k][j] = d = y == kCeIgnored ? 0.f : d;
                if (lane == j) p_out[r * ldp + j] = d;
            }
        }
        if (!grad) continue;
        for (int c = 4 * lane; c < D; c += 128) {
            float4 out[kR];
#pragma unroll
            for (int k = 0; k < kR; ++k) out[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                if (j >= V) break;
                const float4 w = *reinterpret_cast<const float4 *>(wide_smem + j * Dp + c);
#pragma unroll
                for (int k = 0; k < kR; ++k) {
                    out[k].x = fmaf(z[k][j], w.x, out[k].x);
                    out[k].y = fmaf(z[k][j], w.y, out[k].y);
                    out[k].z = fmaf(z[k][j], w.z, out[k].z);
                    out[k].w = fmaf(z[k][j], w.w, out[k].w);
                }
            }
#pragma unroll
            for (int k = 0; k < kR; ++k) {
                if (r0 + k >= N) break;
                // a row without a label is zero whatever the table holds
                if (unlabelled >> k & 1) out[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                float *g = grad + (r0 + k) * D + c;
                if (VEC) {
                    __stcs(reinterpret_cast<float4 *>(g), out[k]);
                } else {
                    g[0] = out[k].x;
                    if (c + 1 < D) g[1] = out[k].y;
                    if (c + 2 < D) g[2] = out[k].z;
                    if (c + 3 < D) g[3] = out[k].w;
                }
            }
        }
    }
}

template <int VP, bool VEC>
__global__ void __launch_bounds__(kNT, 2)
wide_dw_kernel(long long N, int V, int D, const float *__restrict__ features,
               const long long *__restrict__ labels, long long ignore,
               const float *__restrict__ p, float *__restrict__ acc) {
    __shared__ float4 sum[VP][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ldp = (V + 3) / 4 * 4;
    const int c = blockIdx.y * kChunk + 4 * lane;
    float4 a[VP];
#pragma unroll
    for (int j = 0; j < VP; ++j) a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    // contiguous rows a warp, so that its derivatives are too
    const long long warps = (long long)gridDim.x * kWarps, w = blockIdx.x * kWarps + warp;
    const long long first = N * w / warps, last = N * (w + 1) / warps;
#pragma unroll 2
    for (long long r = first; r < last; ++r) {
        const bool keep = labels[r] != ignore;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (keep && c < D) x = load4<VEC>(features + r * D, c, D);
        const float4 *q = reinterpret_cast<const float4 *>(p + r * ldp);
#pragma unroll
        for (int j = 0; j < VP; j += 4) {
            if (j >= V) break;
            const float4 d = q[j / 4];
            const float dv[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (j + i >= V) break;
                a[j + i].x = fmaf(dv[i], x.x, a[j + i].x);
                a[j + i].y = fmaf(dv[i], x.y, a[j + i].y);
                a[j + i].z = fmaf(dv[i], x.z, a[j + i].z);
                a[j + i].w = fmaf(dv[i], x.w, a[j + i].w);
            }
        }
    }
    for (int k = 0; k < kWarps; ++k) {
        if (warp == k) {
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                float4 s = a[j];
                if (k) {
                    const float4 t = sum[j][lane];
                    s = make_float4(s.x + t.x, s.y + t.y, s.z + t.z, s.w + t.w);
                }
                sum[j][lane] = s;
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < V * kChunk; i += kNT) {
        const int j = i / kChunk, d = blockIdx.y * kChunk + i % kChunk;
        if (d < D)
            acc[((long long)blockIdx.x * V + j) * D + d] =
                reinterpret_cast<const float *>(&sum[j][0])[i % kChunk];
    }
}

template <typename F>
cudaError_t by_form(int V, bool vec, bool cap, F f) {
    auto widths = [&](auto v, auto c) {
        if (V <= 4) return f(std::integral_constant<int, 4>{}, v, c);
        if (V <= 8) return f(std::integral_constant<int, 8>{}, v, c);
        if (V <= 12) return f(std::integral_constant<int, 12>{}, v, c);
        return f(std::integral_constant<int, 16>{}, v, c);
    };
    std::true_type yes;
    std::false_type no;
    if (vec) return cap ? widths(yes, yes) : widths(yes, no);
    return cap ? widths(no, yes) : widths(no, no);
}

bool wide_rows(const NarrowArgs &a, const void *grad) {
    return a.D % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.features) |
                             reinterpret_cast<uintptr_t>(a.weight) |
                             reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
}

// the table's shared memory, allowed once a kernel and device
template <typename K>
cudaError_t allow_table(K kernel, std::atomic<unsigned long long> &ready) {
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess || (ready.load() >> (dev & 63) & 1)) return err;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(kWideTable + 16 * kWideV));
    if (err == cudaSuccess) ready.fetch_or(1ull << (dev & 63));
    return err;
}

}  // namespace

WideShape wide_shape(long long N, int V, int D) {
    WideShape s;
    s.row_blocks = (int)std::min(ceil_div(N, kWarps * kR), 2LL * kSMs);
    s.dw_chunks = (int)ceil_div(D, kChunk);
    // parts of 64 rows a warp at least
    s.dw_blocks = (int)std::max(
        1LL, std::min(ceil_div(N, kWarps * 64), std::max(1LL, 4LL * kSMs / s.dw_chunks)));
    return s;
}

cudaError_t launch_wide_fwd(const NarrowArgs &a, float *loss, float2 *sums, cudaStream_t st) {
    return by_form(a.V, wide_rows(a, nullptr), a.opt.cap > 0.f, [&](auto vp, auto vec, auto cap) {
        auto kernel =
            wide_fwd_kernel<decltype(vp)::value, decltype(vec)::value, decltype(cap)::value>;
        static std::atomic<unsigned long long> ready{0};
        const cudaError_t err = allow_table(kernel, ready);
        if (err != cudaSuccess) return err;
        const int Dp = (a.D + 3) / 4 * 4;
        kernel<<<wide_shape(a.N, a.V, a.D).row_blocks, kNT, sizeof(float) * a.V * Dp, st>>>(
            a.N, a.V, a.D, Dp, static_cast<const float *>(a.features),
            static_cast<const float *>(a.weight), a.labels, a.opt, loss, a.lse, a.count, sums);
        count_launches(1);
        return cudaGetLastError();
    });
}

cudaError_t launch_wide_dx(const NarrowArgs &a, const CeUpstream &u, float *grad, float *p,
                           cudaStream_t st) {
    return by_form(a.V, wide_rows(a, grad), a.opt.cap > 0.f, [&](auto vp, auto vec, auto cap) {
        auto kernel =
            wide_dx_kernel<decltype(vp)::value, decltype(vec)::value, decltype(cap)::value>;
        static std::atomic<unsigned long long> ready{0};
        const cudaError_t err = allow_table(kernel, ready);
        if (err != cudaSuccess) return err;
        const int Dp = (a.D + 3) / 4 * 4;
        kernel<<<wide_shape(a.N, a.V, a.D).row_blocks, kNT, sizeof(float) * a.V * Dp, st>>>(
            a.N, a.V, a.D, Dp, static_cast<const float *>(a.features),
            static_cast<const float *>(a.weight), a.labels, a.opt, a.lse, u, grad, p);
        count_launches(1);
        return cudaGetLastError();
    });
}

cudaError_t launch_wide_dw(const NarrowArgs &a, const float *p, float *acc, cudaStream_t st) {
    return by_form(a.V, wide_rows(a, nullptr), false, [&](auto vp, auto vec, auto) {
        const WideShape s = wide_shape(a.N, a.V, a.D);
        wide_dw_kernel<decltype(vp)::value, decltype(vec)::value>
            <<<dim3(s.dw_blocks, s.dw_chunks), kNT, 0, st>>>(
                a.N, a.V, a.D, static_cast<const float *>(a.features), a.labels, a.opt.ignore, p,
                acc);
        count_launches(1);
        return cudaGetLastError();
    });
}

}  // namespace gsv
