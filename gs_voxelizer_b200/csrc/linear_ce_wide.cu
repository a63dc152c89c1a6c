// Linear class loss of at most 16 classes and more than 32 float32 channels,
// on the CUDA cores: a feature volume against a handful of classes.
//
// The features are all there is to move - read forward and for dW, dX written:
// 3 passes of 4 N D bytes. The tensor cores' tiles would first split them into
// three bf16 planes (10 bytes moved for 4, twice) and read those three times:
// 3312 us of kernels at 603768 rows x 9 classes x 440 channels. Here the
// forward stages 32 channels of 256 rows (and of the table) at a time with
// asynchronous copies, the next while one is used; a thread owns two rows, so
// that the V sums of a row need no exchange, and every value of the table read
// from shared memory serves both. It keeps the scores (V floats a row, less
// than half of the features), and the backward need not form them again:
// derivatives P from them, then dX with a lane's four columns of the table in
// registers and whole rows written, and dW with V x 4 sums a lane. V
// multiply-adds a channel against the 11 floats a clock and SM that HBM
// delivers; it reaches 2.4 to 3 TB/s a pass, bound by the loads in flight that
// this choice of stages leaves: 74 KB of them a block in the forward, 10 to 25 %
// of the warps resident. (More and smaller stages were not tried.) 603768 x
// 9 x 440: 1237 us of kernels (scores formed again and dX written by their
// threads: 1518; a warp a row with sums by shuffles: 2437); 147949 x 6 x 1578:
// 1063 (1906).
#include <atomic>

#include "ce_wide.cuh"

namespace gsv {
namespace {

constexpr int kNT = 128;                 // forward
constexpr int kR = 2;                    // rows a thread
constexpr int kRows = kNT * kR;          // rows a tile
constexpr int kDepth = 32;               // channels staged at once
// floats of a staged row: rows 16-byte words apart by an odd number of them,
// which reads of a word a lane take without bank conflicts
constexpr int kPitch = kDepth + 4;
constexpr int kDwNT = 256, kDwWarps = kDwNT / 32;
constexpr int kDwRows = 64;              // rows a tile of dW, eight a warp
constexpr int kChunk = 128;              // channels of a dW block
// rows that a warp of dW adds up before its sums join the block's
constexpr int kDwChain = 1024;

template <int VP>
struct alignas(16) Stage {
    float x[kRows][kPitch];
    float w[VP][kDepth];
};

__device__ __forceinline__ void copy16(float *dst, const float *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src)
                 : "memory");
}
__device__ __forceinline__ void copy4(float *dst, const float *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src)
                 : "memory");
}
// four floats of which `valid` exist, zeros after them; VEC: all or none, and
// aligned to 16 bytes
template <bool VEC>
__device__ __forceinline__ void copy_word(float *dst, const float *src, int valid) {
    if (VEC && valid > 0) {
        copy16(dst, src);
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (k < valid)
            copy4(dst + k, src + k);
        else
            dst[k] = 0.f;
    }
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// channels [c0, c0 + 32) of the table, zeros past D
template <int VP, bool VEC>
__device__ __forceinline__ void stage_table(float (&dst)[VP][kDepth], const float *w, int V, int D,
                                            int c0) {
    for (int i = threadIdx.x; i < V * (kDepth / 4); i += kNT) {
        const int j = i / (kDepth / 4), c = i % (kDepth / 4) * 4;
        copy_word<VEC>(&dst[j][c], w + (long long)j * D + c0 + c, D - c0 - c);
    }
}

// the same channels of rows [r0, r0 + 256), zeros past D and N
template <bool VEC>
__device__ __forceinline__ void stage_rows(float (&dst)[kRows][kPitch], const float *x,
                                           long long r0, long long N, int D, int c0) {
    if (!VEC) {
        // a warp copies a row's 128 bytes, a word a lane
#pragma unroll 8
        for (int i = threadIdx.x; i < kRows * kDepth; i += kNT) {
            const int r = i / kDepth, c = i % kDepth;
            if (r0 + r < N && c0 + c < D)
                copy4(&dst[r][c], x + (r0 + r) * D + c0 + c);
            else
                dst[r][c] = 0.f;
        }
        return;
    }
#pragma unroll 4
    for (int i = threadIdx.x; i < kRows * (kDepth / 4); i += kNT) {
        const int r = i / (kDepth / 4), c = i % (kDepth / 4) * 4;
        copy_word<VEC>(&dst[r][c], x + (r0 + r) * D + c0 + c, r0 + r < N ? D - c0 - c : 0);
    }
}

// scores of the thread's rows r0 + threadIdx.x (+ 128)
template <int VP, bool VEC>
__device__ __forceinline__ void scores_of(float (&z)[kR][VP], Stage<VP> *st, const float *x,
                                          const float *w, long long r0, long long N, int V,
                                          int D) {
    const int chunks = (D + kDepth - 1) / kDepth;
    float2 s[kR][VP];
#pragma unroll
    for (int k = 0; k < kR; ++k)
#pragma unroll
        for (int j = 0; j < VP; ++j) s[k][j] = make_float2(0.f, 0.f);
    __syncthreads();  // the stages are free
    stage_rows<VEC>(st[0].x, x, r0, N, D, 0);
    stage_table<VP, VEC>(st[0].w, w, V, D, 0);
    copies_end_group();
    for (int i = 0; i < chunks; ++i) {
        if (i + 1 < chunks) {
            Stage<VP> &next = st[(i + 1) & 1];
            stage_rows<VEC>(next.x, x, r0, N, D, (i + 1) * kDepth);
            stage_table<VP, VEC>(next.w, w, V, D, (i + 1) * kDepth);
        }
        copies_end_group();
        copies_wait<1>();
        __syncthreads();
        const Stage<VP> &cur = st[i & 1];
#pragma unroll 2
        for (int c = 0; c < kDepth; c += 4) {
            float4 v[kR];
#pragma unroll
            for (int k = 0; k < kR; ++k)
                v[k] = *reinterpret_cast<const float4 *>(&cur.x[k * kNT + threadIdx.x][c]);
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                if (j >= V) break;
                const float4 q = *reinterpret_cast<const float4 *>(&cur.w[j][c]);
#pragma unroll
                for (int k = 0; k < kR; ++k) {
                    s[k][j] = __ffma2_rn(make_float2(v[k].x, v[k].y), make_float2(q.x, q.y),
                                         s[k][j]);
                    s[k][j] = __ffma2_rn(make_float2(v[k].z, v[k].w), make_float2(q.z, q.w),
                                         s[k][j]);
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kR; ++k)
#pragma unroll
        for (int j = 0; j < VP; ++j) z[k][j] = s[k][j].x + s[k][j].y;
}

template <int VP, bool VEC, bool CAP>
__global__ void __launch_bounds__(kNT)
wide_fwd_kernel(long long N, int V, int D, const float *__restrict__ features,
                const float *__restrict__ weight, const long long *__restrict__ labels, CeOpt o,
                float *__restrict__ loss, float2 *__restrict__ lse_out, float *__restrict__ z_out,
                float *__restrict__ count, float2 *__restrict__ sums) {
    extern __shared__ __align__(16) unsigned char wide_smem[];
    __shared__ float2 sh[kNT / 32];
    Stage<VP> *st = reinterpret_cast<Stage<VP> *>(wide_smem);
    CeSum lsum;
    float cnt = 0.f;
    for (long long r0 = (long long)blockIdx.x * kRows; r0 < N;
         r0 += (long long)gridDim.x * kRows) {
        float z[kR][VP];
        scores_of<VP, VEC>(z, st, features, weight, r0, N, V, D);
#pragma unroll
        for (int k = 0; k < kR; ++k) {
            const long long r = r0 + k * kNT + threadIdx.x;
            if (r >= N) break;
            const int y = ce_label(labels[r], o.ignore, V);
            CeAcc a;
            a.init();
            float zy = 0.f;
#pragma unroll
            for (int j = 0; j < VP; ++j)
                if (j < V) {
                    if (CAP) z[k][j] = o.cap * ce_tanh<false>(z[k][j], o.cap);
                    a.m = fmaxf(a.m, z[k][j]);
                    a.sz += z[k][j];
                    zy = y == j ? z[k][j] : zy;
                }
            const float b = CeAcc::base(a.m);
#pragma unroll
            for (int j = 0; j < VP; ++j)
                if (j < V) a.s += ex2((z[k][j] - b) * kLog2e);
            float2 lse = a.lse();
            float l = 0.f;
            if (y >= 0)
                l = ce_row_loss(lse, zy, a.sz, V, o);
            else if (y == kCeInvalid)
                l = lse.x = ce_nan();
            lse_out[r] = lse;
            if (z_out) {
                float4 *to = reinterpret_cast<float4 *>(z_out) + r * ((V + 3) / 4);
#pragma unroll
                for (int j = 0; j < VP; j += 4)
                    if (j < V)
                        to[j / 4] = make_float4(z[k][j], z[k][j + 1], z[k][j + 2], z[k][j + 3]);
            }
            if (o.reduction == kCeNone) loss[r] = l;
            lsum.add(l);
            cnt += y == kCeIgnored ? 0.f : 1.f;
        }
    }
    const float2 s = ce_block_sum<kNT>(lsum.value(), cnt, sh);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1)
            ce_finish(s.x, s.y, o.reduction, loss, count);
        else
            sums[blockIdx.x] = s;
    }
}

// the loss's derivative in the scores; rows of V floats, rounded up to four
// and zeros there, in both
template <int VP, bool CAP>
__global__ void __launch_bounds__(kDwNT)
wide_probs_kernel(long long N, int V, const long long *__restrict__ labels, CeOpt o,
                  const float2 *__restrict__ lse, CeUpstream u, const float4 *__restrict__ z_in,
                  float4 *__restrict__ p_out) {
    const long long r = (long long)blockIdx.x * kDwNT + threadIdx.x;
    if (r >= N) return;
    const int words = (V + 3) / 4;
    const float *per_row = u.reduction == kCeNone ? u.g : nullptr;
    const int y = ce_label(labels[r], o.ignore, V);
    const bool keep = y != kCeIgnored;
    RowGrad q{};
    if (keep) q = row_grad<true>(r, y, lse[r], o, per_row, common_grad(u), o.eps / (float)V);
#pragma unroll
    for (int w = 0; w < VP / 4; ++w) {
        if (w >= words) break;
        const float4 in = z_in[r * words + w];
        const float z[4] = {in.x, in.y, in.z, in.w};
        float d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = 4 * w + i;
            d[i] = 0.f;
            if (j < V && keep) {
                d[i] = fmaf(q.kz, ce_prob(z[i], q.lse), -q.e);
                if (y == j) d[i] -= q.hit;
                if (CAP) {
                    const float t = z[i] / o.cap;
                    d[i] *= fmaf(-t, t, 1.f);
                }
            }
        }
        p_out[r * words + w] = make_float4(d[0], d[1], d[2], d[3]);
    }
}

// a tile's derivatives and which rows have a label
template <int VP>
struct Derivatives {
    float4 p[2][kDwRows][VP / 4];
    int keep[2][kDwRows];

    __device__ __forceinline__ void load(int b, const float4 *src, const long long *labels,
                                         long long ignore, long long r0, long long N,
                                         int words) {
        for (int i = threadIdx.x; i < kDwRows * words; i += kDwNT) {
            const int r = i / words;
            p[b][r][i % words] = r0 + r < N ? src[(r0 + r) * words + i % words]
                                            : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (threadIdx.x < kDwRows)
            keep[b][threadIdx.x] =
                r0 + threadIdx.x < N && labels[r0 + threadIdx.x] != ignore;
    }
};

// A lane's columns of a block's 128: four side by side (VEC), else every 32nd,
// so that a warp's accesses stay side by side.
template <int VP, bool VEC>
__global__ void __launch_bounds__(kDwNT, 2)
wide_dx_kernel(long long N, int V, int D, const float *__restrict__ weight,
               const long long *__restrict__ labels, long long ignore,
               const float4 *__restrict__ p, float *__restrict__ grad) {
    constexpr int kPer = kDwRows / kDwWarps;
    __shared__ Derivatives<VP> ds;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, words = (V + 3) / 4;
    const int c = blockIdx.y * kChunk + (VEC ? 4 * lane : lane);
    float2 w[VP][2];
#pragma unroll
    for (int j = 0; j < VP; ++j) {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = c + (VEC ? i : 32 * i);
            q[i] = j < V && col < D ? weight[(long long)j * D + col] : 0.f;
        }
        w[j][0] = make_float2(q[0], q[1]);
        w[j][1] = make_float2(q[2], q[3]);
    }
    int b = 0;
    for (long long r0 = (long long)blockIdx.x * kDwRows; r0 < N;
         r0 += (long long)gridDim.x * kDwRows, b ^= 1) {
        ds.load(b, p, labels, ignore, r0, N, words);
        __syncthreads();
#pragma unroll 4
        for (int k = 0; k < kPer; ++k) {
            const int r = warp * kPer + k;
            if (r0 + r >= N) break;
            float2 a[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            // a row without a label is zero whatever the table holds
            if (ds.keep[b][r]) {
#pragma unroll
                for (int j = 0; j < VP; j += 4) {
                    if (j >= V) break;
                    const float4 d = ds.p[b][r][j / 4];
                    const float dv[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        a[0] = __ffma2_rn(f2(dv[i]), w[j + i][0], a[0]);
                        a[1] = __ffma2_rn(f2(dv[i]), w[j + i][1], a[1]);
                    }
                }
            }
            float *to = grad + (r0 + r) * D + c;
            if (VEC) {
                if (c < D)
                    __stcs(reinterpret_cast<float4 *>(to),
                           make_float4(a[0].x, a[0].y, a[1].x, a[1].y));
            } else {
                if (c < D) to[0] = a[0].x;
                if (c + 32 < D) to[32] = a[0].y;
                if (c + 64 < D) to[64] = a[1].x;
                if (c + 96 < D) to[96] = a[1].y;
            }
        }
    }
}

template <bool VEC>
__device__ __forceinline__ float4 load4(const float *p, int c, int D) {
    if (VEC) return *reinterpret_cast<const float4 *>(p + c);
    return make_float4(p[c], c + 32 < D ? p[c + 32] : 0.f, c + 64 < D ? p[c + 64] : 0.f,
                       c + 96 < D ? p[c + 96] : 0.f);
}

template <int VP, bool VEC>
__global__ void __launch_bounds__(kDwNT, 2)
wide_dw_kernel(long long N, int V, int D, const float *__restrict__ features,
               const long long *__restrict__ labels, long long ignore,
               const float4 *__restrict__ p, float *__restrict__ acc) {
    constexpr int kPer = kDwRows / kDwWarps;
    __shared__ float4 sum[VP][32];
    __shared__ Derivatives<VP> ds;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, words = (V + 3) / 4;
    const int c = blockIdx.y * kChunk + (VEC ? 4 * lane : lane);
    int b = 0;
    long long r0 = (long long)blockIdx.x * kDwRows;
    for (bool first = true; r0 < N; first = false) {
        float4 a[VP];
#pragma unroll
        for (int j = 0; j < VP; ++j) a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < kDwChain / kPer && r0 < N;
             ++i, r0 += (long long)gridDim.x * kDwRows, b ^= 1) {
            // eight rows of features a warp on their way with the derivatives
            ds.load(b, p, labels, ignore, r0, N, words);
            float4 x[kPer];
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const long long r = r0 + warp * kPer + k;
                x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < N && c < D) x[k] = load4<VEC>(features + r * D, c, D);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int r = warp * kPer + k;
                if (!ds.keep[b][r]) continue;  // the whole warp alike
#pragma unroll
                for (int j = 0; j < VP; j += 4) {
                    if (j >= V) break;
                    const float4 d = ds.p[b][r][j / 4];
                    const float dv[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        a[j + i].x = fmaf(dv[i], x[k].x, a[j + i].x);
                        a[j + i].y = fmaf(dv[i], x[k].y, a[j + i].y);
                        a[j + i].z = fmaf(dv[i], x[k].z, a[j + i].z);
                        a[j + i].w = fmaf(dv[i], x[k].w, a[j + i].w);
                    }
                }
            }
        }
        for (int k = 0; k < kDwWarps; ++k) {
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
        for (int i = threadIdx.x; i < V * kChunk; i += kDwNT) {
            const int j = i / kChunk, k = i % kChunk, d = blockIdx.y * kChunk + k;
            // column k: lane and component
            const int at = VEC ? k : k % 32 * 4 + k / 32;
            if (d < D) {
                float *to = acc + ((long long)blockIdx.x * V + j) * D + d;
                const float v = reinterpret_cast<const float *>(&sum[j][0])[at];
                *to = first ? v : *to + v;
            }
        }
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

// two stages of shared memory, allowed once a kernel and device
template <int VP, typename K>
cudaError_t allow_stages(K kernel, std::atomic<unsigned long long> &ready) {
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess || (ready.load() >> (dev & 63) & 1)) return err;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(2 * sizeof(Stage<VP>)));
    if (err == cudaSuccess) ready.fetch_or(1ull << (dev & 63));
    return err;
}

}  // namespace

WideShape wide_shape(long long N, int V, int D) {
    WideShape s;
    // three blocks an SM (two stages of 37 KB each)
    s.row_blocks = (int)std::min(ceil_div(N, kRows), 3LL * kSMs);
    s.dw_chunks = (int)ceil_div(D, kChunk);
    s.dx_blocks = (int)std::min(ceil_div(N, kDwRows), std::max(1LL, 4LL * kSMs / s.dw_chunks));
    s.dw_blocks = (int)std::max(
        1LL, std::min(ceil_div(N, 4 * kDwRows), std::max(1LL, 2LL * kSMs / s.dw_chunks)));
    return s;
}

cudaError_t launch_wide_fwd(const NarrowArgs &a, float *z, float *loss, float2 *sums,
                            cudaStream_t st) {
    return by_form(a.V, wide_rows(a, nullptr), a.opt.cap > 0.f, [&](auto vp, auto vec, auto cap) {
        constexpr int VP = decltype(vp)::value;
        auto kernel = wide_fwd_kernel<VP, decltype(vec)::value, decltype(cap)::value>;
        static std::atomic<unsigned long long> ready{0};
        const cudaError_t err = allow_stages<VP>(kernel, ready);
        if (err != cudaSuccess) return err;
        kernel<<<wide_shape(a.N, a.V, a.D).row_blocks, kNT, 2 * sizeof(Stage<VP>), st>>>(
            a.N, a.V, a.D, static_cast<const float *>(a.features),
            static_cast<const float *>(a.weight), a.labels, a.opt, loss, a.lse, z, a.count,
            sums);
        count_launches(1);
        return cudaGetLastError();
    });
}

cudaError_t launch_wide_probs(const NarrowArgs &a, const CeUpstream &u, const float *z, float *p,
                              cudaStream_t st) {
    return by_form(a.V, true, a.opt.cap > 0.f, [&](auto vp, auto, auto cap) {
        wide_probs_kernel<decltype(vp)::value, decltype(cap)::value>
            <<<(unsigned)ceil_div(a.N, kDwNT), kDwNT, 0, st>>>(
                a.N, a.V, a.labels, a.opt, a.lse, u, reinterpret_cast<const float4 *>(z),
                reinterpret_cast<float4 *>(p));
        count_launches(1);
        return cudaGetLastError();
    });
}

cudaError_t launch_wide_dx(const NarrowArgs &a, const float *p, float *grad, cudaStream_t st) {
    return by_form(a.V, wide_rows(a, grad), false, [&](auto vp, auto vec, auto) {
        const WideShape s = wide_shape(a.N, a.V, a.D);
        wide_dx_kernel<decltype(vp)::value, decltype(vec)::value>
            <<<dim3(s.dx_blocks, s.dw_chunks), kDwNT, 0, st>>>(
                a.N, a.V, a.D, static_cast<const float *>(a.weight), a.labels, a.opt.ignore,
                reinterpret_cast<const float4 *>(p), grad);
        count_launches(1);
        return cudaGetLastError();
    });
}

cudaError_t launch_wide_dw(const NarrowArgs &a, const float *p, float *acc, cudaStream_t st) {
    return by_form(a.V, wide_rows(a, nullptr), false, [&](auto vp, auto vec, auto) {
        const WideShape s = wide_shape(a.N, a.V, a.D);
        wide_dw_kernel<decltype(vp)::value, decltype(vec)::value>
            <<<dim3(s.dw_blocks, s.dw_chunks), kDwNT, 0, st>>>(
                a.N, a.V, a.D, static_cast<const float *>(a.features), a.labels, a.opt.ignore,
                reinterpret_cast<const float4 *>(p), acc);
        count_launches(1);
        return cudaGetLastError();
    });
}

}  // namespace gsv
