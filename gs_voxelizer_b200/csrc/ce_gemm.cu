// The matrix products of the linear class loss: plain tiles on the CUDA
// cores. A block computes 64 x 64 of the product from 16-deep slices staged
// in shared memory as float32 (the planes of a float32 operand summed), then
// each of 64 threads takes one row of the tile through the epilogue.
#include "ce_gemm.cuh"

namespace gsv {
namespace {

constexpr int kT = 64, kKB = 16;

__device__ __forceinline__ float load16(const void *p, long long i, bool bf16) {
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i])
                : __half2float(static_cast<const __half *>(p)[i]);
}

__device__ __forceinline__ float at(const CeMat &m, long long r, long long c, int planes,
                                    bool bf16) {
    if (r >= m.rows || c >= m.cols) return 0.f;
    float v = 0.f;
    for (int p = planes - 1; p >= 0; --p)
        v += load16(m.ptr, p * m.plane + r * m.ld + c, bf16);
    return v;
}

__global__ void __launch_bounds__(256)
gemm_kernel(CeGemm g) {
    __shared__ float As[kKB][kT + 1], Bs[kKB][kT + 1], C[kT][kT + 1];
    const long long m0 = (long long)blockIdx.x * kT, n0 = (long long)blockIdx.y * kT;
    long long live = g.rows;
    if (g.count) live = max(0LL, min(live, (long long)*g.count - g.row0));
    const bool scores = g.product <= kCeProbs;
    long long k0 = 0, k1 = scores ? g.D : g.product == kCeGradX ? g.nv : live;
    // the probabilities are written (as zeros) up to whole 128-row tiles
    if (g.product != kCeGradW && m0 >= (live + 127) / 128 * 128) return;
    if (!scores) {
        const long long per = ((k1 + g.splits - 1) / g.splits + kKB - 1) / kKB * kKB;
        k0 = min(k1, per * blockIdx.z);
        k1 = min(k1, k0 + per);
    }
    float acc[4][4] = {};
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (long long k = k0; k < k1; k += kKB) {
        for (int e = threadIdx.x; e < kKB * kT; e += 256) {
            const int i = e % kT, kk = e / kT;
            float a = 0.f, b = 0.f;
            if (k + kk < k1) {
                if (scores) {
                    a = at(g.X, g.row0 + m0 + i, k + kk, g.planes, g.bf16);
                    b = at(g.W, g.v0 + n0 + i, k + kk, g.planes, g.bf16);
                } else if (g.product == kCeGradX) {
                    a = at(g.P, m0 + i, k + kk, g.planes, g.bf16);
                    b = at(g.W, g.v0 + k + kk, n0 + i, g.planes, g.bf16);
                } else {
                    a = at(g.P, k + kk, m0 + i, g.planes, g.bf16);
                    b = at(g.X, g.row0 + k + kk, n0 + i, g.planes, g.bf16);
                }
            }
            As[kk][i] = a;
            Bs[kk][i] = b;
        }
        __syncthreads();
        for (int kk = 0; kk < kKB; ++kk)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = fmaf(As[kk][ty * 4 + i], Bs[kk][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    if (!scores) {
        const long long M = g.product == kCeGradX ? g.rows : g.nv;
        float *out = g.out + blockIdx.z * g.out_split;
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const long long m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
                if (m < M && n < g.D)
                    out[m * g.D + n] = (g.add ? out[m * g.D + n] : 0.f) + acc[i][j];
            }
        return;
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) C[ty * 4 + i][tx * 4 + j] = acc[i][j];
    __syncthreads();
    if (threadIdx.x >= kT) return;
    const long long r = m0 + threadIdx.x;  // row of the piece
    if (r >= g.rows) return;
    const float *c = C[threadIdx.x];
    int y = kCeIgnored;
    if (r < live)
        y = g.lab ? g.lab[g.row0 + r] : ce_label(g.labels[g.row0 + r], g.opt.ignore, g.V);
    const int ncols = (int)min((long long)kT, g.nv - n0);
    if (g.product == kCeScores) {
        CeAcc a;
        a.init();
        for (int j = 0; j < ncols; ++j) {
            const float z = ce_cap(c[j], g.opt.cap);
            a.merge(z, 1.f, z);
            if (y == g.v0 + n0 + j) g.zt[r] = z;
        }
        g.part[blockIdx.y * g.rows + r] = make_float2(a.m, a.s);
        if (g.psum) g.psum[blockIdx.y * g.rows + r] = a.sz;
        return;
    }
    const long long src = r < live ? (g.idx ? g.idx[g.row0 + r] : g.row0 + r) : 0;
    const float lse = y == kCeIgnored ? 0.f : g.lse[src];
    for (int j = 0; j < kT; ++j) {
        const long long col = n0 + j;
        if (col >= g.P.ld) break;
        float d = 0.f;
        if (y != kCeIgnored && col < g.nv) {
            const float z = ce_cap(c[j], g.opt.cap);
            d = (1.f + 2.f * g.opt.zeta * lse) * ex2(fmaf(z, kLog2e, -lse * kLog2e)) -
                g.opt.eps / (float)g.V;
            if (y == g.v0 + col) d -= 1.f - g.opt.eps;
            if (g.opt.cap > 0.f) d *= 1.f - (z / g.opt.cap) * (z / g.opt.cap);
        }
        d *= g.p_scale;
        for (int p = 0; p < g.planes; ++p) {
            const long long o = p * g.P.plane + r * g.P.ld + col;
            if (g.bf16) {
                const __nv_bfloat16 h = __float2bfloat16_rn(d);
                static_cast<__nv_bfloat16 *>(g.p_out)[o] = h;
                d -= __bfloat162float(h);
            } else {
                static_cast<__half *>(g.p_out)[o] = __float2half_rn(d);
            }
        }
    }
}

}  // namespace

cudaError_t launch_ce_gemm(const CeGemm &g, cudaStream_t stream) {
    long long m = g.rows, n = g.nv;
    int z = 1;
    if (g.product == kCeProbs) n = g.P.ld;
    if (g.product == kCeGradX) n = g.D;
    if (g.product == kCeGradW) m = g.nv, n = g.D;
    if (g.product >= kCeGradX) z = g.splits;
    gemm_kernel<<<dim3((unsigned)((m + kT - 1) / kT), (unsigned)((n + kT - 1) / kT), z), 256, 0,
                  stream>>>(g);
    count_launches(1);
    return cudaGetLastError();
}

}  // namespace gsv
