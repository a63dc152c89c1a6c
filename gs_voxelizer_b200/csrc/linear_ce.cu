// Softmax cross entropy of a linear map: scores X W^T of N feature rows
// against a table of V classes, without keeping the N x V scores.
//
// Forward: the labelled rows are packed into whole 256-row tiles (rows
// without a label cost nothing and cannot leak what they hold), the product
// runs tile by tile and leaves one (maximum, sum) pair per row and class
// tile, and a merge turns the pairs into lse and loss.
// Backward: the scores are computed again in pieces of rows x classes that a
// bounded workspace holds, as P = dloss/dscore in 16 bits, and each piece is
// multiplied into both gradients: dX += P W, dW += P^T X, accumulated in
// float32 and rounded once.
//
// Rounding P to 16 bits costs at most half a step (2^-8 of the value in bf16,
// 2^-11 in fp16), no more than rounding the gradients themselves to the same
// type (against float64: 2.4e-3 of bf16 gradients where the products of an
// unrounded P give 1.7e-3, 2.4e-4 of fp16 ones for 2.1e-4). fp16 keeps P times
// 2^14, over the largest factor that a z-loss brings to a row (as a power of
// two), so that small probabilities stay normal numbers and none overflows.
// float32 inputs keep three bf16 planes of every operand, which hold all 24 bits.
//
// Few channels, few classes of many float32 channels, and few rows have
// kernels of their own (see path_of).
#include "ce_few.cuh"
#include "ce_gemm.cuh"
#include "ce_narrow.cuh"
#include "ce_wide.cuh"

namespace gsv {
namespace {

constexpr int kIdxNT = 1024;
constexpr size_t kPieceBytes = (size_t)256 << 20;  // of P

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }
long long up(long long v, long long a) { return (v + a - 1) / a * a; }

// ------------------------------------------------------------ packed rows

__global__ void __launch_bounds__(kIdxNT)
count_labels_kernel(long long n, const long long *__restrict__ labels, long long ignore,
                    int *__restrict__ counts) {
    const long long i = (long long)blockIdx.x * kIdxNT + threadIdx.x;
    const int c = __syncthreads_count(i < n && labels[i] != ignore);
    if (threadIdx.x == 0) counts[blockIdx.x] = c;
}

// Blocks' counts up to which each block of index_kernel adds up all of them; of
// more it would read the square of their number (391 us for 256^3 rows, 203 with
// a launch that adds them up first).
constexpr int kScan = 64;

// counts -> labelled rows before each block, and total[0] = all of them
__global__ void __launch_bounds__(kIdxNT)
scan_counts_kernel(int nblocks, int *__restrict__ counts, int *__restrict__ total) {
    __shared__ int s_warp[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (nblocks + kIdxNT - 1) / kIdxNT;
    const int b0 = min(nblocks, (int)threadIdx.x * per), b1 = min(nblocks, b0 + per);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += counts[b];
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    int before = upto - mine, all = 0;
    for (int w = 0; w < 32; ++w) {
        if (w < warp) before += s_warp[w];
        all += s_warp[w];
    }
    for (int b = b0; b < b1; ++b) {
        const int c = counts[b];
        counts[b] = before;
        before += c;
    }
    if (threadIdx.x == 0) total[0] = all;
}

// idx / lab of the packed rows in their order; positions from the number of
// labelled rows up to padded are kCeIgnored. total[0] = labelled rows.
__global__ void __launch_bounds__(kIdxNT)
index_kernel(long long n, long long padded, int V, const long long *__restrict__ labels,
             long long ignore, const int *__restrict__ counts, int nblocks,
             int *__restrict__ total, int *__restrict__ idx, int *__restrict__ lab) {
    __shared__ long long s_before[32], s_all[32];
    __shared__ int s_warp[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long i = (long long)blockIdx.x * kIdxNT + threadIdx.x;
    const long long y = i < n ? labels[i] : ignore;
    const bool keep = i < n && y != ignore;
    long long before = 0, all = 0;
    if (nblocks > 1 && nblocks <= kScan) {
        for (int b = threadIdx.x; b < nblocks; b += kIdxNT) {
            const int c = counts[b];
            all += c;
            if (b < (int)blockIdx.x) before += c;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            before += __shfl_xor_sync(0xffffffffu, before, o);
            all += __shfl_xor_sync(0xffffffffu, all, o);
        }
        if (lane == 0) {
            s_before[warp] = before;
            s_all[warp] = all;
        }
    }
    const unsigned ballot = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) s_warp[warp] = __popc(ballot);
    __syncthreads();
    before = all = 0;
    if (nblocks > kScan) {
        before = counts[blockIdx.x];
        all = total[0];
    } else if (nblocks > 1) {
        for (int w = 0; w < 32; ++w) {
            before += s_before[w];
            all += s_all[w];
        }
    }
    int here = 0, block_total = 0;
    for (int w = 0; w < 32; ++w) {
        if (w < warp) here += s_warp[w];
        block_total += s_warp[w];
    }
    if (nblocks == 1) all = block_total;
    if (keep) {
        const long long r = before + here + __popc(ballot & ((1u << lane) - 1u));
        idx[r] = (int)i;
        lab[r] = ce_label(y, ignore, V);
    }
    if (i >= all && i < padded) lab[i] = kCeIgnored;
    if (i == 0) {
        if (nblocks <= kScan) total[0] = (int)all;
        total[1] = 0;  // the merge's ticket
        total[2] = 0;  // the z-loss's largest factor
    }
}

// Splits a float into bf16 planes whose sum it is. Infinities and NaN live
// in the first plane alone, of which the products' sums take them (ce_gemm.cu);
// a finite value that would round to infinity is held at the largest bf16 and
// the remainder follows.
__device__ __forceinline__ void split3(float v, __nv_bfloat16 (&h)[3]) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        h[p] = __float2bfloat16_rn(v);
        float f = __bfloat162float(h[p]);
        if (!isfinite(f)) {
            if (!isfinite(v)) {
                v = 0.f;
                continue;
            }
            h[p] = __ushort_as_bfloat16(v < 0.f ? 0xff7f : 0x7f7f);
            f = __bfloat162float(h[p]);
        }
        v -= f;
    }
}

// How 256 threads cover rows of `chunks` chunks: cx side by side in a row,
// 256 / cx rows.
struct RowShape {
    int cx;
    unsigned blocks;
};
RowShape row_shape(long long rows, long long chunks) {
    int cx = 1;
    while (cx < 256 && cx < chunks) cx *= 2;
    return {cx, (unsigned)((rows + 256 / cx - 1) / (256 / cx))};
}

// dst[plane][rows][ld] = src[idx[r]], rows past the count (up to whole tiles)
// and columns past D zero, eight columns a thread. VEC: rows of src are
// aligned to 16 bytes and D is a multiple of eight.
template <typename T, bool ROWS, bool VEC>
__global__ void __launch_bounds__(256)
pack_kernel(long long rows, int D, long long ld, long long plane, int cx,
            const T *__restrict__ src, const int *__restrict__ idx,
            const int *__restrict__ total, void *__restrict__ dst) {
    const long long r = (long long)blockIdx.x * (256 / cx) + threadIdx.x / cx;
    if (r >= rows) return;
    long long from = r;
    if (ROWS) {
        const long long live = *total;
        if (r >= (live + kCeTileM - 1) / kCeTileM * kCeTileM) return;
        from = r < live ? idx[r] : -1;
    }
    const T *in = src + from * D;
    for (long long c = 8 * (threadIdx.x % cx); c < ld; c += 8 * cx) {
        struct alignas(16) Vec { T t[8]; };
        Vec v;
        if (VEC && from >= 0) {
            v = *reinterpret_cast<const Vec *>(in + c);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v.t[k] = from >= 0 && c + k < D ? in[c + k] : ce_from_float<T>(0.f);
        }
        if constexpr (sizeof(T) == 4) {
            struct alignas(16) Out { __nv_bfloat16 t[8]; };
            Out h[3];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                __nv_bfloat16 q[3];
                split3(v.t[k], q);
#pragma unroll
                for (int p = 0; p < 3; ++p) h[p].t[k] = q[p];
            }
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<Out *>(static_cast<__nv_bfloat16 *>(dst) + p * plane + r * ld +
                                         c) = h[p];
        } else {
            *reinterpret_cast<Vec *>(static_cast<T *>(dst) + r * ld + c) = v;
        }
    }
}

// --------------------------------------------------------- merge and loss

constexpr int kMergeNT = 256;

// One row's (maximum, sum) pairs of all class runs -> lse and loss. SLICES
// parts of the pairs run side by side for 256 / SLICES rows. LOG2: the maxima
// are exponents of two, and stay so in lse. With idx the rows are packed ones:
// lse is kept in their order, the loss goes to the original row, and the pairs
// lie in either order (`packed`).
template <bool LOG2, int SLICES>
__global__ void __launch_bounds__(kMergeNT)
merge_kernel(long long rows, int tiles, int V, bool packed, const float2 *__restrict__ part,
             const float *__restrict__ psum, const float *__restrict__ zt,
             const int *__restrict__ total, const int *__restrict__ idx,
             const int *__restrict__ lab, const long long *__restrict__ labels, CeOpt o,
             float *__restrict__ loss, float2 *__restrict__ lse_out,
             float *__restrict__ count, float2 *__restrict__ block_sums,
             int *__restrict__ ticket, float *__restrict__ zmax) {
    constexpr int kRows = kMergeNT / SLICES;
    __shared__ float sm[SLICES][kRows], ss[SLICES][kRows], sz[SLICES][kRows];
    __shared__ float2 sh[kMergeNT / 32];
    const int lane = threadIdx.x % kRows, slice = threadIdx.x / kRows;
    const long long r = (long long)blockIdx.x * kRows + lane;
    const bool live = r < rows && (!total || r < *total);
    CeAcc a;
    a.init();
    const long long src = live && idx && !packed ? idx[r] : r;
    if (live)
        for (int t = slice; t < tiles; t += SLICES) {
            const float2 p = part[t * rows + src];
            a.merge<LOG2>(p.x, p.y, psum ? psum[t * rows + src] : 0.f);
        }
    if (SLICES > 1) {
        sm[slice][lane] = a.m;
        ss[slice][lane] = a.s;
        sz[slice][lane] = a.sz;
        __syncthreads();
    }
    float l = 0.f, c = 0.f, factor = 0.f;
    if (live && slice == 0) {
        for (int s = 1; s < SLICES; ++s)
            a.merge<LOG2>(sm[s][lane], ss[s][lane], sz[s][lane]);
        const int y = lab ? lab[r] : ce_label(labels[r], o.ignore, V);
        float2 lse = a.lse();
        if (y >= 0)
            l = ce_row_loss(make_float2(LOG2 ? lse.x * kCeLn2 : lse.x, lse.y), zt[src], a.sz, V,
                            o);
        else if (y == kCeInvalid)
            l = lse.x = ce_nan();
        c = y == kCeIgnored ? 0.f : 1.f;
        lse_out[r] = lse;
        if (zmax) factor = ce_z_factor(lse, o);
        if (o.reduction == kCeNone) loss[idx ? idx[r] : r] = l;
    }
    if (zmax) ce_warp_max(factor, zmax);
    const float2 t = ce_block_sum<kMergeNT>(l, c, sh);
    if (gridDim.x == 1) {
        if (threadIdx.x == 0) ce_finish(t.x, t.y, o.reduction, loss, count);
        return;
    }
    if (threadIdx.x == 0) block_sums[blockIdx.x] = t;
    if (!ticket) return;
    // the block that ends last sums all of them, in an order of its own that
    // is the same whichever it is
    __shared__ bool last;
    __shared__ double sl[kMergeNT / 32], sc[kMergeNT / 32];
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(ticket, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double ls = 0.0, cs = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += kMergeNT) {
        const float2 q = __ldcg(block_sums + i);
        ls += q.x;
        cs += q.y;
    }
#pragma unroll
    for (int k = 16; k; k >>= 1) {
        ls += __shfl_xor_sync(0xffffffffu, ls, k);
        cs += __shfl_xor_sync(0xffffffffu, cs, k);
    }
    if ((threadIdx.x & 31) == 0) {
        sl[threadIdx.x >> 5] = ls;
        sc[threadIdx.x >> 5] = cs;
    }
    __syncthreads();
    if (threadIdx.x) return;
    for (int k = 1; k < kMergeNT / 32; ++k) {
        ls += sl[k];
        cs += sc[k];
    }
    ce_finish(ls, cs, o.reduction, loss, count);
}

// few pairs a row: a thread a row; many: eight threads
int merge_rows(int parts) { return parts <= 4 ? kMergeNT : kMergeNT / 8; }

template <bool LOG2>
void launch_merge(long long rows, long long grid_rows, int parts, int V, bool packed,
                  const float2 *part,
                  const float *psum, const float *zt, const int *total, const int *idx,
                  const int *lab, const long long *labels, const CeOpt &o, float *loss,
                  float2 *lse, float *count, float2 *sums, int *ticket, float *zmax,
                  cudaStream_t st) {
    const int per = merge_rows(parts);
    const unsigned blocks = (unsigned)((grid_rows + per - 1) / per);
    const auto kernel = per == kMergeNT ? merge_kernel<LOG2, 1> : merge_kernel<LOG2, 8>;
    kernel<<<blocks, kMergeNT, 0, st>>>(rows, parts, V, packed, part, psum, zt, total, idx, lab,
                                        labels, o, loss, lse, count, sums, ticket, zmax);
    count_launches(1);
}

// -------------------------------------------------------------- gradients

// out[0] (zero before) = largest finite |g| of the labelled rows (an infinite
// one is its own row's, and its factor is infinite over any other)
__global__ void __launch_bounds__(256)
max_abs_kernel(const float *__restrict__ g, const int *__restrict__ idx,
               const int *__restrict__ total, float *__restrict__ out) {
    float m = 0.f;
    const long long n = *total;
    for (long long r = blockIdx.x * 256LL + threadIdx.x; r < n; r += gridDim.x * 256LL) {
        const float a = fabsf(g[idx[r]]);
        if (isfinite(a)) m = fmaxf(m, a);
    }
    ce_warp_max(m, out);
}

// A gradient to be finished: dst[row of r] = scale * sum over splits of
// acc[s][r], rows [0, rows) of a piece that begins at row0, acc's of ld floats
// (a multiple of four). Blocks of 256 threads, cx side by side in a row, four
// columns each. wide: D is a multiple of four and dst aligned to four elements.
struct FinishJob {
    unsigned blocks;
    int cx;
    bool wide;
    long long row0, rows;
    const float *acc;
    long long ld, split;
    int splits;
    void *dst;
};

// ROWS: r is a packed row, and its place idx[row0 + r]
template <typename T, bool ROWS>
__device__ __forceinline__ void finish_block(const FinishJob &f, unsigned block, int D,
                                             const int *idx, const int *total, float scale) {
    const long long r = (long long)block * (256 / f.cx) + threadIdx.x / f.cx;
    if (r >= f.rows) return;
    long long to = r;
    if (ROWS) {
        if (f.row0 + r >= *total) return;
        to = idx[f.row0 + r];
    }
    T *dst = static_cast<T *>(f.dst) + to * D;
    for (long long c = 4 * (threadIdx.x % f.cx); c < D; c += 4 * f.cx) {
        const float *p = f.acc + r * f.ld + c;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < f.splits; ++k) {
            const float4 q = *reinterpret_cast<const float4 *>(p + k * f.split);
            v[0] += q.x;
            v[1] += q.y;
            v[2] += q.z;
            v[3] += q.w;
        }
        if (f.wide) {
            struct alignas(4 * sizeof(T)) Out { T t[4]; };
            Out out;
#pragma unroll
            for (int i = 0; i < 4; ++i) out.t[i] = ce_from_float<T>(v[i] * scale);
            *reinterpret_cast<Out *>(dst + c) = out;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < D) dst[c + i] = ce_from_float<T>(v[i] * scale);
        }
    }
}

// Rows without a label: zero gradient, `bytes` a row. A warp reads 32 labels
// and writes the rows among them.
__device__ __forceinline__ void zero_block(unsigned block, long long n, long long bytes,
                                           const long long *labels, long long ignore,
                                           unsigned char *dst) {
    const long long r = block * 256LL + threadIdx.x;
    const int lane = threadIdx.x & 31;
    unsigned rows = __ballot_sync(0xffffffffu, r < n && labels[r] == ignore);
    while (rows) {
        unsigned char *p = dst + (r - lane + __ffs(rows) - 1) * bytes;
        rows &= rows - 1;
        // whole words from the first aligned byte on (rows are of 2-byte
        // elements at least)
        const int head = (int)min((long long)(-reinterpret_cast<uintptr_t>(p) & 15), bytes);
        for (int i = 2 * lane; i < head; i += 64) *reinterpret_cast<uint16_t *>(p + i) = 0;
        const long long words = (bytes - head) / 16;
        for (long long i = lane; i < words; i += 32)
            reinterpret_cast<int4 *>(p + head)[i] = make_int4(0, 0, 0, 0);
        for (long long i = head + 16 * words + 2 * lane; i < bytes; i += 64)
            *reinterpret_cast<uint16_t *>(p + i) = 0;
    }
}

// What is left of the gradients, in one launch: zero_blocks blocks for the
// rows without a label, x.blocks for the features, w.blocks for the table.
template <typename T>
__global__ void __launch_bounds__(256)
finish_kernel(long long n, int D, const long long *__restrict__ labels, long long ignore,
              T *grad_features, unsigned zero_blocks, const int *__restrict__ idx,
              const int *__restrict__ total, FinishJob x, FinishJob w, CeUpstream upstream) {
    unsigned b = blockIdx.x;
    if (b < zero_blocks) {
        zero_block(b, n, (long long)D * sizeof(T), labels, ignore,
                   reinterpret_cast<unsigned char *>(grad_features));
        return;
    }
    b -= zero_blocks;
    const float scale = ce_grad_scale(upstream);
    if (b < x.blocks)
        finish_block<T, true>(x, b, D, idx, total, scale);
    else
        finish_block<T, false>(w, b - x.blocks, D, idx, total, scale);
}

// dst[i] = sum over splits of acc[s][i], a thread each
template <typename T>
__global__ void __launch_bounds__(256)
sum_splits_kernel(long long n, const float *__restrict__ acc, int splits, T *__restrict__ dst) {
    const long long i = blockIdx.x * 256LL + threadIdx.x;
    if (i >= n) return;
    float v = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) v += acc[s * n + i];
    dst[i] = ce_from_float<T>(v);
}

// the same of few values and many splits: 32 values a block, 32 slices of the
// splits side by side
template <typename T>
__global__ void __launch_bounds__(1024)
reduce_splits_kernel(long long n, const float *__restrict__ acc, int splits,
                     T *__restrict__ dst) {
    __shared__ float sh[32][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const long long i = (long long)blockIdx.x * 32 + lane;
    float v = 0.f;
    if (i < n)
        for (int s = slice; s < splits; s += 32) v += acc[s * n + i];
    sh[slice][lane] = v;
    __syncthreads();
    if (slice || i >= n) return;
    for (int s = 1; s < 32; ++s) v += sh[s][lane];
    dst[i] = ce_from_float<T>(v);
}

// ------------------------------------------------------------------- plan

struct Plan {
    long long N, Np;      // rows, rows in whole tiles
    int V, D, type, planes;
    long long ld;         // of packed features / table
    bool direct;          // the forward reads the rows in place
    bool indexed;         // the labelled rows are listed
    bool pack_w;          // the table cannot be read in place
    bool keep_x, keep_w;  // packed in the state, not in the workspace
    int runs;             // runs of class tiles in the forward
    // backward: pieces and splits
    long long piece_rows, ldp;
    int piece_classes;
    bool one_row_piece;
    bool direct_x, direct_w;  // gradients straight from the product
    int split_x, split_w;
    // workspace offsets (bytes)
    size_t xp, wp, part, psum, zt, sums, gmax, p, dx, dw, bytes;
};

// State (kept between the two directions): count (float, padded to 4 words),
// lse [N] (two floats; of packed rows but on the narrow and wide paths); then,
// where the labelled rows are listed, packed total (int; a ticket and the
// z-loss's largest factor; padded to 4 words), idx [Np], lab [Np], block counts;
// then the packed features and the packed table where they are small: their
// kernels' launches cost more than their memory, and the backward need not
// repeat them. On the wide path the scores instead. A forward without a state
// has its first parts in the workspace.
struct State {
    float *count;
    float2 *lse;
    int *total, *idx, *lab, *counts;
    unsigned char *packed;
};

constexpr size_t kKeepBytes = (size_t)16 << 20;

size_t packed_bytes(long long rows, int D, int type) {
    return (size_t)(type == kCeF32 ? 3 : 1) * rows * up(D, 8) * 2;
}
bool kept(size_t bytes) { return bytes <= kKeepBytes; }

long long state_words(long long N, bool indexed) {
    const long long stats = 4 + up(2 * N, 4);
    if (!indexed) return up(stats, 64);
    return up(stats + 4 + 2 * up(N, kCeTileM) + up((N + kIdxNT - 1) / kIdxNT, 4), 64);
}

State state_of(void *p, long long N, bool indexed) {
    const long long Np = up(N, kCeTileM);
    float *f = static_cast<float *>(p);
    State s{};
    s.count = f;
    s.lse = reinterpret_cast<float2 *>(f + 4);
    if (indexed) {
        s.total = reinterpret_cast<int *>(f + 4 + up(2 * N, 4));
        s.idx = s.total + 4;
        s.lab = s.idx + Np;
        s.counts = s.lab + Np;
    }
    s.packed = reinterpret_cast<unsigned char *>(f + state_words(N, indexed));
    return s;
}

// |dloss / dscore| <= 1 + 2 zeta |lse|. fp16 keeps it times 2^14, and with a
// z-loss over the largest such factor of the labelled rows, which the forward
// leaves in the state. The other types have the range of float32.
float p_scale_of(int type) { return type == kCeF16 ? 16384.f : 1.f; }
float *zmax_of(int type, const CeOpt &o, const State &s) {
    return type == kCeF16 && o.zeta > 0.f ? reinterpret_cast<float *>(s.total + 2) : nullptr;
}

// Parts of the summed axis, at least 512 each. A product of `tiles` tiles takes
// whole rounds of the pairs, and with few tiles that is much more than its
// share: 162 tiles cost 3 rounds for 2.19, four parts each 9 for 8.76 (float32
// table gradient of 8192 x 2086 x 2190: 395 -> 319 us). Every part writes and
// reads 8 bytes a result, which at 5 TB/s is as long as the products of 1000 of
// the summed axis. Up to a part a pair of SMs: 600 us a step of 300000 x 100 x
// 128 float32, 549 of 10^6 x 20 x 64 bf16 and 182 of 100000 x 250 x 256 bf16,
// where 32 parts at most give 646, 587 and 177. `elements` of a part: all take
// 256 MB at most.
int splits_for(long long tiles, long long depth, bool f32, long long elements) {
    int best = 1;
    double cost = 0;
    for (int s = 1; s <= kCePairs && (s == 1 || (depth / s >= 512 &&
                                           s * elements * 4 <= (long long)kPieceBytes)); ++s) {
        const double c = (f32 ? 6. : 1.) * depth / s * ((tiles * s + kCePairs - 1) / kCePairs) +
                         (s > 1 ? 1000. * s * tiles / kCePairs : 0.);
        if (s == 1 || c < cost) {
            cost = c;
            best = s;
        }
    }
    return best;
}

// Which kernels serve a call. kNarrow (linear_ce_narrow.cu, the CUDA cores
// without tiles): where it is the faster. Kernels' time of a training step,
// narrow against tiles (us):
//   rows x classes     D = 8 float32   bf16          D = 4 bf16
//   1000 x 50000       165 : 419       161 : 168     110 : 186
//   16384 x 20000      862 : 2467      839 : 778     500 : 789
//   100000 x 2000      579 : 1464      562 : 553     339 : 554
//   10^6 x 300                         842 : 1265    477 : 1187
//   10^6 x 20                           89 : 514
//                      D = 16 float32  bf16          D = 32 float32  bf16
//   53000 x 203        99 : 180        90 : 98       156 : 170       145 : 80
//   10^6 x 20          148 : 1311      134 : 530                     299 : 530
//   1000 x 50000       267 : 472       250 : 160     584 : 480
// (At D = 8 in 16 bits and thousands of classes the two are level.)
// kWide: few classes, many float32 channels (linear_ce_wide.cu). kFew
// (linear_ce_few.cu): a forward without a backward to follow. Where one follows,
// both directions take tiles: 1 - p of a confident row keeps its digits only if
// its logsumexp comes from the very scores that the backward forms (0.2 % off
// where p = 1 - 1e-5; with sums in another order, the whole of it).
enum Path { kNarrow, kWide, kFew, kTiles };
Path path_of(long long N, int V, int D, int type, CeCall call) {
    const int most = D <= 8 ? INT_MAX
                     : D <= 16 ? (type == kCeF32 ? INT_MAX : 128)
                     : D <= kNarrowD ? (type == kCeF32 ? 256 : 64)
                                     : 0;
    if (V <= most) return kNarrow;
    if (type == kCeF32 && V <= kWideV && N >= kWideRows) return kWide;
    const int few = type == kCeF32 ? kFewRows : kFewRows / 2;
    return call == kCeForwardOnly && N <= few ? kFew : kTiles;
}

// Rows that the forward's tiles read in place, 16 bits and aligned for TMA:
// where packing them costs more than the products of unlabelled rows that it
// saves. Packing moves 4 N D bytes, a share f of unlabelled rows takes
// 2 f N V D operations: at 5 TB/s and 1.4 PFLOP/s they meet at f V = 570.
// One tile of rows cannot become fewer.
bool in_place(long long N, int V, int D, int type) {
    return (N <= kCeTileM || V <= 1024) && type != kCeF32 && D % 8 == 0;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// aligned_x, aligned_w: the inputs are, for TMA
Plan make_plan(long long N, int V, int D, int type, CeCall call, bool aligned_x, bool aligned_w,
               const CeOpt &o) {
    Plan p{};
    p.N = N;
    p.Np = up(N, kCeTileM);
    p.V = V;
    p.D = D;
    p.type = type;
    p.planes = type == kCeF32 ? 3 : 1;
    p.ld = up(D, 8);
    p.pack_w = p.planes == 3 || D % 8 != 0 || !aligned_w;
    p.direct = call != kCeBackward && aligned_x && in_place(N, V, D, type);
    p.indexed = call != kCeForwardOnly || !p.direct;
    size_t at = 0;
    auto take = [&](size_t b) {
        const size_t o = at;
        at += align256(b);
        return o;
    };
    p.sums = take(sizeof(float2) * (size_t)(N / 32 + 1));
    // packed operands: in the state where they are kept
    const size_t xb = packed_bytes(p.Np, D, type), wb = packed_bytes(V, D, type);
    p.keep_x = call != kCeForwardOnly && kept(xb);
    p.keep_w = call != kCeForwardOnly && kept(wb);
    p.xp = p.keep_x ? 0 : take(p.direct ? 0 : xb);
    p.wp = p.keep_w ? (p.keep_x ? align256(xb) : 0) : take(p.pack_w ? wb : 0);
    if (call != kCeBackward) {
        p.runs = ce_runs(N, V, p.planes == 3);
        p.part = take(sizeof(float2) * 2 * (size_t)p.runs * p.Np);
        p.psum = take(o.eps > 0.f ? sizeof(float) * 2 * (size_t)p.runs * p.Np : 0);
        p.zt = take(sizeof(float) * (size_t)p.Np);
        p.bytes = at;
        return p;
    }
    p.gmax = take(sizeof(float));
    // pieces of P: all rows while at least 4096 classes (or all) fit, else
    // 8192 classes (or all) and the rows that fit
    const long long Vp = up(V, 64);
    const long long fit = (long long)(kPieceBytes / (2 * p.planes * p.Np)) / 256 * 256;
    if (fit >= std::min(Vp, 4096LL)) {
        p.piece_rows = p.Np;
        p.ldp = std::min(Vp, fit);
    } else {
        p.ldp = std::min(Vp, 8192LL);
        p.piece_rows = std::max(
            (long long)kCeTileM,
            (long long)(kPieceBytes / (2 * p.planes * p.ldp)) / kCeTileM * kCeTileM);
    }
    p.piece_classes = (int)std::min((long long)V, p.ldp);
    p.one_row_piece = p.piece_rows >= p.Np;
    const bool one_class_piece = p.piece_classes >= V;
    p.piece_rows = std::min(p.piece_rows, p.Np);
    p.p = take((size_t)p.planes * p.piece_rows * p.ldp * 2);
    const int nt = ce_grad_tile(D, p.planes == 3);
    const long long tn = (D + nt - 1) / nt;
    const size_t lda = (size_t)up(D, 4);  // of the float32 sums
    p.split_x = splits_for(p.piece_rows / kCeTileM * tn, p.piece_classes, p.planes == 3,
                           p.piece_rows * lda);
    p.split_w = splits_for(up(p.piece_classes, kCeTileM) / kCeTileM * tn, p.piece_rows,
                           p.planes == 3, (p.one_row_piece ? p.piece_classes : V) * lda);
    p.direct_x = one_class_piece && p.split_x == 1;
    p.direct_w = p.one_row_piece && p.split_w == 1;
    p.dx = take(p.direct_x ? 0 : sizeof(float) * (size_t)p.split_x * p.piece_rows * lda);
    p.dw = take(p.direct_w ? 0
                           : sizeof(float) * (size_t)p.split_w *
                                 (p.one_row_piece ? p.piece_classes : V) * lda);
    p.bytes = at;
    return p;
}

template <typename T>
cudaError_t pack(const Plan &p, bool rows, const void *src, const State &s, void *dst,
                 cudaStream_t st) {
    const bool vec = p.D % 8 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    const long long n = rows ? p.Np : p.V;
    const RowShape g = row_shape(n, p.ld / 8);
    const T *in = static_cast<const T *>(src);
    const auto kernel = rows ? (vec ? pack_kernel<T, true, true> : pack_kernel<T, true, false>)
                             : (vec ? pack_kernel<T, false, true> : pack_kernel<T, false, false>);
    kernel<<<g.blocks, 256, 0, st>>>(n, p.D, p.ld, n * p.ld, g.cx, in, s.idx, s.total, dst);
    count_launches(1);
    return cudaGetLastError();
}

cudaError_t pack_any(const Plan &p, bool rows, const void *src, const State &s, void *dst,
                     cudaStream_t st) {
    switch (p.type) {
        case kCeF32: return pack<float>(p, rows, src, s, dst, st);
        case kCeBf16: return pack<__nv_bfloat16>(p, rows, src, s, dst, st);
        default: return pack<__half>(p, rows, src, s, dst, st);
    }
}

FinishJob finish_job(const Plan &p, long long row0, long long rows, const float *acc,
                     long long split, int splits, void *dst) {
    const int size = p.type == kCeF32 ? 4 : 2;
    const RowShape g = row_shape(rows, (p.D + 3) / 4);
    const bool wide =
        p.D % 4 == 0 && (reinterpret_cast<uintptr_t>(dst) & (4 * size - 1)) == 0;
    return {g.blocks, g.cx, wide, row0, rows, acc, up(p.D, 4), split, splits, dst};
}

template <typename T>
cudaError_t finish(const Plan &p, const State &s, const long long *labels, long long ignore,
                   void *zero, const FinishJob &x, const FinishJob &w, const CeUpstream &u,
                   cudaStream_t st) {
    const unsigned zeros = zero ? (unsigned)((p.N + 255) / 256) : 0;
    const unsigned blocks = zeros + x.blocks + w.blocks;
    if (!blocks) return cudaSuccess;
    finish_kernel<T><<<blocks, 256, 0, st>>>(p.N, p.D, labels, ignore, static_cast<T *>(zero),
                                             zeros, s.idx, s.total, x, w, u);
    count_launches(1);
    return cudaGetLastError();
}

cudaError_t finish_any(const Plan &p, const State &s, const long long *labels, long long ignore,
                       void *zero, const FinishJob &x, const FinishJob &w, const CeUpstream &u,
                       cudaStream_t st) {
    switch (p.type) {
        case kCeF32: return finish<float>(p, s, labels, ignore, zero, x, w, u, st);
        case kCeBf16: return finish<__nv_bfloat16>(p, s, labels, ignore, zero, x, w, u, st);
        default: return finish<__half>(p, s, labels, ignore, zero, x, w, u, st);
    }
}

#define GSV_CE_TRY(expr)                              \
    do {                                              \
        const cudaError_t err_ = (expr);              \
        if (err_ != cudaSuccess) return err_;         \
    } while (0)

unsigned char *x_of(const Plan &p, const State &s, unsigned char *ws) {
    return (p.keep_x ? s.packed : ws) + p.xp;
}
unsigned char *w_of(const Plan &p, const State &s, unsigned char *ws) {
    return (p.keep_w ? s.packed : ws) + p.wp;
}

CeGemm gemm_of(const Plan &p, const State &s, const void *weight, unsigned char *ws,
               const CeOpt &o) {
    CeGemm g{};
    g.bf16 = p.type != kCeF16;
    g.planes = p.planes;
    g.V = p.V;
    g.D = p.D;
    g.opt = o;
    g.splits = 1;
    g.X = {x_of(p, s, ws), p.Np, p.D, p.ld, p.Np * p.ld};
    g.W = p.pack_w ? CeMat{w_of(p, s, ws), p.V, p.D, p.ld, p.V * p.ld}
                   : CeMat{weight, p.V, p.D, p.D, 0};
    g.count = s.total;
    g.lab = s.lab;
    g.idx = s.idx;
    return g;
}

// Workspace of the narrow path: per-block sums, parts of the class splits,
// parts of dX, parts of dW.
struct NarrowPlan {
    int splits, dw_splits;
    long long row_blocks;
    size_t sums, part, psum, zt, dx, dw, bytes;
};

NarrowPlan narrow_plan(long long N, int V, int D, bool backward, const CeOpt &o) {
    NarrowPlan p{};
    const NarrowShape shape = narrow_shape(N, V, D);
    p.splits = shape.class_splits;
    p.dw_splits = shape.dw_blocks;
    p.row_blocks = shape.row_blocks;
    size_t at = 0;
    auto take = [&](size_t b) {
        const size_t a = at;
        at += align256(b);
        return a;
    };
    const size_t parts = p.splits > 1 ? (size_t)p.splits * N : 0;
    if (backward) {
        p.dx = take(parts * D * sizeof(float));
        p.dw = take(sizeof(float) * (size_t)p.dw_splits * V * D);
    } else {
        p.sums = take(sizeof(float2) * (size_t)std::max(p.row_blocks, N / 32 + 1));
        p.part = take(parts * sizeof(float2));
        p.psum = take(o.eps > 0.f ? parts * sizeof(float) : 0);
        p.zt = take(parts ? sizeof(float) * (size_t)N : 0);
    }
    p.bytes = at;
    return p;
}

template <typename T>
cudaError_t narrow_forward(const NarrowArgs &a, float *loss, unsigned char *ws,
                           cudaStream_t st) {
    const NarrowPlan p = narrow_plan(a.N, a.V, a.D, false, a.opt);
    float2 *sums = reinterpret_cast<float2 *>(ws + p.sums);
    float2 *part = reinterpret_cast<float2 *>(ws + p.part);
    float *psum = a.opt.eps > 0.f ? reinterpret_cast<float *>(ws + p.psum) : nullptr;
    float *zt = reinterpret_cast<float *>(ws + p.zt);
    GSV_CE_TRY(launch_narrow_fwd<T>(a, loss, sums, part, psum, zt, st));
    long long blocks = p.row_blocks;
    if (p.splits > 1) {
        blocks = (a.N + merge_rows(p.splits) - 1) / merge_rows(p.splits);
        const auto merge = a.opt.cap > 0.f ? launch_merge<false> : launch_merge<true>;
        merge(a.N, a.N, p.splits, a.V, false, part, psum, zt, nullptr, nullptr, nullptr, a.labels,
              a.opt, loss, a.lse, a.count, sums, nullptr, nullptr, st);
        GSV_CE_TRY(cudaGetLastError());
    }
    if (blocks > 1)
        GSV_CE_TRY(launch_ce_finish(sums, (int)blocks, a.opt.reduction, loss, a.count, st));
    return cudaSuccess;
}

template <typename T>
cudaError_t reduce_splits(long long n, const float *acc, int splits, void *dst,
                          cudaStream_t st) {
    if (n >= 64 * 1024)  // two threads a lane of the device
        sum_splits_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
            n, acc, splits, static_cast<T *>(dst));
    else
        reduce_splits_kernel<T><<<(unsigned)((n + 31) / 32), 1024, 0, st>>>(
            n, acc, splits, static_cast<T *>(dst));
    count_launches(1);
    return cudaGetLastError();
}

template <typename T>
cudaError_t narrow_backward(const NarrowArgs &a, const float *grad_loss, void *gx, void *gw,
                            unsigned char *ws, cudaStream_t st) {
    const NarrowPlan p = narrow_plan(a.N, a.V, a.D, true, a.opt);
    const CeUpstream u{grad_loss, a.count, nullptr, 1.f, a.opt.reduction};
    float *dx = reinterpret_cast<float *>(ws + p.dx), *dw = reinterpret_cast<float *>(ws + p.dw);
    if (gx) {
        GSV_CE_TRY(launch_narrow_dx<T>(a, u, gx, dx, st));
        if (p.splits > 1) GSV_CE_TRY(reduce_splits<T>(a.N * a.D, dx, p.splits, gx, st));
    }
    if (gw) {
        GSV_CE_TRY(launch_narrow_dw<T>(a, u, dw, st));
        GSV_CE_TRY(reduce_splits<T>((long long)a.V * a.D, dw, p.dw_splits, gw, st));
    }
    return cudaSuccess;
}

// Workspace of the wide path: per-block sums; or P, then parts of dW.
struct WidePlan {
    size_t dw, bytes;
};
WidePlan wide_plan(long long N, int V, int D, bool backward) {
    const WideShape s = wide_shape(N, V, D);
    WidePlan w{};
    if (backward) {
        w.dw = align256(wide_p_bytes(N, V));
        w.bytes = w.dw + align256(sizeof(float) * (size_t)s.dw_blocks * V * D);
    } else {
        w.bytes = align256(sizeof(float2) * s.row_blocks);
    }
    return w;
}

cudaError_t wide_forward(const NarrowArgs &a, float *z, float *loss, unsigned char *ws,
                         cudaStream_t st) {
    float2 *sums = reinterpret_cast<float2 *>(ws);
    GSV_CE_TRY(launch_wide_fwd(a, z, loss, sums, st));
    const int blocks = wide_shape(a.N, a.V, a.D).row_blocks;
    if (blocks > 1)
        GSV_CE_TRY(launch_ce_finish(sums, blocks, a.opt.reduction, loss, a.count, st));
    return cudaSuccess;
}

cudaError_t wide_backward(const NarrowArgs &a, const float *z, const float *grad_loss, void *gx,
                          void *gw, unsigned char *ws, cudaStream_t st) {
    const WidePlan w = wide_plan(a.N, a.V, a.D, true);
    const CeUpstream u{grad_loss, a.count, nullptr, 1.f, a.opt.reduction};
    float *p = reinterpret_cast<float *>(ws), *dw = reinterpret_cast<float *>(ws + w.dw);
    GSV_CE_TRY(launch_wide_probs(a, u, z, p, st));
    if (gx) GSV_CE_TRY(launch_wide_dx(a, p, static_cast<float *>(gx), st));
    if (!gw) return cudaSuccess;
    GSV_CE_TRY(launch_wide_dw(a, p, dw, st));
    return reduce_splits<float>((long long)a.V * a.D, dw, wide_shape(a.N, a.V, a.D).dw_blocks,
                                gw, st);
}

// What a forward with a state has packed and kept whatever its pointers were:
// the backward's may be others (of the same contents), and what the forward
// packed only for its pointers' alignment is packed again.
bool x_is_kept(const Plan &p) { return p.keep_x && !in_place(p.N, p.V, p.D, p.type); }
bool w_is_kept(const Plan &p) { return p.keep_w && (p.planes == 3 || p.D % 8 != 0); }

}  // namespace

size_t linear_ce_state_bytes(long long N, int V, int D, int type) {
    const Path path = path_of(N, V, D, type, kCeForward);
    size_t b = 4 * (size_t)state_words(N, path == kTiles);
    if (path == kNarrow) return b;
    if (path == kWide) return b + wide_p_bytes(N, V);
    const size_t xb = packed_bytes(up(N, kCeTileM), D, type), wb = packed_bytes(V, D, type);
    if (kept(xb)) b += align256(xb);
    if (kept(wb)) b += align256(wb);
    return b;
}

size_t linear_ce_workspace_bytes(long long N, int V, int D, int type, CeCall call, bool aligned_x,
                                 bool aligned_w, const CeOpt &o) {
    const bool backward = call == kCeBackward;
    const Path path = path_of(N, V, D, type, call);
    Plan p{};
    if (path == kTiles) p = make_plan(N, V, D, type, call, aligned_x, aligned_w, o);
    // a forward without a state keeps its statistics (and, of tiles, the
    // labelled rows' list) here
    const size_t own =
        call == kCeForwardOnly ? align256(4 * (size_t)state_words(N, p.indexed)) : 0;
    if (path == kTiles) return own + p.bytes;
    return own + (path == kNarrow ? narrow_plan(N, V, D, backward, o).bytes
                  : path == kWide ? wide_plan(N, V, D, backward).bytes
                                  : few_workspace_bytes((int)N, V));
}

cudaError_t launch_linear_ce_forward(long long N, int V, int D, int type,
                                     const void *features, const void *weight,
                                     const long long *labels, const CeOpt &o, float *loss,
                                     void *state, void *workspace, cudaStream_t st) {
    const bool forward_only = state == nullptr;
    const CeCall call = forward_only ? kCeForwardOnly : kCeForward;
    const Path path = path_of(N, V, D, type, call);
    Plan p{};
    if (path == kTiles)
        p = make_plan(N, V, D, type, call, aligned16(features), aligned16(weight), o);
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    const State s = state_of(forward_only ? ws : state, N, p.indexed);
    if (forward_only) ws += align256(4 * (size_t)state_words(N, p.indexed));
    if (path == kNarrow) {
        const NarrowArgs a{N, V, D, features, weight, labels, o, s.lse, s.count};
        switch (type) {
            case kCeF32: return narrow_forward<float>(a, loss, ws, st);
            case kCeBf16: return narrow_forward<__nv_bfloat16>(a, loss, ws, st);
            default: return narrow_forward<__half>(a, loss, ws, st);
        }
    }
    if (path == kWide)
        return wide_forward({N, V, D, features, weight, labels, o, s.lse, s.count},
                            forward_only ? nullptr : reinterpret_cast<float *>(s.packed), loss,
                            ws, st);
    if (path == kFew)
        return launch_few_forward({(int)N, V, D, features, weight, labels, o, s.count},
                                  type, loss, ws, st);
    float *zmax = forward_only ? nullptr : zmax_of(type, o, s);
    if (p.indexed) {
        const int nb = (int)((p.Np + kIdxNT - 1) / kIdxNT);
        if (nb > 1) {
            count_labels_kernel<<<nb, kIdxNT, 0, st>>>(N, labels, o.ignore, s.counts);
            count_launches(1);
        }
        if (nb > kScan) {
            scan_counts_kernel<<<1, kIdxNT, 0, st>>>(nb, s.counts, s.total);
            count_launches(1);
        }
        index_kernel<<<nb, kIdxNT, 0, st>>>(N, p.Np, V, labels, o.ignore, s.counts, nb, s.total,
                                            s.idx, s.lab);
        count_launches(1);
        GSV_CE_TRY(cudaGetLastError());
    }
    // merged by packed rows, which leaves out those without a label
    if (o.reduction == kCeNone && p.indexed)
        GSV_CE_TRY(cudaMemsetAsync(loss, 0, sizeof(float) * (size_t)N, st));
    if (!p.direct) GSV_CE_TRY(pack_any(p, true, features, s, x_of(p, s, ws), st));
    if (p.pack_w) GSV_CE_TRY(pack_any(p, false, weight, s, w_of(p, s, ws), st));
    CeGemm g = gemm_of(p, s, weight, ws, o);
    g.product = kCeScores;
    g.rows = p.Np;
    g.nv = V;
    g.runs = p.runs;
    g.part = reinterpret_cast<float2 *>(ws + p.part);
    g.psum = o.eps > 0.f ? reinterpret_cast<float *>(ws + p.psum) : nullptr;
    g.zt = reinterpret_cast<float *>(ws + p.zt);
    if (p.direct) {
        g.X = {features, N, D, D, 0};
        g.rows = N;
        g.count = g.lab = g.idx = nullptr;
        g.labels = labels;
    }
    GSV_CE_TRY(launch_ce_gemm(g, st));
    const int per = merge_rows(2 * p.runs), mb = (int)((N + per - 1) / per);
    float2 *sums = reinterpret_cast<float2 *>(ws + p.sums);
    launch_merge<false>(g.rows, N, 2 * p.runs, V, !p.direct, g.part, g.psum, g.zt,
                        s.total, s.idx, s.lab, labels, o, loss, s.lse, s.count, sums,
                        p.indexed ? s.total + 1 : nullptr, zmax, st);
    GSV_CE_TRY(cudaGetLastError());
    if (mb > 1 && !p.indexed)
        GSV_CE_TRY(launch_ce_finish(sums, mb, o.reduction, loss, s.count, st));
    return cudaSuccess;
}

cudaError_t launch_linear_ce_backward(long long N, int V, int D, int type,
                                      const void *features, const void *weight,
                                      const long long *labels, const CeOpt &o, void *state,
                                      const float *grad_loss, void *grad_features,
                                      void *grad_weight, void *workspace, cudaStream_t st) {
    if (!grad_features && !grad_weight) return cudaSuccess;
    const Path path = path_of(N, V, D, type, kCeBackward);
    const State s = state_of(state, N, path == kTiles);
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    if (path == kNarrow) {
        const NarrowArgs a{N, V, D, features, weight, labels, o, s.lse, s.count};
#define GSV_CE_T(T) narrow_backward<T>(a, grad_loss, grad_features, grad_weight, ws, st)
        switch (type) {
            case kCeF32: return GSV_CE_T(float);
            case kCeBf16: return GSV_CE_T(__nv_bfloat16);
            default: return GSV_CE_T(__half);
        }
#undef GSV_CE_T
    }
    if (path == kWide)
        return wide_backward({N, V, D, features, weight, labels, o, s.lse, s.count},
                             reinterpret_cast<const float *>(s.packed), grad_loss, grad_features,
                             grad_weight, ws, st);
    const Plan p =
        make_plan(N, V, D, type, kCeBackward, aligned16(features), aligned16(weight), o);
    float *gmax = type == kCeF16 ? reinterpret_cast<float *>(ws + p.gmax) : nullptr;
    const bool none = o.reduction == kCeNone;
    if (!x_is_kept(p)) GSV_CE_TRY(pack_any(p, true, features, s, x_of(p, s, ws), st));
    if (p.pack_w && !w_is_kept(p))
        GSV_CE_TRY(pack_any(p, false, weight, s, w_of(p, s, ws), st));
    if (none && gmax) {
        GSV_CE_TRY(cudaMemsetAsync(gmax, 0, sizeof(float), st));
        const int nb = (int)std::min<long long>(kSMs, (N + 1023) / 1024);
        max_abs_kernel<<<nb, 256, 0, st>>>(grad_loss, s.idx, s.total, gmax);
        count_launches(1);
        GSV_CE_TRY(cudaGetLastError());
    }
    CeGemm g = gemm_of(p, s, weight, ws, o);
    g.lse = s.lse;
    g.p_out = ws + p.p;
    g.p_scale = p_scale_of(type);
    g.grow = none ? grad_loss : nullptr;
    g.gmax = gmax;
    g.up = {grad_loss, s.count, gmax, 1.f / g.p_scale, o.reduction, zmax_of(type, o, s)};
    float *dx = reinterpret_cast<float *>(ws + p.dx);
    float *dw = reinterpret_cast<float *>(ws + p.dw);
    g.acc_ld = up(D, 4);
    const long long x_split = p.piece_rows * g.acc_ld;
    const long long w_split = (long long)(p.one_row_piece ? p.piece_classes : V) * g.acc_ld;
    for (long long r0 = 0; r0 < p.Np; r0 += p.piece_rows) {
        g.row0 = r0;
        g.rows = std::min(p.piece_rows, p.Np - r0);
        for (int v0 = 0; v0 < V; v0 += p.piece_classes) {
            g.v0 = v0;
            g.nv = std::min(p.piece_classes, V - v0);
            g.P = {ws + p.p, g.rows, g.nv, p.ldp, p.piece_rows * p.ldp};
            g.product = kCeProbs;
            GSV_CE_TRY(launch_ce_gemm(g, st));
            if (grad_features) {
                CeGemm x = g;
                x.product = kCeGradX;
                x.splits = p.split_x;
                x.acc = dx;
                x.acc_split = x_split;
                x.add = v0 > 0;
                x.dst = p.direct_x ? grad_features : nullptr;
                GSV_CE_TRY(launch_ce_gemm(x, st));
            }
            if (grad_weight) {
                CeGemm w = g;
                w.product = kCeGradW;
                w.splits = p.split_w;
                w.acc = p.one_row_piece ? dw : dw + (long long)v0 * g.acc_ld;
                w.acc_split = w_split;
                w.add = r0 > 0;
                w.dst = p.direct_w ? grad_weight : nullptr;
                GSV_CE_TRY(launch_ce_gemm(w, st));
                // one class piece of several: the buffer is the next one's
                if (p.one_row_piece && !p.direct_w && p.piece_classes < V)
                    GSV_CE_TRY(finish_any(
                        p, s, labels, o.ignore, nullptr, FinishJob{},
                        finish_job(p, 0, g.nv, dw, w_split, p.split_w,
                                   static_cast<unsigned char *>(grad_weight) +
                                       (size_t)v0 * D * (type == kCeF32 ? 4 : 2)),
                        g.up, st));
            }
        }
        if (grad_features && !p.direct_x && !p.one_row_piece)
            GSV_CE_TRY(finish_any(
                p, s, labels, o.ignore, nullptr,
                finish_job(p, r0, g.rows, dx, x_split, p.split_x, grad_features), FinishJob{},
                g.up, st));
    }
    FinishJob x{}, w{};
    if (grad_features && !p.direct_x && p.one_row_piece)
        x = finish_job(p, 0, p.Np, dx, x_split, p.split_x, grad_features);
    if (grad_weight && !p.direct_w && (!p.one_row_piece || p.piece_classes >= V))
        w = finish_job(p, 0, V, dw, w_split, p.split_w, grad_weight);
    return finish_any(p, s, labels, o.ignore, grad_features, x, w, g.up, st);
}

}  // namespace gsv
