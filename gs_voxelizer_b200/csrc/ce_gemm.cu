// The matrix products of the linear class loss on the 5th-generation tensor
// cores: 256 x 256 tiles by pairs of SMs (tcgen05 cta_group::2), operands
// staged by TMA, accumulators in tensor memory, the loss in the epilogue.
//
// Work: a CTA pair takes units of the product one after another (persistent,
// one CTA a SM). Each CTA stages its 128 rows of A and its half of B, 64 deep
// a stage; the leader's MMA thread multiplies both halves. 256 x 256 tiles
// need 32 KB of operands a stage and SM for 2 x 256 x 256 x 64 products, two
// thirds of what 128 x 256 tiles of a single SM load: the L2 could not feed
// those at the tensor cores' rate. (float32: 256 x 128 tiles of three planes,
// 72 KB of operands for six products.) Two accumulators alternate, so that the
// epilogue of a tile (eight warps) runs under the next tile's products.
//
// Operand layouts: X W^T reads both operands along the contiguous axis
// (K-major); the gradients sum over rows or classes, the strided axis, and
// read P, W and X in place as MN-major tiles. No operand is transposed.
//
// What bounds it: the power limit. The MMAs take 99.5 % of the cycles (8192 x
// 32768 x 4096: 1.845 of 1.835 million ideal ones), the clock falls to what
// 1000 W allow; 8192 x 131072 x 4096 takes 6.6 to 6.7 ms a product, 1.32
// PFLOP/s, against 1.39 of a plain library product sustained (42765 x 26421 x
// 621 in float32, six products each: 5.6 to 8.1 ms, 1.50 to 1.04 PFLOP/s). Small products
// are bound by their turn-around, about 6 us a launch.
//
// Waits are bounded: on a timeout a role sets g_ce_error, leaves its loop and
// the kernel ends, its copies done and its tensor memory freed; the result is
// invalid.
#include <cuda.h>

#include <atomic>

#include "ce_gemm.cuh"

namespace gsv {

// Nonzero after a product gave up on a barrier wait; read and cleared
// through the C ABI (gsv_device_error).
__device__ int g_ce_error = 0;

namespace {

constexpr int kDepth = 64;                       // K a stage
constexpr int kABytes = 128 * kDepth * 2;        // per CTA and plane
constexpr int kEpiWarps = 8;
// A stage holds all planes of its A and B halves: six plane pairs are
// multiplied out of one float32 stage, which is half the loads of a stage a
// pair (those bound the tiles of 128 columns at 1.09 PFLOP/s).
template <bool F32>
struct Shape {
    static constexpr int kPlanes = F32 ? 3 : 1;
    static constexpr int kStages = F32 ? 3 : 6;
    static constexpr int kTile = F32 ? 128 : kCeTileN;  // columns, at most
    static constexpr int kBBytes = kTile / 2 * kDepth * 2;
    static constexpr int kStageBytes = kPlanes * (kABytes + kBBytes);
    // rows of 32 that a warp turns at a time
    static constexpr int kTurn = F32 ? 8 : 32;
    static constexpr int kSmemBytes =
        kStages * kStageBytes + 1024 + kEpiWarps * kTurn * 33 * 4;
};
constexpr int kMaxStages = 6;
constexpr int kThreads = (4 + kEpiWarps) * 32;
constexpr int kCols = 512;
constexpr int kSpinLimit = 1 << 24;

struct Barriers {
    uint64_t full[kMaxStages], empty[kMaxStages], tfull[2], tempty[2];
    uint32_t tmem;
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// One lane of the warp. The compiler knows it for one thread, which a test of
// the lane number does not tell it: with that test each tcgen05.mma was
// issued behind a loop over the active lanes, and the MMAs ran at 190 clocks
// each instead of 128 (256 x 256 x 16), whatever fed them.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(p));
    return p != 0;
}
// address of the leader's copy of a barrier
__device__ __forceinline__ uint32_t in_leader(uint32_t a) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ void bar_init(uint64_t *b, int n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(n));
}
__device__ __forceinline__ bool bar_wait(uint64_t *b, uint32_t parity) {
    const uint32_t a = smem_addr(b);
    for (int it = 0; it < kSpinLimit; ++it) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(a), "r"(parity)
            : "memory");
        if (done) return true;
    }
    atomicExch(&g_ce_error, 1);
    return false;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
                 "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// box of 64 columns from column x, rows from y on, plane z, into shared
// memory at dst; its bytes are counted at the leader's barrier
__device__ __forceinline__ void tma_load(const CUtensorMap *map, uint32_t dst, uint32_t bar,
                                         int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile"
        ".mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Shared-memory descriptors of 128-byte-swizzled tiles (8 rows of 128 bytes
// repeat every 1024). K-major: rows of the tile, 64 K each; MN-major: rows
// of K, 64 of M or N each, the next 64 in another box 8 KB on.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, bool mn_major) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(mn_major ? 8192 >> 4 : 1) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// 16 K further: 32 bytes of a row, or 16 rows
__device__ __forceinline__ uint64_t k_step(bool mn_major) { return mn_major ? 128 : 2; }

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                    uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrives at the barrier of both CTAs when the MMAs so far are done
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster"
        ".multicast::cluster.b64 [%0], %1;"
        ::"r"(smem_addr(bar)), "h"((unsigned short)3)
        : "memory");
}

__device__ __forceinline__ void load32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void load_wait(uint32_t (&r)[32]) {
    // the registers pass through, so that no use moves above the wait
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                   "+r"(r[27]), "+r"(r[28])
                 ::"memory");
    asm volatile("" : "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}

__device__ __forceinline__ void store8(void *p, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void store4(void *p, const uint32_t *v) {
    asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3])
                 : "memory");
}
__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return reinterpret_cast<const uint32_t &>(h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return reinterpret_cast<const uint32_t &>(h);
}

// The grid's work, the same for every role: units (m tile, n tile, split or
// run), each `tiles` accumulators long.
struct Work {
    int mtiles, ntiles, units;
    int kblocks;          // 64-deep blocks a plane pair
    long long K;
    long long live;       // rows in use of the piece
};

template <int PRODUCT>
__device__ __forceinline__ Work work_of(const CeGemm &g, int nt) {
    Work w;
    w.live = g.rows;
    if (g.count) w.live = max(0LL, min(w.live, (long long)*g.count - g.row0));
    const long long M = PRODUCT == kCeGradW ? g.nv : w.live;
    w.mtiles = (int)((M + kCeTileM - 1) / kCeTileM);
    w.ntiles = ((PRODUCT <= kCeProbs ? g.nv : g.D) + nt - 1) / nt;
    w.K = PRODUCT <= kCeProbs ? g.D : PRODUCT == kCeGradX ? g.nv : w.live;
    w.kblocks = (int)((w.K + kDepth - 1) / kDepth);
    w.units = w.mtiles * (PRODUCT == kCeScores ? g.runs : w.ntiles * g.splits);
    return w;
}

struct Unit {
    int m, n0, n1, split, k0, k1;  // n tiles [n0, n1), K blocks [k0, k1)
    int chunks;                    // parts of [k0, k1), see kChunk
    // the unit's accumulators, one after another
    __device__ __forceinline__ int steps() const { return (n1 - n0) * chunks; }
};

// float32 products are accumulated in tensor memory over 512 of K at most
// and summed in registers from there: the tensor cores truncate
// each addition, which over 4000 of K cost 4e-6 of the result (16 at a time;
// 5e-7 over 512). 16-bit results do not see it.
constexpr int kChunk = 512 / kDepth;

// Scores: m fastest, so that the pairs in flight share class tiles and the
// rows stay in L2. Gradients: the channels' tiles fastest, so that the pairs
// in flight share P, which is the larger operand and is then read once (with
// m fastest, the table's gradient read a 131 MB P three and a half times).
template <int PRODUCT, bool F32>
__device__ __forceinline__ Unit unit_of(const CeGemm &g, const Work &w, int u) {
    Unit t;
    t.split = 0;
    t.k0 = 0;
    t.k1 = w.kblocks;
    if (PRODUCT <= kCeProbs) {
        t.m = u % w.mtiles;
        u /= w.mtiles;
    } else {
        t.n0 = u % w.ntiles;
        u /= w.ntiles;
        t.m = u % w.mtiles;
        u /= w.mtiles;
    }
    if (PRODUCT == kCeScores) {
        // products below 2^32 (2^22 tiles at most, 2 kCePairs runs), divided
        // in 32 bits: every role does this for every unit
        t.n0 = (int)((unsigned)w.ntiles * (unsigned)u / (unsigned)g.runs);
        t.n1 = (int)((unsigned)w.ntiles * (unsigned)(u + 1) / (unsigned)g.runs);
        t.split = u;
    } else {
        if (PRODUCT == kCeProbs) t.n0 = u;
        t.n1 = t.n0 + 1;
    }
    if (PRODUCT >= kCeGradX) {
        t.split = u;
        // (2^25 blocks at most, kCePairs splits)
        t.k0 = (int)((unsigned)w.kblocks * (unsigned)t.split / (unsigned)g.splits);
        t.k1 = (int)((unsigned)w.kblocks * (unsigned)(t.split + 1) / (unsigned)g.splits);
    }
    t.chunks = F32 ? max(1, (t.k1 - t.k0 + kChunk - 1) / kChunk) : 1;
    return t;
}

// What the epilogue needs of a row: its class, logsumexp, upstream gradient.
struct RowInfo {
    int y;
    float2 lse;
    float g;
};

// Plane pairs of a float32 product: (2,0) (0,2) (1,1) (1,0) (0,1), summed in
// an accumulator of their own beside the first, and (0,0): what the tensor
// cores truncate is relative to the sum at hand. The pairs left out are below
// 2^-26 of the whole.
constexpr int kPairs32 = 6;
__device__ __forceinline__ constexpr int plane_a(int p) { return (0x001102 >> (4 * p)) & 3; }
__device__ __forceinline__ constexpr int plane_b(int p) { return (0x010120 >> (4 * p)) & 3; }

// F32: three planes
template <int PRODUCT, bool CAP, bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
ce_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const CeGemm g, const int nt) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ Barriers S;
    using Sh = Shape<F32>;
    constexpr int kStages = Sh::kStages, kStageBytes = Sh::kStageBytes;
    // the same offset in both CTAs: the MMA reads both through one descriptor
    const uint32_t smem0 = (smem_addr(smem_raw) + 1023) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    constexpr bool kAMn = PRODUCT == kCeGradW;
    constexpr bool kBMn = PRODUCT >= kCeGradX;
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            bar_init(&S.full[i], 1);
            bar_init(&S.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&S.tfull[i], 1);
            bar_init(&S.tempty[i], 2 * kEpiWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_addr(&S.tmem)),
                     "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        fence_before();
    }
    __syncthreads();
    cluster_sync();
    fence_after();
    const uint32_t tmem = S.tmem;
    const Work w = work_of<PRODUCT>(g, nt);

    if (warp == 0 && elect_one()) {
        // ------------------------------------------------------ producer
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        const uint32_t bytes = 2 * Sh::kPlanes * (kABytes + nt / 2 * kDepth * 2);
        for (int u = first; ok && u < w.units; u += step) {
            const Unit t = unit_of<PRODUCT, F32>(g, w, u);
            const int m_at = t.m * kCeTileM + (int)rank * 128;
            for (int i = 0; ok && i < t.steps(); ++i) {
                const int n_at = (t.n0 + i / t.chunks) * nt + (int)rank * (nt / 2);
                const int k0 = t.k0 + (F32 ? i % t.chunks * kChunk : 0);
                const int k1 = F32 ? min(t.k1, k0 + kChunk) : t.k1;
                for (int k = k0; k < k1; ++k) {
                    if (!bar_wait(&S.empty[stage], phase ^ 1)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = in_leader(smem_addr(&S.full[stage]));
                    if (rank == 0)
                        asm volatile(
                            "mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                                smem_addr(&S.full[stage])),
                            "r"(bytes)
                            : "memory");
                    const int kk = k * kDepth;
#pragma unroll
                    for (int p = 0; p < Sh::kPlanes; ++p) {
                        const uint32_t a = smem0 + stage * kStageBytes + p * kABytes;
                        const uint32_t b = smem0 + stage * kStageBytes +
                                           Sh::kPlanes * kABytes + p * Sh::kBBytes;
                        if (kAMn) {
                            tma_load(&map_a, a, bar, m_at, kk, p);
                            tma_load(&map_a, a + 8192, bar, m_at + 64, kk, p);
                        } else {
                            const long long r0 = PRODUCT == kCeGradX ? 0 : g.row0;
                            tma_load(&map_a, a, bar, kk, (int)(r0 + m_at), p);
                        }
                        if (kBMn) {
                            const int r0 = PRODUCT == kCeGradX ? g.v0 : (int)g.row0;
                            for (int h = 0; h < nt / 2; h += 64)
                                tma_load(&map_b, b + h * 128, bar, n_at + h, r0 + kk, p);
                        } else {
                            tma_load(&map_b, b, bar, kk, g.v0 + n_at, p);
                        }
                    }
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        // After a timeout (seconds) a millisecond more for copies in flight.
        for (int i = 0; !ok && i < 1000; ++i) __nanosleep(1000);
        // Every load is consumed, and every arrival at this CTA's barriers
        // has come, before the CTA may end.
        for (int i = 0; ok && i < kStages; ++i) {
            ok = bar_wait(&S.empty[stage], phase ^ 1);
            if (++stage == kStages) {
                stage = 0;
                phase ^= 1;
            }
        }
    } else if (warp == 1 && rank == 0 && elect_one()) {
        // ----------------------------------------------------------- MMA
        // D float32, A and B bf16 or fp16, M = 256
        const uint32_t type = g.bf16 ? 1u : 0u;
        const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)kAMn << 15) |
                               ((uint32_t)kBMn << 16) | ((uint32_t)(nt >> 3) << 17) |
                               ((256u >> 4) << 24);
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int u = first; ok && u < w.units; u += step) {
            const Unit t = unit_of<PRODUCT, F32>(g, w, u);
            if (t.k0 == t.k1) continue;
            for (int i = 0; ok && i < t.steps(); ++i) {
                const int k0 = t.k0 + (F32 ? i % t.chunks * kChunk : 0);
                const int k1 = F32 ? min(t.k1, k0 + kChunk) : t.k1;
                if (!bar_wait(&S.tempty[acc], acc_phase ^ 1)) {
                    ok = false;
                    break;
                }
                fence_after();
                const uint32_t d = tmem + acc * kCeTileN;
                for (int k = k0; k < k1; ++k) {
                    if (!bar_wait(&S.full[stage], phase)) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    const uint32_t a = smem0 + stage * kStageBytes;
                    const uint32_t b = a + Sh::kPlanes * kABytes;
                    // the last block may end early (its rest is zeros)
                    const long long left = w.K - (long long)k * kDepth;
                    const int steps = left >= kDepth ? 4 : (int)((left + 15) / 16);
#pragma unroll
                    for (int p = 0; p < (F32 ? kPairs32 : 1); ++p) {
                        const int pa = F32 ? plane_a(p) : 0, pb = F32 ? plane_b(p) : 0;
                        uint64_t da = tile_desc(a + pa * kABytes, kAMn);
                        uint64_t db = tile_desc(b + pb * Sh::kBBytes, kBMn);
                        const bool small = F32 && p < kPairs32 - 1;
                        uint32_t accumulate = k > k0 || (small && p > 0);
                        for (int j = 0; j < steps; ++j) {
                            mma(d + (small ? Sh::kTile : 0), da, db, idesc, accumulate);
                            accumulate = 1;
                            da += k_step(kAMn);
                            db += k_step(kBMn);
                        }
                    }
                    commit(&S.empty[stage]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                commit(&S.tfull[acc]);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------ epilogue
        const int q = warp & 3, half = (warp - 4) >> 2;
        const uint32_t tlane = tmem + ((uint32_t)(q * 32) << 16);
        const int chunks = (nt + 31) / 32;
        const CeOpt o = g.opt;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        float scale = 1.f;
        bool wide = true;  // output rows aligned to 16 bytes
        float *stage_out = reinterpret_cast<float *>(
            smem_raw + (smem0 - smem_addr(smem_raw)) + kStages * kStageBytes);
        if (PRODUCT >= kCeGradX) {
            wide = !g.dst || (g.D % (F32 ? 4 : 8) == 0 &&
                              (reinterpret_cast<uintptr_t>(g.dst) & 15) == 0);
            if (g.dst) scale = ce_grad_scale(g.up);
        }
        // A row's upstream gradient over gmax: by a power of two, so that neither
        // a vanishing nor a huge gmax has an infinite or vanishing reciprocal.
        float g_power = 1.f, g_inv = 1.f;
        if (PRODUCT == kCeProbs && g.grow && g.gmax && *g.gmax > 0.f) {
            const float top = *g.gmax;
            g_power = top < 0x1p-64f ? 0x1p64f : top > 0x1p64f ? 0x1p-64f : 1.f;
            g_inv = 1.f / (top * g_power);
        }
        const float unit_scale = PRODUCT == kCeProbs ? g.p_scale / ce_z_scale(g.up) : 1.f;
        // a unit's row, read a unit ahead: units of few classes and channels
        // take no longer than these loads
        auto row_of = [&](int u) {
            RowInfo x{kCeIgnored, make_float2(0.f, 0.f), 1.f};
            if (PRODUCT > kCeProbs || u >= w.units) return x;
            const Unit t = unit_of<PRODUCT, F32>(g, w, u);
            const long long r = (long long)t.m * kCeTileM + rank * 128 + q * 32 + lane;
            if (r >= w.live) return x;
            x.y = g.lab ? g.lab[g.row0 + r] : ce_label(g.labels[g.row0 + r], o.ignore, g.V);
            if (PRODUCT == kCeProbs) {
                x.lse = g.lse[g.row0 + r];
                if (g.grow) x.g = g.grow[g.idx[g.row0 + r]];
            }
            return x;
        };
        RowInfo next = row_of(first);
        for (int u = first; ok && u < w.units; u += step) {
            const Unit t = unit_of<PRODUCT, F32>(g, w, u);
            const long long r = (long long)t.m * kCeTileM + rank * 128 + q * 32 + lane;
            const RowInfo row = next;
            next = row_of(u + step);
            const int y = row.y;
            const float2 lse = row.lse;
            float top = ce_neg_inf(), s = 0.f, sz = 0.f;
            float kz = 1.f, e = 0.f, hit = 0.f;
            if (PRODUCT == kCeProbs) {
                const float f = unit_scale * (row.g * g_power * g_inv);
                kz = (1.f + 2.f * o.zeta * ce_lse(lse)) * f;
                e = o.eps / (float)g.V * f;
                hit = (1.f - o.eps) * f;
            }
            float sum[F32 ? 2 : 1][32];
            for (int i = 0; ok && i < t.steps(); ++i) {
                const int n = t.n0 + i / t.chunks, chunk = i % t.chunks;
                const bool last = chunk == t.chunks - 1;
                const bool empty = t.k0 == t.k1;
                if (!empty) {
                    ok = __all_sync(0xffffffffu, bar_wait(&S.tfull[acc], acc_phase));
                    if (!ok) break;
                    fence_after();
                }
                uint32_t v[32];
#pragma unroll(F32 ? 2 : 1)
                for (int h = 0; h < (F32 ? 2 : 4); ++h) {
                    const int c = 2 * h + half;
                    if (c >= chunks) continue;
                    const int col0 = n * nt + c * 32;  // within the piece
                    if (empty) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = 0;
                    } else {
                        load32(tlane + acc * kCeTileN + c * 32, v);
                        load_wait(v);
                    }
                    if constexpr (F32) {
                        // both accumulators and the chunks of K, in float32
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float a = __uint_as_float(v[j]);
                            sum[h][j] = chunk ? sum[h][j] + a : a;
                        }
                        if (!empty) {
                            load32(tlane + acc * kCeTileN + Sh::kTile + c * 32, v);
                            load_wait(v);
                        }
                        // An infinite operand is infinite in its first plane
                        // and meets the other one's zeros and signs in the
                        // small pairs: there the first pair alone counts.
                        // (Looked for in pairs of columns first: an element's
                        // own test costs 3 % of the derivatives' product.)
                        float2 q = make_float2(0.f, 0.f);
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            q = __ffma2_rn(make_float2(sum[h][j], sum[h][j + 1]),
                                           make_float2(0.f, 0.f), q);
                        if (__all_sync(0xffffffffu, q.x + q.y == 0.f)) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) sum[h][j] += __uint_as_float(v[j]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (isfinite(sum[h][j])) sum[h][j] += __uint_as_float(v[j]);
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(sum[h][j]);
                        if (!last) continue;
                    }
                    if constexpr (PRODUCT == kCeScores) {
                        const int valid = g.nv - col0;
                        float z[32], m = top;
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            z[j] = __uint_as_float(v[j]);
                            if (CAP) z[j] = o.cap * ce_tanh<!F32>(z[j], o.cap);
                        }
                        if (y >= col0 && y < col0 + 32) {
                            float zy = 0.f;
#pragma unroll
                            for (int j = 0; j < 32; ++j) zy = y == col0 + j ? z[j] : zy;
                            g.zt[r] = zy;
                        }
                        if (g.psum) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) sz += j < valid ? z[j] : 0.f;
                        }
                        if (valid < 32) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (j >= valid) z[j] = ce_neg_inf();
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) m = fmaxf(m, z[j]);
                        const float base = CeAcc::base(m);
                        s *= ex2((top - base) * kLog2e);
                        top = m;
                        float s4[4] = {s, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            s4[j & 3] += ex2((z[j] - base) * kLog2e);
                        s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
                    } else if constexpr (PRODUCT == kCeProbs) {
                        if (col0 < g.P.ld) {
                            float d[32];
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                float z = __uint_as_float(v[j]), slope = 1.f;
                                if (CAP) {
                                    const float th = ce_tanh<!F32>(z, o.cap);
                                    z = o.cap * th;
                                    slope = fmaf(-th, th, 1.f);
                                }
                                float x = fmaf(kz, ce_prob(z, lse), -e);
                                if (y == g.v0 + col0 + j) x -= hit;
                                if (CAP) x *= slope;
                                d[j] = y != kCeIgnored && col0 + j < g.nv ? x : 0.f;
                            }
                            for (int p = 0; p < (F32 ? 3 : 1); ++p) {
                                uint32_t out[16];
#pragma unroll
                                for (int j = 0; j < 16; ++j) {
                                    out[j] = pack2(d[2 * j], d[2 * j + 1], F32 || g.bf16);
                                    if (F32) {
                                        d[2 * j] -= __uint_as_float(out[j] << 16);
                                        d[2 * j + 1] -= __uint_as_float(out[j] & 0xffff0000u);
                                    }
                                }
                                char *to = static_cast<char *>(g.p_out) +
                                           2 * (p * g.P.plane + r * g.P.ld + col0);
                                store8(to, out);
                                store8(to + 32, out + 8);
                            }
                        }
                    } else {
                        const long long M = PRODUCT == kCeGradW ? g.nv : w.live;
                        const int cols = min(32, g.D - col0);
                        const bool direct = g.dst != nullptr;
                        const bool add = !direct && g.add;
                        long long to = r;  // row of the output
                        if (direct && PRODUCT == kCeGradX && r < M)
                            to = g.idx ? g.idx[g.row0 + r] : g.row0 + r;
                        if (direct && PRODUCT == kCeGradW) to += g.v0;
                        to *= direct ? g.D : g.acc_ld;
                        // float32 sums, or float32 gradients; 16-bit gradients
                        float *out32 = F32 && direct ? static_cast<float *>(g.dst)
                                                     : g.acc + t.split * g.acc_split;
                        uint16_t *out16 = static_cast<uint16_t *>(g.dst);
                        if (wide) {
                            if (r < M && !F32 && direct) {
#pragma unroll
                                for (int j = 0; j < 32; j += 8) {
                                    if (j >= cols) continue;
                                    uint32_t out[4];
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        out[i] = pack2(__uint_as_float(v[j + 2 * i]) * scale,
                                                       __uint_as_float(v[j + 2 * i + 1]) * scale,
                                                       g.bf16);
                                    store4(out16 + to + col0 + j, out);
                                }
                            } else if (r < M) {
                                float4 *p = reinterpret_cast<float4 *>(out32 + to + col0);
                                // all reads before the first write: one latency
                                float4 old[8];
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    old[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                                    if (add && 4 * j < cols) old[j] = p[j];
                                }
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    if (4 * j >= cols) continue;
                                    p[j] = make_float4(
                                        fmaf(__uint_as_float(v[4 * j]), scale, old[j].x),
                                        fmaf(__uint_as_float(v[4 * j + 1]), scale, old[j].y),
                                        fmaf(__uint_as_float(v[4 * j + 2]), scale, old[j].z),
                                        fmaf(__uint_as_float(v[4 * j + 3]), scale, old[j].w));
                                }
                            }
                        } else if (cols > 0) {
                            // gradients of no alignment: the warp turns its 32
                            // x 32 and writes row by row
                            float *turn = stage_out + (warp - 4) * Sh::kTurn * 33;
                            const int n_rows = (int)max(0LL, min(32LL, M - (r - lane)));
#pragma unroll 1
                            for (int i0 = 0; i0 < n_rows; i0 += Sh::kTurn) {
                                if (lane / Sh::kTurn == i0 / Sh::kTurn) {
#pragma unroll
                                    for (int j = 0; j < 32; ++j)
                                        turn[lane % Sh::kTurn * 33 + j] =
                                            __uint_as_float(v[j]) * scale;
                                }
                                __syncwarp();
                                // eight rows together: one latency
                                for (int i = i0; i < min(n_rows, i0 + Sh::kTurn); i += 8) {
                                    float x[8];
#pragma unroll
                                    for (int k = 0; k < 8; ++k)
                                        x[k] = turn[(i - i0 + k) * 33 + lane];
#pragma unroll
                                    for (int k = 0; k < 8; ++k) {
                                        const long long at =
                                            __shfl_sync(0xffffffffu, to, i + k) + col0 + lane;
                                        if (lane >= cols || i + k >= n_rows) continue;
                                        if (F32)
                                            out32[at] = x[k];
                                        else
                                            out16[at] = (uint16_t)pack2(x[k], 0.f, g.bf16);
                                    }
                                }
                                __syncwarp();
                            }
                        }
                    }
                }
                if (!empty) {
                    // this warp has read its part of the accumulator
                    fence_before();
                    if (lane == 0)
                        asm volatile(
                            "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                in_leader(smem_addr(&S.tempty[acc])))
                            : "memory");
                    __syncwarp();
                    if (++acc == 2) {
                        acc = 0;
                        acc_phase ^= 1;
                    }
                }
            }
            if (PRODUCT == kCeScores && r < w.live) {
                const long long at = (2LL * t.split + half) * g.rows + r;
                g.part[at] = make_float2(top, s);
                if (g.psum) g.psum[at] = sz;
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    cluster_sync();
    fence_after();
    if (warp == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(kCols));
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                              const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult st;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000,
                                             cudaEnableDefault, &st) != cudaSuccess ||
            st != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// boxes of 64 columns x box_rows rows of one plane, 128-byte swizzle, zeros
// outside the matrix
bool make_map(CUtensorMap *map, const CeMat &m, int planes, bool bf16, int box_rows) {
    const EncodeFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t plane = planes > 1 ? (cuuint64_t)m.plane : (cuuint64_t)m.ld * m.rows;
    const cuuint64_t dims[3] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)m.ld * 2, plane * 2};
    const cuuint32_t box[3] = {kDepth, (cuuint32_t)box_rows, 1}, one[3] = {1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
              const_cast<void *>(m.ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Classes of a tile of scores: the width, in steps of 32, with which the pairs
// are done first. A tile costs its width, below 64 no less (A's rows are read
// all the same), and about 32 to turn around: 256 where there is much to do,
// 160 for 1001 rows x 5003 classes (2 rounds instead of 2 wider ones), 64 for
// 18 rows x 3021 (48 tiles instead of 24 at the same memory). float32: 128
// at most, as for the gradients.
int score_tile(long long rows, int nv, bool f32) {
    const long long mt = (rows + kCeTileM - 1) / kCeTileM;
    int best = 32;
    long long cost = LLONG_MAX;
    for (int nt = 32; nt <= (f32 ? 128 : kCeTileN); nt += 32) {
        const long long units = mt * ((nv + nt - 1) / nt);
        const long long c = (units + kCePairs - 1) / kCePairs * (std::max(nt, 64) + 32);
        if (c <= cost) {
            cost = c;
            best = nt;
        }
        if (nt >= nv) break;
    }
    return best;
}

template <int PRODUCT, bool CAP, bool F32>
cudaError_t launch(const CeGemm &g, cudaStream_t st) {
    constexpr bool kAMn = PRODUCT == kCeGradW, kBMn = PRODUCT >= kCeGradX;
    const int nt = kBMn ? ce_grad_tile(g.D, F32) : score_tile(g.rows, g.nv, F32);
    // The driver encodes tensor maps only where a context is current, and this
    // may be the calling thread's first work (autograd's): setting the device
    // makes its context current.
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err == cudaSuccess) err = cudaSetDevice(dev);
    if (err != cudaSuccess) return err;
    CUtensorMap a, b;
    const CeMat &ma = PRODUCT >= kCeGradX ? g.P : g.X;
    const CeMat &mb = PRODUCT == kCeGradW ? g.X : g.W;
    if (!make_map(&a, ma, g.planes, g.bf16, kAMn ? 64 : 128) ||
        !make_map(&b, mb, g.planes, g.bf16, kBMn ? 64 : nt / 2))
        return cudaErrorInvalidValue;
    auto kernel = ce_gemm_kernel<PRODUCT, CAP, F32>;
    // once a device (a repeated call is harmless)
    static std::atomic<unsigned long long> ready{0};
    if (!(ready.load() >> (dev & 63) & 1)) {
        err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   Shape<F32>::kSmemBytes);
        if (err != cudaSuccess) return err;
        ready.fetch_or(1ull << (dev & 63));
    }
    const long long M = PRODUCT == kCeGradW ? g.nv : g.rows;
    const long long mt = (M + kCeTileM - 1) / kCeTileM;
    const long long n = (PRODUCT <= kCeProbs ? g.nv : g.D);
    const long long units =
        mt * (PRODUCT == kCeScores ? g.runs : (n + nt - 1) / nt * g.splits);
    const int grid = 2 * (int)std::min<long long>(kCePairs, units);
    kernel<<<grid, kThreads, Shape<F32>::kSmemBytes, st>>>(a, b, g, nt);
    count_launches(1);
    return cudaGetLastError();
}

}  // namespace

// Columns of a gradient's tile (MN-major B: multiples of 128). float32 keeps
// a tile's sums in registers, 64 a thread: 128 at most. (256 wide, summed in
// memory a chunk at a time, the two gradients of 42765 x 26421 x 621 took 36
// ms, with the planes loaded once a stage 14.)
int ce_grad_tile(int cols, bool f32) { return f32 || cols <= 128 ? 128 : kCeTileN; }

int ce_runs(long long rows, int V, bool f32) {
    // (rows below 2^31: 2^23 tiles, 2^31 units at most)
    const unsigned mt = (unsigned)((rows + kCeTileM - 1) / kCeTileM);
    const int nt = score_tile(rows, V, f32);
    const unsigned tiles = (unsigned)((V + nt - 1) / nt);
    // the longest pair's tiles, and about a third of a tile to begin a run
    int best = 1;
    double cost = 1e300;
    for (unsigned r = 1; r <= std::min(tiles, 2u * kCePairs); ++r) {
        const double c = (double)((mt * r + kCePairs - 1) / kCePairs) *
                         ((tiles + r - 1) / r + 0.33);
        if (c < cost - 1e-9) {
            cost = c;
            best = r;
        }
    }
    return best;
}

int ce_error_flag(bool clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_ce_error, sizeof(v)) != cudaSuccess) return -1;
    if (clear && v) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_ce_error, &zero, sizeof(zero));
    }
    return v;
}

cudaError_t launch_ce_gemm(const CeGemm &g, cudaStream_t st) {
    const bool cap = g.opt.cap > 0.f, f32 = g.planes == 3;
    switch (g.product) {
        case kCeScores:
            if (f32)
                return cap ? launch<kCeScores, true, true>(g, st)
                           : launch<kCeScores, false, true>(g, st);
            return cap ? launch<kCeScores, true, false>(g, st)
                       : launch<kCeScores, false, false>(g, st);
        case kCeProbs:
            if (f32)
                return cap ? launch<kCeProbs, true, true>(g, st)
                           : launch<kCeProbs, false, true>(g, st);
            return cap ? launch<kCeProbs, true, false>(g, st)
                       : launch<kCeProbs, false, false>(g, st);
        case kCeGradX:
            return f32 ? launch<kCeGradX, false, true>(g, st)
                       : launch<kCeGradX, false, false>(g, st);
        default:
            return f32 ? launch<kCeGradW, false, true>(g, st)
                       : launch<kCeGradW, false, false>(g, st);
    }
}

}  // namespace gsv
