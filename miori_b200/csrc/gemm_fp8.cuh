// Products in 8-bit floating point: C[m][n] = sum_b sa[m][b] sw[n / 128][b] sum_{k in block b} a[m][k] w[n][k], a and w e4m3 with
// K contiguous, blocks of 128 along K (a: one row, w: 128 rows), sums in fp32.
//
// The tensor core adds up one block (four tcgen05.mma of kind::f8f6f4, 32 elements each); the scales differ from block to block,
// so what it has summed leaves tensor memory once a block and is added, times the block's scale, to fp32
// accumulators in registers.  That is one tcgen05.ld and half a packed FMA (fma.rn.f32x2) an element and block: of the 512 cycles that the
// matrix unit takes for a 128 x 256 x 128 block, 256 of the tensor memory's reading and 128 to 256 of issue, beside it.  Two
// or four blocks' sums fit tensor memory, so that the unit works on some while others are read.  It waits for the readers all the same: half of
// its cycles are busy in the largest products, and those take a fifth less time without the additions.
// (Scales that are powers of two could ride along inside the MMA; a checkpoint's are any fp32.)
//
// Two kernels:
//   pair   more than a hundred rows or so: 256 x 256 or 256 x 128 tiles on SM pairs (cta_group::2), persistent; each CTA pulls 32 KB a
//          block through L2 for 512 cycles of its matrix unit, and takes some 800 for them.  16384 x 16384 x 2048: 557 us in a burst, 1.97 PFLOP/s
//          (633 under the power limit, which holds the clock at 1.58 GHz in the one and 1.39 in the other); 1024 x 2048 x 8192: 23 us.
//   swap   few rows, or few tiles: 128 rows of w are the MMA's M, up to 128 rows of a its N; K is split over the CTAs of a
//          cluster and the partial sums meet in distributed shared memory, in rank order.  8 x 16384 x 2048: 7.2 us, 4.7 TB/s; one row of 2048 x 2048: 3.4 us
//          in a chain; 64 x 16384 x 2048: 10.2 us.  A slice's scales lie in shared memory, which has room for K of 16384; beyond that few rows go through
//          tiles of 256 too (1 x 8192 x 16384 27 us, x 28672 100; 8 rows 72).
// Ends of M, N and K are zeros by TMA; what lies behind N in a row of C is left as it was.  Every wait is bounded.
#pragma once
#include "common.cuh"
#include "tma_host.cuh"

namespace miori_b200 {
namespace fp8 {

constexpr int KB_BYTES = 128;               // a k-block of a row: one row of the 128-byte swizzle
constexpr int UMMA_KB = 32;                 // bytes of K an MMA takes
constexpr uint32_t PEER_MASK = 0xFEFFFFFFu;  // clears the CTA-rank bit of a shared::cluster address

struct GemmArgs {
    void* c;
    const float *sa, *sw;
    int64_t ldc, sa_row, sa_col, sw_row, sw_col;  // elements
    uint32_t M, N, K;
    uint32_t bf16;
    uint32_t by_tma;  // C's rows begin and end on 16-byte boundaries: stored by TMA, or by words
};

// K-major, 128-byte swizzle: rows of 128 bytes, eight of them an atom of 1024 bytes.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// D fp32, A and B e4m3, both K-major, shape m x n.
__host__ __device__ constexpr uint32_t idesc_e4m3(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }

template <int CTAS>
__device__ __forceinline__ void umma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CTAS == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit_one(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// the same barrier offset in both CTAs of the pair
__device__ __forceinline__ void commit_both(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// Hands over tensor memory and nothing else: behind fence_before, and waited for with Order TENSOR in front of fence_after.
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, 0;\n\tmbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [ra];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void load_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr));
}
// The registers pass through the wait, so that nothing that reads them can be moved in front of it.
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
          "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]) :: "memory");
    asm volatile("" : "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
// mbar_wait by a whole warp, with one answer for it.  (By one lane, that tells the others: 100 cycles more a wait.)
template <Order O = Order::OWN>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t where) {
    if (__all_sync(0xFFFFFFFFu, mbar_try<O>(bar, parity))) return true;
    return __all_sync(0xFFFFFFFFu, mbar_wait<false, O>(bar, parity, abort, where));
}
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0u;
}
// A value that all lanes hold, for the compiler to know that they do.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xFFFFFFFFu, x, 0); }
// (acc.x + v.x s, acc.y + v.y s)
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t v, uint64_t s) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(v), "l"(s)); }

// ---- 256-row tiles on SM pairs ----------------------------------------------------------------------------

// BN: columns of a tile, 256 or 128; it is worked on in halves of 128, the columns of a block of w, so that four of a half's sums fit tensor
// memory and a half is read while the unit works on the next.
template <int BN>
struct PairCfg {
    static constexpr int HALVES = BN / 128;
    static constexpr int A_BYTES = 128 * KB_BYTES, HALF_BYTES = 64 * KB_BYTES, STAGE_BYTES = A_BYTES + HALVES * HALF_BYTES;  // a CTA's: 128 rows of a, 64 of each half of w
    static constexpr int STAGES = BN == 256 ? 5 : 6;
    static constexpr int BUFS = 4;
    static constexpr int OUT_BYTES = 8 * 2 * 32 * 128;  // two buffers of 32 rows x 128 bytes an epilogue warp
    static constexpr int SMEM = STAGES * STAGE_BYTES + OUT_BYTES + 1024 + 256;
};
// A warpgroup that copies and issues and two that read: at 168 registers a thread when launched, 24 and 240 then (128 x 24 + 256 x 240 = 384 x 168).  Sixteen
// reading warps of 112 registers had to wait for each other's sums and spilled (16384 x 16384 x 2048: 749 us).
constexpr int PAIR_THREADS = 384;
constexpr uint32_t GROUP_TILES = 8;  // row tiles that share what L2 holds of w

struct Tile {
    uint32_t m, n;
};
__device__ __forceinline__ Tile tile_at(uint32_t t, uint32_t m_tiles, uint32_t n_tiles) {
    const uint32_t per_group = GROUP_TILES * n_tiles, group = t / per_group, first = group * GROUP_TILES;
    const uint32_t gm = min(GROUP_TILES, m_tiles - first), r = t - group * per_group;
    return {first + r % gm, r / gm};
}

template <int BN>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_c,
                     const GemmArgs g) {
    using C = PairCfg<BN>;
    constexpr int STAGES = C::STAGES, STAGE_BYTES = C::STAGE_BYTES, BUFS = C::BUFS, HALVES = C::HALVES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t abort_flag;
    const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u, out_stage = ring + STAGES * STAGE_BYTES, bars = out_stage + C::OUT_BYTES;
    auto full = [&](uint32_t s) { return bars + 8u * s; };
    auto empty = [&](uint32_t s) { return bars + 8u * (STAGES + s); };
    auto summed = [&](uint32_t b) { return bars + 8u * (2 * STAGES + b); };
    auto taken = [&](uint32_t b) { return bars + 8u * (2 * STAGES + BUFS + b); };

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t m_tiles = (g.M + 255u) / 256u, n_tiles = (g.N + BN - 1u) / BN, tiles = m_tiles * n_tiles;
    const uint32_t k_blocks = (g.K + KB_BYTES - 1u) / KB_BYTES;

    if (threadIdx.x == 0) {
        abort_flag = 0u;
        for (int s = 0; s < STAGES; ++s) mbar_init(full(s), 1), mbar_init(empty(s), HALVES);
        for (int b = 0; b < BUFS; ++b) mbar_init(summed(b), 1), mbar_init(taken(b), rank == 0u ? 9 : 8);  // eight epilogue warps; the leader's: and the other CTA's word for its own
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_c) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        pdl_launch_dependents();  // with its columns in hand
    }
    fence_before();
    __syncthreads();
    cluster_barrier();  // both CTAs' barriers exist before anything arrives from the other
    fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait_prior();

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
        if (warp == 0 && lane == 0) {
            uint32_t s = 0, parity = 1u;
            bool ok = true;
            for (uint32_t t = pair; t < tiles && ok; t += pairs) {
                const Tile tc = tile_at(t, m_tiles, n_tiles);
                const int m = (int)(tc.m * 256u + rank * 128u), n = (int)(tc.n * BN + rank * 64u);
                for (uint32_t kb = 0; kb < k_blocks; ++kb) {
                    if (!(ok = mbar_wait(empty(s), parity, &abort_flag, 0x71))) break;
                    const uint32_t at = ring + s * STAGE_BYTES, bar = full(s) & PEER_MASK;
                    if (rank == 0) mbar_expect_tx(full(s), 2u * STAGE_BYTES);
                    load_pair(at, &map_a, (int)(kb * KB_BYTES), m, bar);
#pragma unroll
                    for (int h = 0; h < HALVES; ++h) load_pair(at + C::A_BYTES + h * C::HALF_BYTES, &map_w, (int)(kb * KB_BYTES), n + h * 128, bar);
                    if (++s == STAGES) s = 0u, parity ^= 1u;
                }
            }
        } else if (warp >= 1 && warp <= HALVES && rank != 0) {
            // one arrival from CTA to CTA a half: eight of them, each of which waits for what its thread wrote before, took longer than the MMAs
            if (lane == 0) {
                uint32_t b = warp - 1u, b_parity = 0u;
                bool ok = true;
                for (uint32_t t = pair; t < tiles && ok; t += pairs)
                    for (uint32_t i = 0; i < k_blocks; ++i) {
                        if (!(ok = mbar_wait(taken(b), b_parity, &abort_flag, 0x79))) break;
                        fence_after();
                        fence_before();
                        arrive_leader(taken(b));
                        if ((b += HALVES) >= BUFS) b -= BUFS, b_parity ^= 1u;
                    }
            }
        } else if (warp >= 1 && warp <= HALVES) {
            // A warp for each half.  The whole warp walks the loop and one elected thread issues: descriptors and addresses stay in uniform
            // registers (a k-block's eight MMAs, three waits and three commits by one thread: 1300 cycles, by one warp so 800).
            constexpr uint32_t idesc = idesc_e4m3(256, 128);
            const uint32_t tm = uniform(tmem), half = uniform(warp - 1u);
            const uint64_t first = desc_sw128(uniform(ring));
            uint32_t s = 0, parity = 0u, b = half, b_parity = 1u;
            bool ok = true;
            for (uint32_t t = pair; t < tiles && ok; t += pairs) {
                for (uint32_t kb = 0; kb < k_blocks; ++kb) {
                    if (!(ok = warp_wait<Order::TENSOR>(taken(b), b_parity, &abort_flag, 0x72))) break;
                    if (!(ok = warp_wait(full(s), parity, &abort_flag, 0x73))) break;
                    fence_after();
                    if (elect_one()) {
                        const uint64_t ad = first + s * (STAGE_BYTES / 16u), wd = ad + (C::A_BYTES + half * C::HALF_BYTES) / 16u;
#pragma unroll
                        for (uint32_t k = 0; k < KB_BYTES / UMMA_KB; ++k) umma_e4m3<2>(tm + b * 128u, ad + 2u * k, wd + 2u * k, idesc, k != 0u);
                        commit_both(summed(b));
                        commit_both(empty(s));
                    }
                    __syncwarp();
                    if ((b += HALVES) >= BUFS) b -= BUFS, b_parity ^= 1u;
                    if (++s == STAGES) s = 0u, parity ^= 1u;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 240;");
        const uint32_t quad = warp & 3u, part = (warp - 4u) >> 2;  // TMEM lanes of this warp, and which 64 columns of a half
        const uint32_t bufs = out_stage + (warp - 4u) * 8192u, sw_lane = lane & 7u;
        uint32_t b = 0, b_parity = 0u, fills = 0;
        bool ok = true;
        for (uint32_t t = pair; t < tiles && ok; t += pairs) {
            const Tile tc = tile_at(t, m_tiles, n_tiles);
            const uint32_t row0 = tc.m * 256u + rank * 128u + quad * 32u;
            // scales two k-blocks ahead
            const float* sa = g.sa + (int64_t)min(row0 + lane, g.M - 1u) * g.sa_row;
            const float* sw = g.sw + (int64_t)(tc.n * HALVES) * g.sw_row;
            const int64_t next_half = HALVES == 2 && tc.n * BN + 128u < g.N ? g.sw_row : 0;  // a half behind N has no scale
            float x[2], y[2][HALVES];
            auto scales = [&](int to) {
                x[to] = ld_fresh(sa), y[to][0] = ld_fresh(sw);
                if (HALVES == 2) y[to][HALVES - 1] = ld_fresh(sw + next_half);
                sa += g.sa_col, sw += g.sw_col;
            };
            scales(0);
            if (k_blocks > 1u) scales(1);
            uint64_t acc[HALVES][32];
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[h][i] = 0ull;
            // A step is a half of a k-block; the next one's sums are on their way while this one's are added.
            const uint32_t from = tmem + ((quad * 32u) << 16) + part * 64u;
            uint32_t r[2][32];
            if (!(ok = warp_wait(summed(b), b_parity, &abort_flag, 0x74))) break;
            fence_after();
            tmem_ld32(from + b * 128u, r[0]);
            tmem_ld32(from + b * 128u + 32u, r[1]);
            auto block = [&](int at, uint32_t kb) {
                float scale[HALVES];
#pragma unroll
                for (int h = 0; h < HALVES; ++h) scale[h] = __fmul_rn(x[at], y[at][h]);
                if (kb + 2u < k_blocks) scales(at);
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    tmem_wait32(r[0]);
                    tmem_wait32(r[1]);
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(taken(b));  // before the sums are used
                    if (++b == BUFS) b = 0u, b_parity ^= 1u;
                    const bool more = h + 1 < HALVES || kb + 1u < k_blocks;
                    const bool there = mbar_test(summed(b), b_parity);  // asked for now, looked at when these sums have been added: an answer takes 100 cycles
                    const uint64_t s2 = pack2(__float_as_uint(scale[h]), __float_as_uint(scale[h]));
#pragma unroll
                    for (int j = 0; j < 16; ++j) fma2(acc[h][j], pack2(r[0][2 * j], r[0][2 * j + 1]), s2);
                    if (more) {
                        if (!__all_sync(0xFFFFFFFFu, there)) ok = warp_wait(summed(b), b_parity, &abort_flag, 0x74);
                        if (!ok) return;
                        fence_after();
                        tmem_ld32(from + b * 128u, r[0]);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) fma2(acc[h][16 + j], pack2(r[1][2 * j], r[1][2 * j + 1]), s2);
                    if (more) tmem_ld32(from + b * 128u + 32u, r[1]);
                }
            };
            for (uint32_t kb = 0; kb < k_blocks && ok; kb += 2u) {
                block(0, kb);
                if (ok && kb + 1u < k_blocks) block(1, kb + 1u);
            }
            if (!ok) break;
            // 32 rows x 128 bytes at a time through shared memory, in the 128-byte swizzle
            if (row0 >= g.M) continue;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                const uint32_t col0 = tc.n * BN + h * 128u + part * 64u;
                auto word = [&](int i) { return (uint32_t)(i & 1 ? acc[h][i >> 1] >> 32 : acc[h][i >> 1]); };
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    if (g.bf16 && f > 0) break;  // 64 columns are 128 bytes
                    if (col0 + f * 32u >= g.N) break;
                    const uint32_t buf = bufs + (fills++ & 1u) * 4096u, rowp = buf + lane * 128u;
                    if (lane == 0) tma_store_wait_read<1>();  // the store issued two buffers ago has read this one
                    __syncwarp();
                    if (g.bf16) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            uint32_t v[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = pack_bf16(__uint_as_float(word(j * 8 + e * 2)), __uint_as_float(word(j * 8 + e * 2 + 1)));
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                                         ::"r"(rowp + (((uint32_t)j ^ sw_lane) << 4)), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                                         ::"r"(rowp + (((uint32_t)j ^ sw_lane) << 4)), "r"(word(f * 32 + j * 4)), "r"(word(f * 32 + j * 4 + 1)),
                                           "r"(word(f * 32 + j * 4 + 2)), "r"(word(f * 32 + j * 4 + 3)) : "memory");
                    }
                    if (g.by_tma) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_3d(&map_c, (int)(col0 + f * 32u), (int)row0, 0, buf);
                            tma_store_commit();
                        }
                    } else {
                        __syncwarp();
                        const uint32_t rows = min(32u, g.M - row0), col = col0 + f * 32u + lane * (g.bf16 ? 2u : 1u);
                        for (uint32_t r = 0; r < rows; ++r) {
                            uint32_t w;
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(buf + r * 128u + (((lane >> 2) ^ (r & 7u)) << 4) + (lane & 3u) * 4u) : "memory");
                            const int64_t at = (int64_t)(row0 + r) * g.ldc + col;
                            if (g.bf16) {
                                if (col < g.N) static_cast<uint16_t*>(g.c)[at] = (uint16_t)w;
                                if (col + 1u < g.N) static_cast<uint16_t*>(g.c)[at + 1] = (uint16_t)(w >> 16);
                            } else if (col < g.N) {
                                static_cast<uint32_t*>(g.c)[at] = w;
                            }
                        }
                        __syncwarp();
                    }
                }
            }
        }
        if (lane == 0) tma_store_wait_read<0>();  // shared memory is read; the writes are the grid's to complete
    }

    // teardown: on abort give in-flight copies and MMAs time to land before freeing TMEM
    __syncwarp();
    if (abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) __nanosleep(1000);
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    cluster_barrier();  // the other CTA may still signal this one's barriers or read its shared memory
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---- few rows: w's rows as the MMA's M, K over a cluster ------------------------------------------------------

constexpr int SWAP_THREADS = 224;  // a copying, two MMA and four epilogue warps
constexpr int SWAP_MAX_STAGES = 8;
__host__ __device__ constexpr int SWAP_BUFS(int mp) { return mp >= 128 ? 2 : 4; }  // at most 256 columns: two CTAs an SM fit

struct SwapGeo {
    uint32_t cs, stages, m_tiles;
};

// MP: columns of the MMA, rows of a padded to 16, 32, 64 or 128
template <int MP>
__global__ void __launch_bounds__(SWAP_THREADS)
gemm_fp8_swap_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const GemmArgs g, const SwapGeo geo) {
    constexpr int W_BYTES = 128 * KB_BYTES, A_BYTES = MP * KB_BYTES, STAGE_BYTES = W_BYTES + A_BYTES, BUFS = SWAP_BUFS(MP);
    constexpr uint32_t TMEM_COLS = BUFS * MP < 32 ? 32 : BUFS * MP;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars_mem[2 * SWAP_MAX_STAGES + 2 * BUFS];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t abort_flag;
    const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u, bars = smem_addr(bars_mem);
    auto full = [&](uint32_t s) { return bars + 8u * s; };
    auto empty = [&](uint32_t s) { return bars + 8u * (SWAP_MAX_STAGES + s); };
    auto summed = [&](uint32_t b) { return bars + 8u * (2 * SWAP_MAX_STAGES + b); };
    auto taken = [&](uint32_t b) { return bars + 8u * (2 * SWAP_MAX_STAGES + BUFS + b); };
    const uint32_t scales = ring + geo.stages * STAGE_BYTES;  // [k-block of the slice][MP]

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t rank = blockIdx.x % geo.cs, tile = blockIdx.x / geo.cs, m_tile = tile % geo.m_tiles, n_tile = tile / geo.m_tiles;
    const uint32_t m0 = m_tile * MP;
    const uint32_t k_blocks = (g.K + KB_BYTES - 1u) / KB_BYTES;
    const uint32_t kb0 = rank * k_blocks / geo.cs, nkb = (rank + 1u) * k_blocks / geo.cs - kb0;

    if (threadIdx.x == 0) {
        abort_flag = 0u;
        for (uint32_t s = 0; s < geo.stages; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
        for (uint32_t b = 0; b < (uint32_t)BUFS; ++b) mbar_init(summed(b), 1), mbar_init(taken(b), 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        pdl_launch_dependents();  // with its columns in hand
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait_prior();

    bool ok = true;
    float acc[MP];
    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, parity = 1u;
            for (uint32_t i = 0; i < nkb; ++i) {
                if (!(ok = mbar_wait(empty(s), parity, &abort_flag, 0x75))) break;
                mbar_expect_tx(full(s), STAGE_BYTES);
                const uint32_t at = ring + s * STAGE_BYTES;
                tma_load_2d(at, &map_w, (int)((kb0 + i) * KB_BYTES), (int)(n_tile * 128u), full(s));
                tma_load_2d(at + W_BYTES, &map_a, (int)((kb0 + i) * KB_BYTES), (int)m0, full(s));
                if (++s == geo.stages) s = 0u, parity ^= 1u;
            }
        }
    } else if (warp < 3) {
        // Two warps take the k-blocks in turns: a block's waits, MMAs and commits are 500 cycles of one of them, more than its bytes take.
        constexpr uint32_t idesc = idesc_e4m3(128, MP);
        const uint32_t tm = uniform(tmem), turn = uniform(warp - 1u);
        const uint64_t first = desc_sw128(uniform(ring));
        uint32_t s = turn % geo.stages, parity = turn / geo.stages & 1u, b = turn, b_parity = 1u;
        for (uint32_t i = turn; i < nkb; i += 2u) {
            if (!(ok = warp_wait(taken(b), b_parity, &abort_flag, 0x76))) break;
            if (!(ok = warp_wait(full(s), parity, &abort_flag, 0x77))) break;
            fence_after();
            if (elect_one()) {
                const uint64_t wd = first + s * (STAGE_BYTES / 16u), ad = wd + W_BYTES / 16u;
#pragma unroll
                for (uint32_t k = 0; k < KB_BYTES / UMMA_KB; ++k) umma_e4m3<1>(tm + b * MP, wd + 2u * k, ad + 2u * k, idesc, k != 0u);
                commit_one(summed(b));
                commit_one(empty(s));
            }
            __syncwarp();
            for (uint32_t n = 0; n < 2u; ++n)
                if (++s == geo.stages) s = 0u, parity ^= 1u;
            b ^= 2u % BUFS;
            if (BUFS == 2 || b < 2u) b_parity ^= 1u;
        }
    } else {
        // the slice's scales, multiplied out: no row's weight is read twice
        const float* sw = g.sw + (int64_t)n_tile * g.sw_row + (int64_t)kb0 * g.sw_col;
        for (uint32_t i = threadIdx.x - 96u; i < nkb * MP; i += 128u) {
            const uint32_t kb = i / MP, m = m0 + i % MP;
            float v = 0.0f;
            if (m < g.M) v = __fmul_rn(ld_fresh(g.sa + (int64_t)m * g.sa_row + (int64_t)(kb0 + kb) * g.sa_col), ld_fresh(sw + (int64_t)kb * g.sw_col));
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(scales + i * 4u), "f"(v) : "memory");
        }
        __syncwarp();
        asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
        for (int j = 0; j < MP; ++j) acc[j] = 0.0f;
        uint32_t b = 0, b_parity = 0u;
        for (uint32_t i = 0; i < nkb; ++i) {
            ok = warp_wait(summed(b), b_parity, &abort_flag, 0x78);
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int c = 0; c < MP; c += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + (((warp & 3u) * 32u) << 16) + b * MP + c, r);
                tmem_wait16(r);
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    float4 s;
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(s.x), "=f"(s.y), "=f"(s.z), "=f"(s.w) : "r"(scales + (i * MP + c + j) * 4u) : "memory");
                    acc[c + j] = __fmaf_rn(__uint_as_float(r[j]), s.x, acc[c + j]);
                    acc[c + j + 1] = __fmaf_rn(__uint_as_float(r[j + 1]), s.y, acc[c + j + 1]);
                    acc[c + j + 2] = __fmaf_rn(__uint_as_float(r[j + 2]), s.z, acc[c + j + 2]);
                    acc[c + j + 3] = __fmaf_rn(__uint_as_float(r[j + 3]), s.w, acc[c + j + 3]);
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(taken(b));
            if (++b == (uint32_t)BUFS) b = 0u, b_parity ^= 1u;
        }
    }
    __syncwarp();

    // The sums go to shared memory, [row of a][row of w]: all MMAs are done and, after a barrier of their readers, the scales are read.  From there
    // CTA r of the cluster takes rows r, r + cs, ... of a, each by a warp, and adds them up in rank order.  (Stored by the threads that hold them
    // a row was 160 cycles: its instructions, which nothing had run before, took that long to come.)
    // Tensor memory is free before other CTAs are waited for: one of the cluster may still wait for columns that somebody holds who waits in turn.
    bool freed = false;
    if (warp == 1u) {
        asm volatile("bar.sync 2, 160;" ::: "memory");  // its readers
        freed = __all_sync(0xFFFFFFFFu, abort_flag == 0u);
        if (freed) {
            fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
        }
    }
    if (warp >= 3u) {
        fence_before();
        asm volatile("bar.arrive 2, 160;" ::: "memory");
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const uint32_t to = ring + ((warp & 3u) * 32u + lane) * 4u;
#pragma unroll
        for (int j = 0; j < MP; ++j) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + j * 512u), "f"(acc[j]) : "memory");
    }
    if (geo.cs > 1u) cluster_barrier();
    else __syncthreads();
    const uint32_t rows = min((uint32_t)MP, g.M - m0), n = n_tile * 128u + lane * 4u;
#pragma unroll 1
    for (uint32_t m = rank + geo.cs * warp; m < rows && !abort_flag; m += geo.cs * (SWAP_THREADS / 32u)) {
        const uint32_t from = ring + m * 512u + lane * 16u;
        float4 v[8];
#pragma unroll
        for (uint32_t p = 0; p < 8u; ++p) {
            if (p >= geo.cs) break;
            uint32_t at;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(from), "r"(p));
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[p].x), "=f"(v[p].y), "=f"(v[p].z), "=f"(v[p].w) : "r"(at) : "memory");
        }
        float4 t = v[0];
#pragma unroll
        for (uint32_t p = 1; p < 8u; ++p) {
            if (p >= geo.cs) break;
            t.x += v[p].x, t.y += v[p].y, t.z += v[p].z, t.w += v[p].w;
        }
        const int64_t at = (int64_t)(m0 + m) * g.ldc + n;
        if (g.by_tma) {  // rows begin and end on 16-byte boundaries: four columns are all there or none is
            if (n >= g.N) continue;
            if (g.bf16) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(g.c) + at) = make_uint2(pack_bf16(t.x, t.y), pack_bf16(t.z, t.w));
            else *reinterpret_cast<float4*>(static_cast<float*>(g.c) + at) = t;
        } else {
            const float e[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                if (n + i >= g.N) break;
                if (g.bf16) static_cast<uint16_t*>(g.c)[at + i] = (uint16_t)pack_bf16(e[i], 0.0f);
                else static_cast<float*>(g.c)[at + i] = e[i];
            }
        }
    }
    __syncwarp();  // lanes leave the stores at different times, and the barrier is one of whole warps
    if (geo.cs > 1u) cluster_barrier();  // nobody leaves while its sums are read

    if (abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) __nanosleep(1000);
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 1 && !freed) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// ---- launches -------------------------------------------------------------------------------------------------

struct GemmOperands {
    const void *a, *w;
    int64_t lda, ldw;
};
inline int bytes_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t K, uint32_t box_rows, int64_t pitch) {
    return make_tmap_2d(map, base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, rows, KB_BYTES, box_rows, CU_TENSOR_MAP_SWIZZLE_128B, (uint64_t)pitch);
}

template <int BN>
inline int launch_pair(const GemmOperands& o, GemmArgs g, cudaStream_t stream) {
    CUtensorMap ma, mw, mc;
    if (const int rc = bytes_map(&ma, o.a, g.M, g.K, 128, o.lda)) return rc;
    if (const int rc = bytes_map(&mw, o.w, g.N, g.K, 64, o.ldw)) return rc;
    mc = ma;  // unused where C is stored otherwise
    if (g.by_tma) {
        const int rc = g.bf16 ? make_tmap_3d(&mc, g.c, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, g.N, g.M, 1, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B, (uint64_t)g.ldc)
                              : make_tmap_3d(&mc, g.c, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, g.N, g.M, 1, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B, (uint64_t)g.ldc);
        if (rc) return rc;
    }
    const uint64_t tiles = (uint64_t)((g.M + 255u) / 256u) * ((g.N + BN - 1u) / BN);
    const uint32_t pairs = (uint32_t)(tiles < (uint64_t)(sm_count() / 2) ? tiles : (uint64_t)(sm_count() / 2));
    const cudaError_t e = launch_cluster(gemm_fp8_pair_kernel<BN>, 2u * pairs, PAIR_THREADS, PairCfg<BN>::SMEM, 2, stream, ma, mw, mc, g);
    return e == cudaSuccess ? MIORI_OK : cuda_fail(e, "gemm_fp8 (pair) launch");
}

template <int MP>
inline int launch_swap(const GemmOperands& o, const GemmArgs& g, uint32_t cs, cudaStream_t stream) {
    constexpr uint32_t STAGE_BYTES = (128 + MP) * KB_BYTES;
    CUtensorMap ma, mw;
    if (const int rc = bytes_map(&mw, o.w, g.N, g.K, 128, o.ldw)) return rc;
    if (const int rc = bytes_map(&ma, o.a, g.M, g.K, MP, o.lda)) return rc;
    SwapGeo geo;
    geo.cs = cs;
    geo.m_tiles = (g.M + MP - 1u) / MP;
    const uint32_t k_blocks = (g.K + KB_BYTES - 1u) / KB_BYTES, slice = (k_blocks + cs - 1u) / cs;
    const uint32_t scale_bytes = slice * MP * 4u;
    // clusters of eight find a place on half SMs only
    const uint32_t budget = (cs == 8u ? 108u : 200u) * 1024u - scale_bytes;
    geo.stages = budget / STAGE_BYTES;
    if (geo.stages > (uint32_t)SWAP_MAX_STAGES) geo.stages = SWAP_MAX_STAGES;
    if (geo.stages > slice) geo.stages = slice;
    size_t smem = (size_t)geo.stages * STAGE_BYTES + scale_bytes;
    if (smem < MP * 512u) smem = MP * 512u;  // the sums
    const cudaError_t e = launch_cluster(gemm_fp8_swap_kernel<MP>, (g.N + 127u) / 128u * geo.m_tiles * cs, SWAP_THREADS, smem + 1024, cs, stream, mw, ma, g, geo);
    return e == cudaSuccess ? MIORI_OK : cuda_fail(e, "gemm_fp8 (few rows) launch");
}

// Which kernel takes a product, and how.
struct GemmPlan {
    uint32_t pair_n;  // columns of a pair's tile, 0: the kernel of few rows
    uint32_t mp, cs;
};
// The cheapest by a small model (us), whose numbers are what the kernels take a k-block once they run: 0.31 and 0.56 the tiles of pairs, of 128 and 256
// columns; 0.2, 0.23, 0.33 and 0.6 the kernel of few rows with 16, 32, 64 and 128 of them, which has 0.025 a row at its end and 0.7 where K is split; a
// wave's beginning and end on top; what HBM takes to deliver w is a floor.
inline GemmPlan plan_gemm_fp8(uint32_t M, uint32_t N, uint32_t K, uint32_t flags) {
    if (const uint32_t f = flags >> MIORI_TUNE_FP8_SHIFT & 7u) {
        if (f >= 5u) return {f == 5u ? 128u : 256u, 0, 0};
        return {0, 8u << f, 1u << (flags >> (MIORI_TUNE_FP8_SHIFT + 3) & 3u)};
    }
    const uint32_t sms = (uint32_t)sm_count(), k_blocks = (K + KB_BYTES - 1u) / KB_BYTES;
    auto waves = [](uint64_t n, uint32_t at_once) { return (double)((n + at_once - 1u) / at_once); };
    const double floor = (double)N * K / 5.5e6;
    GemmPlan best = {128, 0, 0};
    double best_t = 1e30;
    auto consider = [&](const GemmPlan& p, double t) {
        if (t < floor) t = floor;
        if (t < best_t) best_t = t, best = p;
    };
    const uint64_t m256 = (M + 255u) / 256u;
    consider({128, 0, 0}, waves(m256 * ((N + 127u) / 128u), sms / 2) * (k_blocks * 0.31 + 1.0) + 0.8);
    consider({256, 0, 0}, waves(m256 * ((N + 255u) / 256u), sms / 2) * (k_blocks * 0.56 + 1.4) + 0.8);
    if (k_blocks > 128u) return best;  // the kernel of few rows keeps its scales in shared memory
    static const double per_block[4] = {0.2, 0.23, 0.33, 0.6};
    for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t mp = 16u << i;
        if (mp >= 2u * M && mp > 16u) break;
        const uint64_t tiles = (uint64_t)((N + 127u) / 128u) * ((M + mp - 1u) / mp);
        for (uint32_t cs = 1; cs <= (mp == 128u ? 4u : 8u) && k_blocks >= cs; cs *= 2u) {  // 128 rows are an SM's registers: eight such SMs side by side are rare
            if (cs > 1u && tiles * cs > sms) break;
            consider({0, mp, cs}, waves(tiles * cs, sms) * ((k_blocks + cs - 1u) / cs * per_block[i] + mp * 0.025) + (cs > 1u ? 0.7 : 0.0));
        }
    }
    return best;
}

}  // namespace fp8
}  // namespace miori_b200
