// Attention of prompts and of chunks of them on the 5th-generation tensor cores: packed keys or the paged cache, causal or not.
//
// Tensor-bound: 4 * D operations a (row, key) pair, and one exponential.
//
// * An item has up to 256 rows: two tiles of 128 rows (tokens x the heads that share the key head).  Per tile of 128 keys a row
//   tile takes S = Q K^T (128 x 128 x D) into TMEM, its softmax, and O += P V (128 x D x 128) with P read from TMEM.
//   TMEM: O0, O1 (D columns each), P0, P1 (64 each), and S in what is left: with D = 64 128 columns for each row tile, with D = 128
//   128 that both use in turn, which they can since a softmax loads its S whole and at once.
// * MMAs with different accumulators complete in no order that is promised, so what one reads and another writes is handed over by
//   barriers and commits alone.  D = 64: the next scores are issued behind a tile's product, so that the commit that hands them to
//   the softmax says that the product is complete too, O stands still and P may be written.  D = 128: the next scores are issued in front
//   of it, once the softmax of the other row tile has loaded its own (s_free), and the softmax waits for the product
//   by itself (o_full).  Scores over the P that a product may still be reading would save those two waits
//   (prompts of up to 8192 tokens of 128 dimensions 376 us, so 387), in an order that nothing guarantees.
// * Warps 0-3 and 4-7 are the softmax of the two row tiles, a thread a row: no shuffle anywhere.  The two take turns on the
//   tensor cores: while one exponentiates, the other's products run.  Warp 8 issues the copies (TMA, 128-byte swizzle, a
//   ring of tiles: keys, values, keys, ...), an elected thread of warp 9 the MMAs, warps 10-11 look through the values of edge tiles.
// * The running maximum moves only when a row's exceeds it by 2^8: until then p grows up to 256 and O stays where it is.  O is rescaled
//   by the softmax warps themselves, in TMEM.
// * P is rounded to bf16 for the second product, as the values are, since an MMA has one type for both; l sums the rounded p, so that
//   O / l is a mean of values whatever their weights are off by: a key that outweighs all others is weighed by one, although its p
//   is not one with a maximum that stands still.  (Sums of the unrounded p: prompts of up to 8192 tokens 387 us, so 395, but off by up
//   to 2^-8 where one key dominates.  The rounded p unpacked and added as fp32 pairs 404, added on mma.sync 401.)
// * 432 GFLOP of prompts of up to 8192 tokens, 16 heads of 128 over 4: 456 us (0.95 PFLOP/s) call after call, when the power limit holds the
//   SMs at 1.66 GHz, and 387 (1.12) in a short graph.  Chunks of up to 512 tokens over 16 thousand: 177 and 148 us (0.85 and 1.02).
//   Narrow heads: 103 and 102.  The tensor pipe is active 60 % of the cycles and the special-function unit 56 % (one prompt of 8192).  A softmax
//   warp is busy nearly all the time (heads of 128; 3.3 thousand cycles a tile of keys, of which its exponentials alone would take one), two to an
//   SM's quarter: what it does one after the other bounds the kernel, and each branch in its loop costs percents.
// * Tried and dropped, all before the issue order, registers and sums as they are now, and so no proof against them (us, 404 then): an MMA warp
//   for each row tile (454), the MMAs issued by the softmax warps (473), scores of 64 keys double-buffered (684), the product begun at
//   half of the probabilities (403 - 430), a quarter or half of the exponentials by a polynomial on the FMA pipe (404, 466),
//   exponentials with the maximum of the tile before, taken again where that is too low (401).
// * Edge tiles (keys that some rows do not see, or past the end).  Their scores are masked one by one.  Their values are looked
//   through before the product: rows past the end are zeroed (a page's unwritten tail, the next prompt's rows) and so are
//   numbers that are not finite, since 0 * inf would reach rows that do not see them; rows that do see them get them added
//   at the end.
// * Positions whose table entry is no page of the cache are seen by nobody: the copying warp clears their rows of the tile, which hold what
//   was there before, and leaves word of them in `absent` for the softmax, which gives them no weight.
// * Shares of the items' key tiles are cut anywhere (attention.cuh); parts of an item meet in attention_join_kernel.
#pragma once
#include "attention.cuh"
#include "tma_host.cuh"

namespace miori_b200 {
namespace attention {

constexpr int PROMPT_THREADS = 384, KEYS = 128, ROW_TILE = 128;
constexpr uint32_t ITEM_COST = 384;     // an item's set-up and end, in positions: long prompts, narrow heads, chunks 387, 102, 148 us (256 389, 99, 150; 640 397, 109, 150)
constexpr uint32_t LEAST_SHARE = 256;   // positions; a tile of keys at least
// From here on scores are scaled first and then held against the maximum, which was rounded as they are.  The one fma that does both rounds
// at the end only, so that p is off by 2^(half an ulp of the maximum), the same for the whole row: by two here, and beyond fp32 at 2^31.
constexpr float HUGE_SCORE = 0x1p25f;

template <int D>
struct PromptCfg {
    static constexpr int HALVES = D / 64;                  // 128-byte columns of a row
    static constexpr int BLOCK = KEYS * 128;               // one of them, 128 rows
    static constexpr int TILE_BYTES = HALVES * BLOCK;
    static constexpr int STAGES = D == 128 ? 5 : 10;
    static constexpr int SMEM = 1024 + (2 + STAGES) * TILE_BYTES;
    static constexpr int PART_FLOATS = 2 * ROW_TILE * (D + 2);  // [D / 4][256] pieces of O, then m and l
    // columns of TMEM, 512 in all
    static constexpr int SCORES = D == 64 ? 2 : 1;         // places for S
    static constexpr int P_COLUMN = SCORES * KEYS, O_COLUMN = P_COLUMN + KEYS;
    static_assert(O_COLUMN + 2 * D == 512, "TMEM");
};
constexpr int SETMAXNREG_SOFTMAX = 200, SETMAXNREG_OTHERS = 104;  // 256 * 200 + 128 * 104 = 384 * 168, what a launch has; 192 and 120, 184 and 136 0.5 % slower, 208 and 88 5 %
static_assert(256 * SETMAXNREG_SOFTMAX + 128 * SETMAXNREG_OTHERS <= PROMPT_THREADS * 168, "a split above the launch's registers waits forever");

// ---- how the work is dealt ---------------------------------------------------------------
//
// An item costs ITEM_COST + the positions that its last token sees, so that the sum over the items of a head has a closed form
// (a product and a square) and a CTA finds its share in about a microsecond, however long the prompts are.  Tile k of an item belongs to
// the share that holds unit start + ITEM_COST - 1 + 128 k.  A share is never shorter than a tile of keys: of the shares between the
// first and the last of an item each holds at least one of its tiles.

__device__ __forceinline__ uint32_t item_tokens(const Args& a) { return 2u * (ROW_TILE / a.group); }
// Positions that the last token of item t sees.
__device__ __forceinline__ uint32_t item_seen(const Args& a, const Request& x, uint32_t t, uint32_t step) { return seen(a, x, min((t + 1u) * step, x.n) - 1u); }
// Cost of items 0 .. t-1 of one head.
__device__ __forceinline__ uint64_t cost_before(const Args& a, const Request& x, uint32_t t, uint32_t items, uint32_t step) {
    uint64_t cost = (uint64_t)t * ITEM_COST;
    if (!a.causal) return cost + (uint64_t)t * x.len;
    uint32_t full = t;
    if (t == items && t) cost += item_seen(a, x, t - 1u, step), --full;  // the last one may hold fewer tokens
    const int64_t before = x.before, after = (int64_t)x.len - before;
    const uint32_t none = before < 0 ? min((uint32_t)-before / step, full) : 0u;  // items none of whose tokens sees anything
    if (after < (int64_t)x.n) {  // and those whose last token stands at the end of what is there, or behind it
        const uint32_t in_front = after > 0 ? max(min(((uint32_t)after + step - 1u) / step - 1u, full), none) : none;
        cost += (uint64_t)(full - in_front) * x.len, full = in_front;
    }
    // item i sees before + (i + 1) step
    return cost + (uint64_t)((int64_t)(full - none) * before) + (((uint64_t)full * (full + 1u) - (uint64_t)none * (none + 1u)) / 2u) * step;
}

struct Item {
    Request x;
    uint32_t r, head, t, items, sees, tiles;
    uint64_t start;  // its first unit
    __device__ __forceinline__ void measure(const Args& a, uint32_t step) {
        sees = item_seen(a, x, t, step);
        tiles = max((sees + KEYS - 1u) / KEYS, 1u);
    }
    __device__ __forceinline__ uint64_t mark() const { return start + ITEM_COST - 1u; }  // of its first tile
    __device__ __forceinline__ uint64_t last_mark() const { return mark() + (uint64_t)(tiles - 1u) * KEYS; }
    template <bool PAGED>
    __device__ __forceinline__ void next(const Args& a, uint32_t step, uint64_t end) {
        start += ITEM_COST + sees;
        if (start >= end) return;  // there may be no further request
        if (++t == items) {
            t = 0u;
            if (++head == a.kv_heads) {
                head = 0u;
                do {
                    x = request<PAGED>(a, ++r);
                    items = (x.n + step - 1u) / step;
                } while (items == 0u && r + 1u < a.requests);
            }
        }
        measure(a, step);
    }
};
// This CTA's share and the item that it begins in (begin == end: nothing to do).  By a whole warp.
struct Start {
    Shares shares;
    uint64_t begin, end;
    Item it;
};
template <bool PAGED>
__device__ __forceinline__ Start find_share(const Args& a) {
    const uint32_t lane = threadIdx.x & 31u, step = item_tokens(a);
    Request mine = {};
    auto cost_of = [&](uint32_t r0) -> uint64_t {
        if (r0 + lane >= a.requests) return 0;
        mine = request<PAGED>(a, r0 + lane);
        const uint32_t items = (mine.n + step - 1u) / step;
        return cost_before(a, mine, items, items, step) * a.kv_heads;
    };
    uint64_t total = 0, cost = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 32u) {
        cost = cost_of(r0);
        total += warp_sum(cost);
    }
    Start st = {Shares(total, gridDim.x, LEAST_SHARE), 0, 0, {}};
    st.begin = st.shares.begin(blockIdx.x), st.end = st.shares.begin(blockIdx.x + 1u);
    if (st.begin == st.end) {
        st.it.start = st.end;  // no item before the end
        return st;
    }
    uint64_t before = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 32u) {
        if (a.requests > 32u) cost = cost_of(r0);
        const uint64_t sum = warp_prefix_sum(cost);
        const uint32_t past = __ballot_sync(0xFFFFFFFFu, before + sum > st.begin);
        if (past) {
            const uint32_t l = __ffs(past) - 1u;
            before += __shfl_sync(0xFFFFFFFFu, sum - cost, l);
            st.it.r = r0 + l;
            st.it.x.q0 = __shfl_sync(0xFFFFFFFFu, mine.q0, l), st.it.x.n = __shfl_sync(0xFFFFFFFFu, mine.n, l);
            st.it.x.k0 = __shfl_sync(0xFFFFFFFFu, mine.k0, l), st.it.x.len = __shfl_sync(0xFFFFFFFFu, mine.len, l);
            st.it.x.before = __shfl_sync(0xFFFFFFFFu, mine.before, l);
            break;
        }
        before += __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    Item& it = st.it;
    it.items = (it.x.n + step - 1u) / step;
    const uint64_t per_head = cost_before(a, it.x, it.items, it.items, step);
    it.head = small_quotient(st.begin - before, per_head);
    it.start = before + it.head * per_head;
    const uint64_t in = st.begin - it.start;
    uint32_t lo = 0, width = it.items;  // the item is in [lo, lo + width)
    while (width > 1u) {
        const uint32_t stride = (width + 31u) / 32u;
        const uint32_t below = __ballot_sync(0xFFFFFFFFu, lane * stride < width && cost_before(a, it.x, lo + lane * stride, it.items, step) <= in);
        const uint32_t l = 31u - __clz(below);  // lane 0 always is
        lo += l * stride;
        width = min(stride, width - l * stride);
    }
    it.t = lo;
    it.start += cost_before(a, it.x, lo, it.items, step);
    it.measure(a, step);
    return st;
}
// What of an item's key tiles falls into the share [begin, end).  Without a workspace items stay whole.
struct Span {
    uint32_t k0, k1;
    bool whole;
};
__device__ __forceinline__ uint32_t tiles_below(const Item& it, uint64_t unit) {
    return unit <= it.mark() ? 0u : (uint32_t)min((unit - it.mark() + KEYS - 1u) / KEYS, (uint64_t)it.tiles);
}
__device__ __forceinline__ Span span_of(const Item& it, uint64_t begin, uint64_t end, bool split) {
    Span s;
    s.k0 = tiles_below(it, begin);
    s.k1 = tiles_below(it, end);
    if (!split && s.k1 > s.k0) {
        if (s.k0 > 0u) s.k1 = s.k0;
        else s.k1 = it.tiles;
    }
    s.whole = s.k0 == 0u && s.k1 == it.tiles;
    return s;
}

// ---- tensor-core and TMEM instructions -------------------------------------------------------

// Shared-memory matrix descriptor, 128-byte swizzle, version of sm_100.  K-major: rows of 64 elements, 8-row atoms 1024 bytes
// apart.  MN-major (values: 64 dimensions contiguous, keys down the rows): lead = bytes from one 64 dimensions to the next.
__device__ __forceinline__ uint64_t smem_desc(uint32_t at, uint32_t lead) {
    return (uint64_t)((at & 0x3FFFFu) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction descriptor: D fp32, A and B bf16, 128 x n; B MN-major where `transposed`.
__device__ __forceinline__ constexpr uint32_t mma_desc(uint32_t n, bool transposed) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((transposed ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((uint32_t)(ROW_TILE >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_load32(uint32_t at, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]),
          "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]),
          "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]),
          "=f"(r[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]),
          "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
        "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
        "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}

// ---- two fp32 numbers at a time -----------------------------------------------------------

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if any of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// A value that all lanes hold, for the compiler to know that they do.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xFFFFFFFFu, x, 0); }
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0u;
}
// mbar_wait by a whole warp, with one answer for it.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t where) {
    if (__all_sync(0xFFFFFFFFu, mbar_try(bar, parity))) return true;
    return __all_sync(0xFFFFFFFFu, mbar_wait<false>(bar, parity, abort, where));
}

// ---- the kernel ------------------------------------------------------------------------------

template <int D, bool PAGED>
__global__ void __launch_bounds__(PROMPT_THREADS, 1)
attention_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Args a) {
    using C = PromptCfg<D>;
    constexpr uint32_t ST = C::STAGES, BARS = 4 * ST + 11;
    extern __shared__ uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[BARS];
    // Items of either row tile from whose values something was left out.  The ring holds five tiles, and a row tile's next item but one is
    // multiplied only after it has read the word of this one: eight words are enough.
    __shared__ uint32_t tmem_slot, dirty_item[2][8];
    // Of the last eight key tiles, a bit for each eight keys: no page.  Tile n + 8 is copied after the values of tile n + 5 at least have
    // been multiplied, and so after every softmax has read the word of tile n.
    __shared__ volatile uint32_t absent[8];
    __shared__ volatile uint32_t abort_flag;
    const uint32_t base = (smem_addr(smem) + 1023u) & ~1023u;
    const uint32_t q_at = base, ring = base + 2u * C::TILE_BYTES;
    auto bar = [&](uint32_t i) { return smem_addr(&bars[i]); };
    auto full = [&](uint32_t s) { return bar(s); };
    auto empty = [&](uint32_t s) { return bar(ST + s); };
    // The values of an edge tile arrive at `raw`, and the products wait for `checked`, where they have been looked through; everything
    // else arrives at `full`.  A place of the ring is filled again only after its products, so nobody is ever a turn ahead
    // at any of a place's barriers; which turn each is at, one bit a place says (`turns`).
    auto raw = [&](uint32_t s) { return bar(2 * ST + s); };
    auto checked = [&](uint32_t s) { return bar(3 * ST + s); };
    const uint32_t q_full = bar(4 * ST), q_empty = bar(4 * ST + 1);
    auto s_full = [&](uint32_t t) { return bar(4 * ST + 2 + t); };
    auto p_full = [&](uint32_t t) { return bar(4 * ST + 4 + t); };
    auto o_full = [&](uint32_t t) { return bar(4 * ST + 6 + t); };  // the item's O is complete; D = 128: the tile's product is
    auto o_free = [&](uint32_t t) { return bar(4 * ST + 8 + t); };  // the item's O has been read
    const uint32_t s_free = bar(4 * ST + 10);                          // D = 128: S has been loaded
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

    if (threadIdx.x == 0) {
        abort_flag = 0u;
        for (uint32_t i = 0; i < ST; ++i) mbar_init(full(i), 1), mbar_init(empty(i), 1), mbar_init(raw(i), 1), mbar_init(checked(i), 2);
        mbar_init(q_full, 1), mbar_init(q_empty, 1);
        for (uint32_t t = 0; t < 2; ++t) mbar_init(s_full(t), 1), mbar_init(p_full(t), 4), mbar_init(o_full(t), 1), mbar_init(o_free(t), 4);
        mbar_init(s_free, 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
    if (threadIdx.x < 16) dirty_item[threadIdx.x / 8u][threadIdx.x % 8u] = 0u;
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        pdl_launch_dependents();  // with its columns in hand
    }
    pdl_wait_prior();
    const uint32_t group = a.group, per_tile = ROW_TILE / group, per_item = 2u * per_tile;
    const bool split = a.parts != nullptr;
    __shared__ __align__(8) uint32_t plan[sizeof(Start) / 4];
    // where a softmax warp stands: its registers are for the scores (beside them they spilled: prompts of up to 8192 395 us, so 384)
    __shared__ __align__(8) uint32_t places[8][sizeof(Start) / 4];
    if (warp == 8) {  // for all: the code is cold, and one warp fetches it sooner than twelve
        const Start found = find_share<PAGED>(a);
        if (lane == 0) memcpy(plan, &found, sizeof(Start));
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    Start start = {Shares(0, 1, 1), 0, 0, {}};
    memcpy(&start, plan, sizeof(Start));
    Item& it = start.it;
    const uint64_t begin = start.begin, end = start.end;
    auto has_second = [&]() { return it.x.n > it.t * per_item + per_tile; };
    // first key tile of the item that some row does not see to its end
    auto first_edge = [&](uint32_t row_tile) { return seen(a, it.x, it.t * per_item + row_tile * per_tile) / KEYS; };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SETMAXNREG_OTHERS));
        if (warp == 8) {
            // ---- copies
            uint32_t n_tile = 0, n_item = 0;
            bool ok = true;
            while (ok && it.start < end) {
                const Span span = span_of(it, begin, end, split);
                if (span.k1 > span.k0) {
                    if (lane == 0) ok = mbar_wait(q_empty, (n_item & 1u) ^ 1u, &abort_flag, 1);
                    ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
                    if (!ok) break;
                    ++n_item;
                    if (lane == 0) {
                        const uint32_t tiles = has_second() ? 2u : 1u;
                        mbar_expect_tx(q_full, tiles * C::HALVES * per_tile * group * 128u);
                        for (uint32_t t = 0; t < tiles; ++t)
                            for (uint32_t h = 0; h < (uint32_t)C::HALVES; ++h)
                                tma_load_3d(q_at + t * C::TILE_BYTES + h * C::BLOCK, &map_q, (int)(64u * h), (int)(it.head * group),
                                            (int)(it.x.q0 + it.t * per_item + t * per_tile), q_full);
                    }
                    const uint32_t edge = first_edge(0);
                    for (uint32_t k = span.k0; ok && k < span.k1; ++k) {
                        int page = 0, row = (int)(it.x.k0 + k * KEYS);
                        uint32_t boxes = C::HALVES, box_rows = KEYS, mine = lane / C::HALVES;
                        const uint32_t half = lane % C::HALVES;
                        bool issue = lane < (uint32_t)C::HALVES;
                        uint32_t gone = 0;
                        if (PAGED) {
                            const uint32_t key0 = k * KEYS, left = it.x.len > key0 ? min(it.x.len - key0, (uint32_t)KEYS) : 0u;
                            const uint32_t in_box = min(1u << a.page_shift, (uint32_t)KEYS);
                            issue = mine * in_box < left;
                            if (issue) {
                                const uint32_t key = key0 + mine * in_box;
                                page = ld_fresh(a.table + (size_t)it.r * a.width + (key >> a.page_shift));
                                row = (int)(key & ((1u << a.page_shift) - 1u));
                                issue = (uint32_t)page < a.pages;
                            }
                            const uint32_t lost = __ballot_sync(0xFFFFFFFFu, mine * in_box < left && !issue);
                            if (lost) gone = __ballot_sync(0xFFFFFFFFu, lane < KEYS / 8u && lost >> (8u * lane / in_box * C::HALVES) & 1u);
                            box_rows = in_box;
                            boxes = __popc(__ballot_sync(0xFFFFFFFFu, issue));
                        }
#pragma unroll 1
                        for (uint32_t which = 0; which < 2u; ++which, ++n_tile) {
                            const uint32_t s = n_tile % ST, turn = n_tile / ST;
                            if (lane == 0) ok = mbar_wait(empty(s), (turn & 1u) ^ 1u, &abort_flag, 2);
                            ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
                            if (!ok) break;
                            const uint32_t arrive = which && k >= edge ? raw(s) : full(s);
                            if (PAGED && gone) {
                                __syncwarp();
                                for (uint32_t e = lane; e < (uint32_t)C::TILE_BYTES / 16u; e += 32u)
                                    if (gone >> (e / 64u % 16u) & 1u)
                                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + s * C::TILE_BYTES + 16u * e), "r"(0u) : "memory");
                                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                                __syncwarp();
                            }
                            if (PAGED && lane == 0 && which == 0u) absent[n_tile / 2u % 8u] = gone;
                            if (lane == 0) mbar_expect_tx(arrive, boxes * box_rows * 128u);
                            __syncwarp();
                            const uint32_t dst = ring + s * C::TILE_BYTES + half * C::BLOCK + mine * box_rows * 128u;
                            const CUtensorMap* map = which ? &map_v : &map_k;
                            if (issue) {
                                if (PAGED) tma_load_4d(dst, map, (int)(64u * half), row, (int)it.head, page, arrive);
                                else tma_load_3d(dst, map, (int)(64u * half), (int)it.head, row, arrive);
                            }
                        }
                    }
                }
                it.next<PAGED>(a, per_item, end);
            }
        } else if (warp == 9) {
            // ---- products.  The whole warp walks the loop and one elected thread issues: descriptors and addresses then stay in uniform
            // registers.  Issued from a branch of one lane an MMA took 88 cycles beside busy softmax warps, so 75 (and 64 without them); without
            // the __syncwarp behind each issue, lanes that run ahead into the next wait cost 15 % of the whole.
            constexpr uint32_t idesc_s = mma_desc(KEYS, false), idesc_o = mma_desc(D, true);
            const uint32_t tm = uniform(tmem);
            const uint64_t rows = smem_desc(q_at, 16u), keys = smem_desc(ring, 16u), values = smem_desc(ring, C::BLOCK);
            uint32_t place = 0, full_turns = 0, check_turns = 0, n_item = 0, n_p = 0, n_p1 = 0, n_o = 0, n_o1 = 0, n_s = 0;
            auto wait_full = [&](uint32_t s, uint32_t where) {
                const bool there = warp_wait(full(s), full_turns >> s & 1u, &abort_flag, where);
                full_turns ^= 1u << s;
                return there;
            };
            auto scores = [&](uint32_t t, uint32_t s, bool last) {
                if (C::SCORES == 1 && !warp_wait(s_free, (n_s++ & 1u) ^ 1u, &abort_flag, 13)) return false;
                fence_after();
                const uint64_t q = rows + t * (C::TILE_BYTES / 16u), at = keys + s * (C::TILE_BYTES / 16u);
                if (elect_one()) {
#pragma unroll
                    for (uint32_t k = 0; k < D / 16u; ++k) {  // 16 dimensions, 32 bytes further in the 128-byte rows
                        const uint32_t step = (k / 4u) * (C::BLOCK / 16u) + (k % 4u) * 2u;
                        mma_ss(tm + t % C::SCORES * KEYS, q + step, at + step, idesc_s, k > 0u);
                    }
                    mma_commit(s_full(t));
                    if (last) mma_commit(empty(s));  // the keys have been read
                }
                __syncwarp();
                return true;
            };
            while (__all_sync(0xFFFFFFFFu, it.start < end)) {
                const Span span = span_of(it, begin, end, split);
                const uint32_t k0 = uniform(span.k0), k1 = uniform(span.k1), sees = uniform(it.sees), edge = uniform(first_edge(0));
                const bool second = uniform(has_second() ? 1u : 0u) != 0u;
                if (k1 > k0) {
                    if (!warp_wait(q_full, n_item & 1u, &abort_flag, 3)) break;
                    ++n_item;
                    if (!wait_full(place, 4)) break;
                    bool ok = scores(0u, place, !second) && (!second || scores(1u, place, true));
                    if (!ok) break;
                    for (uint32_t k = k0; k < k1; ++k) {
                        const uint32_t vs = place + 1u == ST ? 0u : place + 1u, ks = vs + 1u == ST ? 0u : vs + 1u;
                        const bool more = k + 1u < k1;
                        if (k >= edge) {
                            ok = warp_wait(checked(vs), check_turns >> vs & 1u, &abort_flag, 6);
                            check_turns ^= 1u << vs;
                        } else {
                            ok = wait_full(vs, 5);
                        }
                        if (!ok) break;
                        if (!more && elect_one()) mma_commit(q_empty);  // the last scores are under way
                        if (more && !(ok = wait_full(ks, 4))) break;
                        // groups of 16 keys that some row sees: one at least, which then begins O
                        const uint32_t steps = sees > k * KEYS ? (min(sees - k * KEYS, (uint32_t)KEYS) + 15u) / 16u : 1u;
                        const uint64_t at = values + vs * (C::TILE_BYTES / 16u);
                        auto add = [&](uint32_t t, uint32_t& o_turn, uint32_t& p_turn, bool last) {
                            if (k == k0) {  // the last item's O has been read
                                if (!warp_wait(o_free(t), (o_turn & 1u) ^ 1u, &abort_flag, 7)) return false;
                                ++o_turn;
                            }
                            if (!warp_wait(p_full(t), p_turn & 1u, &abort_flag, 8)) return false;
                            ++p_turn;
                            fence_after();
                            if (elect_one()) {
                                const uint32_t o = tm + C::O_COLUMN + t * D, p = tm + C::P_COLUMN + t * (KEYS / 2);
                                if (steps == KEYS / 16u) {
#pragma unroll
                                    for (uint32_t i = 0; i < KEYS / 16u; ++i) mma_ts(o, p + 8u * i, at + 128u * i, idesc_o, k > k0 || i > 0u);  // 16 keys, 2048 bytes further
                                } else {
#pragma unroll 1
                                    for (uint32_t i = 0; i < steps; ++i) mma_ts(o, p + 8u * i, at + 128u * i, idesc_o, k > k0 || i > 0u);
                                }
                                if (C::SCORES == 1 || !more) mma_commit(o_full(t));
                                if (last) mma_commit(empty(vs));
                            }
                            __syncwarp();
                            return true;
                        };
                        auto go_on = [&](uint32_t t, uint32_t& o_turn, uint32_t& p_turn, bool last) {
                            if (C::SCORES == 2) return add(t, o_turn, p_turn, last) && (!more || scores(t, ks, last));
                            return (!more || scores(t, ks, last)) && add(t, o_turn, p_turn, last);
                        };
                        if (!(ok = go_on(0u, n_o, n_p, !second) && (!second || go_on(1u, n_o1, n_p1, true)))) break;
                        place = ks;
                    }
                    if (!ok) break;
                }
                it.next<PAGED>(a, per_item, end);
            }
        } else {
            // ---- values of edge tiles: half the rows for each of two warps
            uint32_t n_tile = 0, n_item[2] = {}, turns = 0;
            bool ok = true;
            while (ok && it.start < end) {
                const Span span = span_of(it, begin, end, split);
                if (span.k1 > span.k0) {
                    const uint32_t edge = first_edge(0);
                    for (uint32_t k = span.k0; ok && k < span.k1; ++k, n_tile += 2u) {
                        if (k < edge) continue;
                        const uint32_t s = (n_tile + 1u) % ST;
                        ok = mbar_wait(raw(s), turns >> s & 1u, &abort_flag, 9);
                        turns ^= 1u << s;
                        ok = __all_sync(0xFFFFFFFFu, ok);
                        if (!ok) break;
                        const uint32_t there = it.x.len > k * KEYS ? min(it.x.len - k * KEYS, (uint32_t)KEYS) : 0u;
                        // 16-byte pieces; rows are 128 bytes, so the swizzle does not matter.  A number is not finite where its
                        // exponent bits are all set: first the largest exponents, and a second look only where one is
                        const uint32_t row0 = 64u * (warp - 10u), rows = there > row0 ? min(there - row0, 64u) : 0u;
                        auto piece = [&](uint32_t e) { return ring + s * C::TILE_BYTES + (e / 512u) * C::BLOCK + (row0 + e / 8u % 64u) * 128u + e % 8u * 16u; };
                        uint32_t most = 0u;
#pragma unroll 8
                        for (uint32_t e = lane; e < 512u * C::HALVES; e += 32u) {
                            uint32_t w[4];
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(piece(e)) : "memory");
                            const uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7F807F80u, w[1] & 0x7F807F80u), __vmaxu2(w[2] & 0x7F807F80u, w[3] & 0x7F807F80u));
                            if (e / 8u % 64u < rows) most = __vmaxu2(most, top);
                        }
                        const bool bad = __any_sync(0xFFFFFFFFu, (most & 0xFFFFu) == 0x7F80u || most >> 16 == 0x7F80u);
                        // past the end: up to the next multiple of 16 keys, where the product stops
                        const uint32_t stop = there == 0u && warp == 10u ? 16u : min((rows + 15u) & ~15u, 64u);
                        if (rows < stop) {
                            for (uint32_t e = rows * 8u + lane; e < stop * 8u; e += 32u)
#pragma unroll
                                for (uint32_t h = 0; h < (uint32_t)C::HALVES; ++h)
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(piece(e + 512u * h)), "r"(0u) : "memory");
                        }
                        if (bad) {
#pragma unroll 1
                            for (uint32_t e = lane; e < 512u * C::HALVES; e += 32u) {
                                uint32_t w[4] = {};
                                if (e / 8u % 64u < rows) {
                                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(piece(e)) : "memory");
#pragma unroll
                                    for (int i = 0; i < 4; ++i) w[i] = finite_or_zero(w[i]);
                                }
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece(e)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                            }
                        }
                        if (bad || rows < stop) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        if (bad && lane == 0) {
                            dirty_item[0][n_item[0] & 7u] = n_item[0] + 1u;
                            if (has_second()) dirty_item[1][n_item[1] & 7u] = n_item[1] + 1u;
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(checked(s));
                    }
                    ++n_item[0], n_item[1] += has_second();
                }
                it.next<PAGED>(a, per_item, end);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SETMAXNREG_SOFTMAX));
        // ---- softmax of a row tile, a thread a row
        const uint32_t t = warp >> 2, row = threadIdx.x & 127u;
        const uint32_t lanes = ((warp & 3u) * 32u) << 16;
        const uint32_t s_at = tmem + lanes + t % C::SCORES * KEYS, p_at = tmem + lanes + C::P_COLUMN + t * (KEYS / 2), o_at = tmem + lanes + C::O_COLUMN + t * D;
        const bool wide = (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0u && a.o_token % 16 == 0 && a.o_head % 16 == 0;
        uint32_t n_s = 0, n_o = 0, n_item = 0, tile0 = 0;  // tile0: key tiles of the items before
        memcpy(places[warp], plan, sizeof(Start));
        __syncwarp();
        Start& start = *reinterpret_cast<Start*>(places[warp]);
        Item& it = start.it;
        const uint64_t begin = start.begin, end = start.end;
        if (split && threadIdx.x == 0) a.joins[blockIdx.x] = make_uint4(0u, 0u, 0u, 0u);
        bool ok = true;
        auto has_second = [&]() { return it.x.n > it.t * per_item + per_tile; };
        auto first_edge = [&](uint32_t row_tile) { return seen(a, it.x, it.t * per_item + row_tile * per_tile) / KEYS; };
        while (ok && it.start < end) {
            const Span span = span_of(it, begin, end, split);
            if (span.k1 > span.k0) {
                if (t == 0u || has_second()) {
                    const uint32_t item_id = n_item++;
                    const uint32_t i = it.t * per_item + t * per_tile + row / group;
                    const bool there = row < per_tile * group && i < it.x.n;
                    const uint32_t sees = there ? seen(a, it.x, i) : 0u;
                    const uint32_t edge = first_edge(t);
                    float m = -INFINITY, l = 0.0f;
                    for (uint32_t k = span.k0; k < span.k1; ++k, ++n_s) {
                        ok = warp_wait(s_full(t), n_s & 1u, &abort_flag, 10);
                        if (!ok) break;
                        fence_after();
                        const uint32_t gone = PAGED ? absent[(tile0 + k - span.k0) % 8u] : 0u;
                        float s[KEYS];
#pragma unroll
                        for (int c = 0; c < 4; ++c) tmem_load32(s_at + 32u * c, s + 32 * c);
                        tmem_wait_load();
                        if (C::SCORES == 1) {
                            fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(s_free);
                        }
                        if (k >= edge) {
                            const uint32_t key0 = k * KEYS;
                            const uint32_t count = sees > key0 ? sees - key0 : 0u;
#pragma unroll
                            for (uint32_t j = 0; j < KEYS; ++j) s[j] = j < count ? s[j] : -INFINITY;
                        }
                        auto largest = [&] {
                            float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                            for (int j = 4; j + 8 <= KEYS; j += 8) {
#pragma unroll
                                for (int c = 0; c < 4; ++c) top[c] = max3_nan(top[c], s[j + c], s[j + 4 + c]);
                            }
                            const float all = max3_nan(max3_nan(top[0], top[1], top[2]), max3_nan(top[3], s[KEYS - 4], s[KEYS - 3]), max3_nan(s[KEYS - 2], s[KEYS - 1], top[0])) * a.scale_log2;
                            return all == INFINITY ? NAN : all;  // inf - inf, for the whole row
                        };
                        float now = largest();
                        if (C::SCORES == 1 && k > span.k0) {  // the product before is complete: P may be written, O stands still
                            ok = warp_wait(o_full(t), n_o++ & 1u, &abort_flag, 11);
                            if (!ok) break;
                            fence_after();
                        }
                        if (k == span.k0) m = now;
                        if (__any_sync(0xFFFFFFFFu, !(now <= m + 8.0f) || fabsf(m) >= HUGE_SCORE || gone)) {
                            if (gone) {  // scores of no page are zeros so far; here, since a test of its own costs 5 % of a chunk's time
#pragma unroll
                                for (uint32_t j = 0; j < KEYS; ++j) s[j] = gone >> (j / 8u) & 1u ? -INFINITY : s[j];
                                now = largest();
                                if (k == span.k0) m = now;
                            }
                            now = max3_nan(now, m, m);
                            const float keep = now == -INFINITY ? 1.0f : exp2_fast(m - now);
                            m = now;
                            l *= keep;
                            if (fabsf(m) >= HUGE_SCORE && m != -INFINITY) {  // what the fma below makes the difference of
                                const float back = 1.0f / a.scale_log2;
#pragma unroll
                                for (int j = 0; j < KEYS; ++j) s[j] = __fadd_rn(__fmul_rn(s[j], a.scale_log2), -m) * back;
                            }
#pragma unroll 1
                            for (uint32_t c = 0; c < (k > span.k0 ? D : 0u); c += 16u) {
                                float o[16];
                                tmem_load16(o_at + c, o);
                                tmem_wait_load();
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[j] *= keep;
                                tmem_store16(o_at + c, reinterpret_cast<const uint32_t*>(o));
                            }
                            tmem_wait_store();
                        }
                        const float from = fabsf(m) >= HUGE_SCORE ? 0.0f : -m;
                        float sum[4] = {};
                        const uint64_t scale2 = pair(a.scale_log2, a.scale_log2), from2 = pair(from, from);
#pragma unroll
                        for (int c = 0; c < KEYS; c += 32) {
                            uint32_t p[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                float &x = s[c + 2 * j], &y = s[c + 2 * j + 1];
                                uint64_t e = fma2(pair(x, y), scale2, from2);
                                unpair(e, x, y);
                                x = exp2_fast(x), y = exp2_fast(y);
                                p[j] = pack_bf16(x, y);
                                sum[j & 3] = add_bf16(sum[j & 3], p[j]);
                            }
                            tmem_store16(p_at + c / 2, p);
                        }
                        tmem_wait_store();
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_full(t));
                        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    }
                    if (!ok) break;
                    ok = warp_wait(o_full(t), n_o & 1u, &abort_flag, 12);
                    ++n_o;
                    if (!ok) break;
                    fence_after();
                    const bool dirty = *(volatile uint32_t*)&dirty_item[t][item_id & 7u] == item_id + 1u;
                    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // no key: zeros; NaN stays
                    const float factor = span.whole ? inv : 1.0f;
                    uint16_t* const to = a.out + (int64_t)(it.x.q0 + (there ? i : 0u)) * a.o_token + (int64_t)(it.head * group + row % group) * a.o_head;
                    float* part = nullptr;
                    if (!span.whole) {
                        const uint32_t first = start.shares.of(it.mark());
                        if (first == blockIdx.x && threadIdx.x == 0) a.joins[blockIdx.x] = make_uint4(start.shares.of(it.last_mark()) - first + 1u, it.x.q0 + it.t * per_item, it.x.n - it.t * per_item, it.head);
                        part = a.parts + (size_t)(2u * blockIdx.x + (first == blockIdx.x ? 1u : 0u)) * C::PART_FLOATS;
                        part[2u * ROW_TILE * D + t * ROW_TILE + row] = m;
                        part[2u * ROW_TILE * (D + 1) + t * ROW_TILE + row] = l;
                    }
#pragma unroll 1
                    for (uint32_t c = 0; c < D; c += 32u) {
                        float o[32];
                        tmem_load32(o_at + c, o);
                        tmem_wait_load();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] *= factor;
                        if (dirty) {  // values that are not finite, left out of the product, reach the rows that see them
#pragma unroll 1
                            for (uint32_t key = max(first_edge(0), span.k0) * KEYS; key < min(sees, span.k1 * KEYS); ++key) {
                                int64_t at = (int64_t)it.head * a.v_head + c;
                                if (PAGED) {
                                    const uint32_t pg = (uint32_t)ld_fresh(a.table + (size_t)it.r * a.width + (key >> a.page_shift));
                                    if (pg >= a.pages) continue;
                                    at += (int64_t)pg * a.v_page + (int64_t)(key & ((1u << a.page_shift) - 1u)) * a.v_slot;
                                } else {
                                    at += (int64_t)(it.x.k0 + key) * a.v_slot;
                                }
#pragma unroll
                                for (int j = 0; j < 32; ++j) {
                                    const float v = bf16_bits_to_float(ld_fresh(a.v + at + j));
                                    if (!(fabsf(v) < INFINITY)) o[j] += v;
                                }
                            }
                        }
                        if (!span.whole) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                *reinterpret_cast<float4*>(part + ((size_t)(c / 4u + j) * 2u * ROW_TILE + t * ROW_TILE + row) * 4u) =
                                    make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                        } else if (there) {
                            uint32_t w[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) w[j] = pack_bf16(o[2 * j], o[2 * j + 1]);
                            if (wide) {  // whole sectors: a lane's row is its own
#pragma unroll
                                for (int j = 0; j < 2; ++j)
                                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + c + 16 * j), "r"(w[8 * j]), "r"(w[8 * j + 1]),
                                                 "r"(w[8 * j + 2]), "r"(w[8 * j + 3]), "r"(w[8 * j + 4]), "r"(w[8 * j + 5]), "r"(w[8 * j + 6]), "r"(w[8 * j + 7])
                                                 : "memory");
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(to + c + 8 * j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                            }
                        }
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(o_free(t));
                }
                tile0 += span.k1 - span.k0;
            }
            __syncwarp();
            if (lane == 0) it.next<PAGED>(a, per_item, end);
            __syncwarp();
        }
    }

    // on abort give copies and MMAs in flight time to land before TMEM is freed
    __syncwarp();
    if (abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) __nanosleep(1000);
    }
    fence_before();
    __syncthreads();
    if (warp == 9) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Parts of items that more than one CTA worked on, added up in the order of their keys.  CTA (k, y): rows [64 y, 64 y + 64) of the
// item that CTA k of the kernel above began and did not end, if there is one (joins[k]: CTAs, first token, tokens left, key head).
constexpr int JOIN_THREADS = 512, JOIN_ROWS = 64;
template <int D>
__global__ void __launch_bounds__(JOIN_THREADS) attention_join_kernel(const Args a) {
    using C = PromptCfg<D>;
    pdl_launch_dependents();
    pdl_wait_prior();
    const uint4 join = ld_fresh(a.joins + blockIdx.x);
    if (join.x == 0u) return;
    const uint32_t first = blockIdx.x, last = first + join.x - 1u;
    const uint32_t group = a.group, per_tile = ROW_TILE / group;
    auto part = [&](uint32_t c) { return a.parts + (size_t)(2u * c + (c == first ? 1u : 0u)) * C::PART_FLOATS; };
    for (uint32_t e = threadIdx.x; e < JOIN_ROWS * (D / 8u); e += JOIN_THREADS) {
        const uint32_t row = JOIN_ROWS * blockIdx.y + e % JOIN_ROWS, c8 = e / JOIN_ROWS;
        const uint32_t in_tile = row % ROW_TILE, i = (row / ROW_TILE) * per_tile + in_tile / group;
        if (in_tile >= per_tile * group || i >= join.z) continue;
        float m = -INFINITY;
        for (uint32_t c = first; c <= last; ++c) m = fmaxf(m, ld_fresh(part(c) + 2u * ROW_TILE * D + row));
        const float from = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, o[8] = {};
#pragma unroll 4
        for (uint32_t c = first; c <= last; ++c) {
            const float f = exp2_fast(ld_fresh(part(c) + 2u * ROW_TILE * D + row) - from);
            l = fmaf(ld_fresh(part(c) + 2u * ROW_TILE * (D + 1) + row), f, l);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 x = ld_fresh(reinterpret_cast<const float4*>(part(c)) + (size_t)(2u * c8 + h) * 2u * ROW_TILE + row);
                o[4 * h] = fmaf(x.x, f, o[4 * h]), o[4 * h + 1] = fmaf(x.y, f, o[4 * h + 1]);
                o[4 * h + 2] = fmaf(x.z, f, o[4 * h + 2]), o[4 * h + 3] = fmaf(x.w, f, o[4 * h + 3]);
            }
        }
        const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
        uint16_t* to = a.out + (int64_t)(join.y + i) * a.o_token + (int64_t)(join.w * group + in_tile % group) * a.o_head + 8u * c8;
        *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv), pack_bf16(o[4] * inv, o[5] * inv),
                                                   pack_bf16(o[6] * inv, o[7] * inv));
    }
}

}  // namespace attention
}  // namespace miori_b200
