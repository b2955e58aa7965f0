// In front of the attention of a step: which cache slot every new token gets, and the heads of the QKV projection on their
// way into the cache.
//   page_slots  positions, slots and new pages from the requests' lengths   (reference: src/batch.cpp:704-719 fills such
//               arrays on the host for 32 fixed slots of a contiguous cache)
//   rope_kv     head norm, rotary positions of one to four axes, bf16 q, k and v into their slots   (reference, unfused and
//               for one axis: src/engine.cpp:406-483)
#include "common.cuh"

namespace miori_b200 {
namespace pages {

// ---- page_slots -------------------------------------------------------------------------
// With own(x) = ceil(x / page): request r needs own(held + new) - own(held) new pages, they come out of the pool in the order
// of the requests, and token i of request r sits at position held + i of its pages.  Two exclusive prefix sums and a search.
//
// Latency-bound: 8 bytes a request read and 8 a token written.  Every CTA does the prefix sums by itself (8 bytes a request
// from L2), so that none waits for another; they then share the tokens and the new table entries.  A token's page is taken from
// the pool and not from the table entry that another CTA writes beside it, so nothing here depends on the order of the CTAs.
// A request holds 2^31 - 1 positions at most: its further tokens have no slot.
// 32 requests of one token 4.7 us, 64 prompts of 41 thousand tokens 4.5.
constexpr uint32_t SLOT_THREADS = 512, TOKENS_PER_CTA = 4 * SLOT_THREADS, MAX_REQUESTS = 16384, MAX_POSITIONS = 0x7FFFFFFFu;

struct SlotArgs {
    const int32_t *held, *fresh;
    int32_t* table;
    const int32_t *pool, *taken;
    int32_t *slots, *positions, *cu, *held_after, *taken_after;
    uint32_t requests, width, page, pool_size, tokens, aligned;
};

// Number of entries of a[0, n) (ascending) that are <= x, less one: the row whose range holds x.
__device__ __forceinline__ uint32_t row_of(const int32_t* a, uint32_t n, int32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(SLOT_THREADS) page_slots_kernel(const SlotArgs a) {
    extern __shared__ int32_t prefix[];  // first token of each request, then first new page of each
    __shared__ int2 warp_sum[SLOT_THREADS / 32];
    int32_t* const first_token = prefix;
    int32_t* const first_page = prefix + a.requests + 1u;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    pdl_launch_dependents();
    pdl_wait_prior();
    const int32_t cap = (int32_t)a.width;
    const int32_t taken = ld_fresh(a.taken);
    auto owned = [&](int32_t n) { return min((int32_t)(((uint32_t)n + a.page - 1u) / a.page), cap); };
    int2 base = make_int2(0, 0);
    for (uint32_t r0 = 0; r0 < a.requests; r0 += SLOT_THREADS) {
        const uint32_t r = r0 + threadIdx.x;
        int2 mine = make_int2(0, 0);
        if (r < a.requests) {
            const int32_t held = max(ld_fresh(a.held + r), 0);
            mine.x = max(ld_fresh(a.fresh + r), 0);
            const int32_t after = (int32_t)min((uint32_t)held + (uint32_t)mine.x, MAX_POSITIONS);
            mine.y = owned(after) - owned(held);
            if (blockIdx.x == 0) a.held_after[r] = after;
        }
        int2 sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t x = __shfl_up_sync(0xFFFFFFFFu, sum.x, o), y = __shfl_up_sync(0xFFFFFFFFu, sum.y, o);
            if (lane >= (uint32_t)o) sum.x += x, sum.y += y;
        }
        if (lane == 31u) warp_sum[warp] = sum;
        __syncthreads();
        int2 before = base, all = base;
#pragma unroll
        for (uint32_t w = 0; w < SLOT_THREADS / 32u; ++w) {
            const int2 s = warp_sum[w];
            if (w < warp) before.x += s.x, before.y += s.y;
            all.x += s.x, all.y += s.y;
        }
        if (r < a.requests) {
            first_token[r] = before.x + sum.x - mine.x;
            first_page[r] = before.y + sum.y - mine.y;
            if (blockIdx.x == 0) a.cu[r] = before.x + sum.x - mine.x;
        }
        base = all;
        __syncthreads();
    }
    const int32_t total = base.x, new_pages = base.y;
    if (threadIdx.x == 0) {
        first_token[a.requests] = total;
        first_page[a.requests] = new_pages;
        if (blockIdx.x == 0) a.cu[a.requests] = total, *a.taken_after = taken + new_pages;
    }
    __syncthreads();

    auto from_pool = [&](int32_t j) {  // page number j of this step's, -1 once the pool is empty
        const int64_t at = (int64_t)taken + j;
        return at >= 0 && at < (int64_t)a.pool_size ? ld_fresh(a.pool + at) : -1;
    };
    for (uint32_t j = blockIdx.x * SLOT_THREADS + threadIdx.x; j < (uint32_t)new_pages; j += gridDim.x * SLOT_THREADS) {
        const uint32_t r = row_of(first_page, a.requests + 1u, (int32_t)j);
        const int32_t held = max(ld_fresh(a.held + r), 0);
        a.table[(size_t)r * a.width + (uint32_t)(owned(held) + (int32_t)j - first_page[r])] = from_pool((int32_t)j);
    }
    // four tokens a thread, stored as one piece each way where the outputs are 16-byte aligned
    const uint32_t t0 = blockIdx.x * TOKENS_PER_CTA + threadIdx.x * 4u;
    if (t0 >= a.tokens) return;
    int32_t slot[4], pos[4];
    uint32_t r = (int32_t)t0 < total ? row_of(first_token, a.requests + 1u, (int32_t)t0) : a.requests;
    int32_t held = 0, own = 0;
    bool known = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int32_t t = (int32_t)t0 + i;
        slot[i] = -1, pos[i] = 0;
        if (t >= total || t0 + i >= a.tokens) continue;
        while (t >= first_token[r + 1u]) ++r, known = false;
        if (!known) held = max(ld_fresh(a.held + r), 0), own = owned(held), known = true;
        const uint32_t at = (uint32_t)held + ((uint32_t)t - (uint32_t)first_token[r]);
        pos[i] = (int32_t)min(at, MAX_POSITIONS);
        const int32_t col = (int32_t)((uint32_t)pos[i] / a.page);
        if (at >= MAX_POSITIONS || col >= cap) continue;
        const int32_t p = col < own ? ld_fresh(a.table + (size_t)r * a.width + (uint32_t)col) : from_pool(first_page[r] + col - own);
        const int64_t to = (int64_t)p * a.page + (uint32_t)pos[i] % a.page;
        if (to >= 0 && to <= 0x7FFFFFFF) slot[i] = (int32_t)to;  // slots are int32
    }
    if (t0 + 4u <= a.tokens && a.aligned) {
        *reinterpret_cast<int4*>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
        for (uint32_t i = 0; i < 4u && t0 + i < a.tokens; ++i) a.slots[t0 + i] = slot[i], a.positions[t0 + i] = pos[i];
    }
}

// ---- rope_kv ------------------------------------------------------------------------------
// A head x of a token: x <- x * rsqrt(mean(x^2) + eps) * gamma (q and k, where gamma is given), then every pair (a, b) of its
// first `rotary` elements turned by its angle, (a cos - b sin, b cos + a sin); the rest and v pass through.  fp32 throughout,
// rounded to bf16 once at the end.
//
// The angle of pair j is position[axes[j]] * turns[j] in units of 2^-64 turns: a 64-bit product that wraps around drops whole
// turns exactly, so that the angle is as good at position 2^31 as at 1 (an fp32 product is off by 2^-24 of the whole angle: 0.004
// radians at position 65536).  Its upper 32 bits, rounded to the 24 of an fp32, are the sine's argument: off by 2^-26 turns at most.
//
// A thread holds eight pairs, which is two 8-element pieces of a head: D / 16 threads share a head, and for one token the same
// threads take further heads with the same sines.  A warp's threads compute each sine once and hand it to those that need it.
// HBM-bound for many tokens (one warp walks all heads of a token), latency-bound for few (a warp for every 32 / (D / 16) heads):
// `parts` warps share a token.  16384 tokens of 24 heads of 128 in bf16 37.4 us, 5.4 TB/s of reads and writes; 32 tokens of fp32 2.4 us.
constexpr uint32_t ROPE_THREADS = 128;  // 16384 tokens: 37.4 us, with 256 40.3 (fewer warps fit an SM)

struct RopeArgs {
    const void* qkv;
    const uint64_t* turns;
    const int32_t *axes, *positions, *slots;
    const uint16_t *gamma_q, *gamma_k;
    uint16_t *q, *k, *v;
    int64_t row, k_page, k_head, k_slot, v_page, v_head, v_slot;  // strides in elements
    uint32_t tokens, heads, kv_heads, rotary, num_axes, page, pages, parts;
    float eps;
    uint32_t early;  // turns and axes may be read ahead of the wait
};

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
    x[0] = bf16lo(w.x), x[1] = bf16hi(w.x), x[2] = bf16lo(w.y), x[3] = bf16hi(w.y);
    x[4] = bf16lo(w.z), x[5] = bf16hi(w.z), x[6] = bf16lo(w.w), x[7] = bf16hi(w.w);
}
// Eight elements as they lie in memory.
template <bool FP32>
struct Raw8 {
    uint4 w[FP32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* p, int64_t at) {
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + at * (FP32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (FP32 ? 2 : 1); ++i) w[i] = ld_fresh<uint4, true>(from + i);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        if constexpr (FP32) {
            memcpy(x, w, sizeof(x));
        } else {
            unpack8(w[0], x);
        }
    }
};

template <int D, bool FP32, bool ADJACENT>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kv_kernel(const RopeArgs a) {
    constexpr uint32_t TPH = D / 16, HPW = 32u / TPH;  // threads a head, heads a warp
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & 31u, u = lane % TPH;
    const uint32_t id = blockIdx.x * (ROPE_THREADS / 32u) + (threadIdx.x >> 5);
    const uint32_t t = id / a.parts, part = id % a.parts;
    if (t >= a.tokens) return;
    const uint32_t turning = a.rotary / 16u;  // threads of a head whose pairs turn
    // pieces of 8 elements: (u, u + rotary / 16) where pairs are `rotary / 2` apart, neighbours otherwise
    const bool turns_here = u < turning;
    const uint32_t e0 = turns_here && !ADJACENT ? 8u * u : 16u * u;
    const uint32_t e1 = turns_here && !ADJACENT ? e0 + a.rotary / 2u : e0 + 8u;
    // the threads of a warp that hold the same pairs, of HPW heads, compute PER of them each
    constexpr uint32_t PER = 8u / HPW;
    if (!a.early) pdl_wait_prior();
    uint64_t turn[PER] = {};
    uint32_t axis[PER] = {};
    if (turns_here) {
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t j = 8u * u + lane / TPH * PER + i;
            turn[i] = ld_fresh(a.turns + j);
            axis[i] = a.axes ? min((uint32_t)ld_fresh(a.axes + j), a.num_axes - 1u) : 0u;
        }
    }
    pdl_wait_prior();
    const uint32_t all = a.heads + 2u * a.kv_heads, first = part * HPW + lane / TPH;
    const int64_t row = (int64_t)t * a.row;
    // this head's elements, read ahead of what is done with the one before (and of the sines)
    Raw8<FP32> rx, ry;
    auto read = [&](uint32_t h) {
        const int64_t from = row + (int64_t)min(h, all - 1u) * D;
        rx.load(a.qkv, from + e0), ry.load(a.qkv, from + e1);
    };
    read(first);
    const int32_t slot = ld_fresh(a.slots + t);
    float mine_c[PER], mine_s[PER], c[8], s[8];
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        mine_c[i] = 1.0f, mine_s[i] = 0.0f;
        if (!turns_here) continue;
        const int32_t pos = ld_fresh(a.positions + (size_t)axis[i] * a.tokens + t);
        const uint64_t phase = (uint64_t)(int64_t)pos * turn[i];
        sincospif((float)(int32_t)(uint32_t)(phase >> 32) * 0x1p-31f, &mine_s[i], &mine_c[i]);
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        c[j] = __shfl_sync(0xFFFFFFFFu, mine_c[j % PER], j / PER * TPH + u);
        s[j] = __shfl_sync(0xFFFFFFFFu, mine_s[j % PER], j / PER * TPH + u);
    }
    const bool kept = slot >= 0 && (uint32_t)slot < a.pages * a.page;
    const uint32_t in_page = kept ? (uint32_t)slot / a.page : 0u, at = kept ? (uint32_t)slot % a.page : 0u;
#pragma unroll 1
    for (uint32_t h = first; h - lane / TPH < all; h += a.parts * HPW) {
        const bool there = h < all;
        const uint32_t hh = there ? h : all - 1u;
        float x[8], y[8];
        rx.get(x), ry.get(y);
        if (h - lane / TPH + a.parts * HPW < all) read(h + a.parts * HPW);
        const bool is_q = hh < a.heads, is_v = hh >= a.heads + a.kv_heads;
        const uint16_t* gamma = is_v ? nullptr : is_q ? a.gamma_q : a.gamma_k;
        if (a.gamma_q || a.gamma_k) {  // the same for the whole warp: the shuffles are
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], fmaf(y[j], y[j], sum));
#pragma unroll
            for (uint32_t o = TPH / 2u; o > 0u; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (gamma) {
                const float inv = rsqrtf(sum * (1.0f / D) + a.eps);
                float gx[8], gy[8];
                unpack8(ld_fresh(reinterpret_cast<const uint4*>(gamma + e0)), gx);
                unpack8(ld_fresh(reinterpret_cast<const uint4*>(gamma + e1)), gy);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= inv * gx[j], y[j] *= inv * gy[j];
            }
        }
        if (turns_here && !is_v) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float& p = ADJACENT ? (j < 4 ? x[2 * j] : y[2 * j - 8]) : x[j];
                float& q = ADJACENT ? (j < 4 ? x[2 * j + 1] : y[2 * j - 7]) : y[j];
                const float turned = p * c[j] - q * s[j];
                q = q * c[j] + p * s[j];
                p = turned;
            }
        }
        uint16_t* to;
        if (is_q) to = a.q + ((size_t)t * a.heads + hh) * D;
        else if (!is_v) to = a.k + (in_page * a.k_page + (int64_t)(hh - a.heads) * a.k_head + at * a.k_slot);
        else to = a.v + (in_page * a.v_page + (int64_t)(hh - a.heads - a.kv_heads) * a.v_head + at * a.v_slot);
        if (there && (is_q || kept)) {
            *reinterpret_cast<uint4*>(to + e0) = pack8(x);
            *reinterpret_cast<uint4*>(to + e1) = pack8(y);
        }
    }
}

}  // namespace pages
}  // namespace miori_b200

using namespace miori_b200;

MIORI_API int miori_page_slots(const int32_t* held, const int32_t* fresh, int32_t* table, const int32_t* pool, const int32_t* taken,
                               int32_t* slots, int32_t* positions, int32_t* cu, int32_t* held_after, int32_t* taken_after,
                               uint32_t requests, uint32_t width, uint32_t page, uint32_t pool_size, uint32_t tokens, uint32_t flags,
                               void* stream) {
    using namespace pages;
    if (!held || !fresh || !table || !pool || !taken || !cu || !held_after || !taken_after || (tokens && (!slots || !positions)))
        return fail(MIORI_E_INVALID, "page_slots: null pointer");
    if (requests == 0 || requests > MAX_REQUESTS) return fail(MIORI_E_INVALID, "page_slots: 1..%u requests, got %u", MAX_REQUESTS, requests);
    if (width == 0 || page == 0) return fail(MIORI_E_INVALID, "page_slots: empty table or page (width=%u page=%u)", width, page);
    if (page > (1u << 30)) return fail(MIORI_E_INVALID, "page_slots: pages of up to 2^30 positions, got %u", page);
    if ((uint64_t)requests * width > 0x7FFFFFFFull) return fail(MIORI_E_INVALID, "page_slots: a table of 2^31 entries or more");
    if (tokens > 0x7FFFFFFFu - TOKENS_PER_CTA) return fail(MIORI_E_INVALID, "page_slots: too many tokens (%u)", tokens);
    if (held_after == held || held_after == fresh || taken_after == taken || cu == held || cu == fresh)
        return fail(MIORI_E_INVALID, "page_slots: every CTA reads the inputs, none may be an output too");
    const SlotArgs a = {held, fresh, table, pool, taken, slots, positions, cu, held_after, taken_after, requests, width, page, pool_size, tokens,
                        aligned16(slots) && aligned16(positions)};
    const uint32_t grid = tokens ? (tokens + TOKENS_PER_CTA - 1u) / TOKENS_PER_CTA : 1u;
    (void)flags;  // it reads nothing ahead of its wait: every launch may begin beside the one before (slots of a decode step 6.2 us a call without)
    const cudaError_t e = launch(page_slots_kernel, dim3(grid), dim3(SLOT_THREADS), 8u * (requests + 1u), (cudaStream_t)stream, true, a);
    return e == cudaSuccess ? MIORI_OK : cuda_fail(e, "page_slots launch");
}

MIORI_API int miori_rope_kv(const void* qkv, int64_t qkv_row, const uint64_t* turns, const int32_t* axes, const int32_t* positions,
                            const int32_t* slots, const void* gamma_q, const void* gamma_k, float eps, void* q, void* k_cache, void* v_cache,
                            const int64_t* cache_strides, uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t rotary,
                            uint32_t num_axes, uint32_t pages, uint32_t page, uint32_t flags, void* stream) {
    using namespace miori_b200::pages;
    if (!qkv || !turns || !positions || !slots || !q || !k_cache || !v_cache || !cache_strides) return fail(MIORI_E_INVALID, "rope_kv: null pointer");
    if (tokens == 0 || heads == 0 || kv_heads == 0 || pages == 0 || page == 0)
        return fail(MIORI_E_INVALID, "rope_kv: empty shape (tokens=%u heads=%u kv_heads=%u pages=%u page=%u)", tokens, heads, kv_heads, pages, page);
    if (dim != 64 && dim != 128) return fail(MIORI_E_INVALID, "rope_kv: heads of 64 or 128, got %u", dim);
    if (heads > 4096 || kv_heads > 4096) return fail(MIORI_E_INVALID, "rope_kv: at most 4096 heads");
    if (rotary == 0 || rotary > dim || rotary % 16) return fail(MIORI_E_INVALID, "rope_kv: rotary dimensions are a multiple of 16 up to the head's, got %u of %u", rotary, dim);
    if (num_axes == 0 || num_axes > 4) return fail(MIORI_E_INVALID, "rope_kv: one to four axes, got %u", num_axes);
    if ((uint64_t)pages * page > 0x7FFFFFFFull) return fail(MIORI_E_INVALID, "rope_kv: a cache of 2^31 slots or more");
    if (!aligned16(qkv) || !aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(gamma_q) || !aligned16(gamma_k))
        return fail(MIORI_E_INVALID, "rope_kv: pointers must be 16-byte aligned");
    if (qkv_row % 8 || qkv_row < (int64_t)(heads + 2 * kv_heads) * dim) return fail(MIORI_E_INVALID, "rope_kv: rows of qkv are a multiple of 8 elements apart, none overlaps the next");
    for (int i = 0; i < 6; ++i)
        if (cache_strides[i] % 8) return fail(MIORI_E_INVALID, "rope_kv: strides of the caches must be multiples of 8 elements");
    RopeArgs a = {qkv, turns, axes, positions, slots, (const uint16_t*)gamma_q, (const uint16_t*)gamma_k, (uint16_t*)q, (uint16_t*)k_cache, (uint16_t*)v_cache,
                  qkv_row, cache_strides[0], cache_strides[1], cache_strides[2], cache_strides[3], cache_strides[4], cache_strides[5],
                  tokens, heads, kv_heads, rotary, num_axes, page, pages, 1u, eps, flags & MIORI_LAUNCH_PDL};
    // as many warps a token as keep 16 warps an SM busy
    const uint32_t heads_a_warp = 512u / dim, most = (heads + 2u * kv_heads + heads_a_warp - 1u) / heads_a_warp;
    const uint32_t wanted = (16u * (uint32_t)sm_count() + tokens - 1u) / tokens;
    a.parts = wanted < most ? wanted : most;
    const uint64_t warps = (uint64_t)tokens * a.parts;
    if (warps > 0xFFFFFFF0ull) return fail(MIORI_E_INVALID, "rope_kv: too many tokens (%u)", tokens);
    const dim3 grid((uint32_t)((warps + ROPE_THREADS / 32 - 1) / (ROPE_THREADS / 32)));
    const bool fp32 = (flags & MIORI_ROPE_F32) != 0, adjacent = (flags & MIORI_ROPE_ADJACENT) != 0;
    void (*kernel)(const RopeArgs);
    if (dim == 128) kernel = fp32 ? (adjacent ? rope_kv_kernel<128, true, true> : rope_kv_kernel<128, true, false>)
                                  : (adjacent ? rope_kv_kernel<128, false, true> : rope_kv_kernel<128, false, false>);
    else kernel = fp32 ? (adjacent ? rope_kv_kernel<64, true, true> : rope_kv_kernel<64, true, false>)
                       : (adjacent ? rope_kv_kernel<64, false, true> : rope_kv_kernel<64, false, false>);
    const cudaError_t e = launch(kernel, grid, dim3(ROPE_THREADS), 0, (cudaStream_t)stream, true, a);
    return e == cudaSuccess ? MIORI_OK : cuda_fail(e, "rope_kv launch");
}
