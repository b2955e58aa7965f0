// Attention of a few new tokens per request over the paged cache: decoding, and drafted tokens that are checked together.
//
// HBM-bound: every cached key and value is read once, 4 * D bytes a position and key head, for 4 * D * rows operations.  What
// counts is bytes in flight and an even share for every SM.
//
// * An item has up to 8, 16 or 32 rows (NT = 1, 2, 4 columns of eight).  Keys are the MMA's 16 rows and the item's rows its 8 columns:
//   S^T = K Q^T, then O^T = V^T P^T, so that with up to eight rows no half of an MMA is padding.  K is the A operand as it lies
//   in shared memory (ldmatrix), V through ldmatrix.trans; P^T takes one movmatrix per eight keys and columns.
// * A warp owns 16 of a unit's 128 keys, with a ring of its own (STAGES tiles of 16 keys and values), its own running maximum, sum
//   and O: no barrier in the main loop.  cp.async fills the ring, so a page may be as short as 8 positions and strides are
//   free; what lies beyond the length, or in a page that the cache does not have, arrives as zeros, never as what the page or the
//   ring held before.
// * A CTA's share may begin and end inside an item.  The warps' parts meet in shared memory at the end of an item; an item
//   shared by several CTAs meets in the workspace: the CTA that arrives last adds the parts up in the order of the keys, so a
//   result does not depend on which one that is.
// * P is rounded to bf16 for the second product, as the values are, since an MMA has one type for both; l sums the rounded p, so that
//   O / l is a mean of values whatever their weights are off by: a key that outweighs all others is weighed by one, although its p
//   is not one with a maximum that stands still.
//
// 32 requests of up to 32768 positions (719 MB), 16 heads of 128 over 4: 124 us on changing inputs, 5.8 TB/s (a copy reaches 6.56; DRAM reads
// are 1.001 of the bytes), 120 in a graph.  One request of 1000: 8.2 and 8.0 us, latency.  9 requests of 5 drafts and up to 5000 positions, 32
// heads of 64 over 8: 22.1 and 20.6 us, bound by instructions: 32 columns of which 20 are rows.  32 requests of 8000, one token, in a graph:
// 32 heads of 64 over 8 105.6 us (5.0 TB/s); of 4000, 16 heads that share nothing, of 64 106.8 (4.9), of 128 172 (6.1).
#pragma once
#include "attention.cuh"

namespace miori_b200 {
namespace attention {

constexpr uint32_t DECODE_ITEM_COST = 384;  // an item's begin and end, in positions: 32 requests and drafts 119.6, 20.7 us (256 118.8, 21.7; 640 121.5, 20.4)
constexpr int DECODE_WARPS = 8, DECODE_THREADS = DECODE_WARPS * 32, TILE = 16, UNIT = DECODE_WARPS * TILE;

template <int D, int NT>
struct DecodeCfg {
    static constexpr int ROWS = 8 * NT;
    static constexpr int STAGES = D == 128 ? 3 : 6;
    static constexpr int TILE_BYTES = TILE * D * 2;                       // of keys, or of values
    static constexpr int RING = DECODE_WARPS * STAGES * 2 * TILE_BYTES;
    static constexpr int MEET = DECODE_WARPS * 8 * D * 4;                 // eight rows of every warp's O
    static constexpr int SMEM = RING + MEET;
    static constexpr int PART_FLOATS = ROWS * (D + 2);                    // O, then m and l of each row
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
    const uint32_t bytes = there ? 16u : 0u;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// First key of the edge tiles of a request: those with keys that its first token does not see.
__device__ __forceinline__ uint32_t first_edge_key(const Args& a, const Request& x) {
    const uint32_t all_see = seen(a, x, 0u);
    return all_see < x.len ? all_see / TILE * TILE : 0xFFFFFFFFu;
}

// Where a share stands: an item (request, block of its tokens, key head), a unit of its keys, and where the share leaves the item.
// An item costs ITEM_COST + its positions; unit k belongs to the share that holds start + ITEM_COST - 1 + UNIT k (the dealing
// of attention_prompt.cuh, with a request's length for every one of its items).
struct Place {
    Request x;
    uint32_t r, block, blocks, head, units, unit, stop;
    uint64_t start;
    bool more;
    __device__ __forceinline__ uint64_t mark() const { return start + DECODE_ITEM_COST - 1u; }
    __device__ __forceinline__ uint64_t last_mark() const { return mark() + (uint64_t)(units - 1u) * UNIT; }
    __device__ __forceinline__ void measure(uint32_t per_block) {
        blocks = (x.n + per_block - 1u) / per_block;
        units = max((x.len + UNIT - 1u) / UNIT, 1u);
    }
    __device__ __forceinline__ uint32_t units_below(uint64_t at) const {
        return at <= mark() ? 0u : (uint32_t)min((at - mark() + UNIT - 1u) / UNIT, (uint64_t)units);
    }
    __device__ __forceinline__ void cut(uint64_t begin, uint64_t end, bool split) {
        unit = units_below(begin), stop = units_below(end);
        if (!split) stop = unit == 0u && stop > 0u ? units : unit;
    }
    __device__ __forceinline__ void next(const Args& a, uint32_t per_block, uint64_t begin, uint64_t end) {  // item with units in the share
        do {
            start += DECODE_ITEM_COST + x.len;
            if (start >= end) {
                more = false;
                return;
            }
            if (++head == a.kv_heads) {
                head = 0u;
                if (++block == blocks) {
                    block = 0u;
                    do {
                        x = request<true>(a, ++r);
                        measure(per_block);
                    } while (blocks == 0u && r + 1u < a.requests);
                }
            }
            cut(begin, end, a.parts != nullptr);
        } while (unit >= stop);
    }
};

// Values that are not finite and were left out of the products, added for a row that sees them: four dimensions from d on.
__device__ __noinline__ float4 add_left_out(float4 v, const Args& a, const Place& at, uint32_t token, uint32_t d) {
    float e[4] = {v.x, v.y, v.z, v.w};
    const uint32_t stop = seen(a, at.x, token);
    for (uint32_t j = first_edge_key(a, at.x); j < stop; ++j) {
        const uint32_t pg = (uint32_t)ld_fresh(a.table + (size_t)at.r * a.width + (j >> a.page_shift));
        if (pg >= a.pages) continue;
        const uint16_t* vp = a.v + (int64_t)pg * a.v_page + (int64_t)at.head * a.v_head + (int64_t)(j & ((1u << a.page_shift) - 1u)) * a.v_slot + d;
        for (int c = 0; c < 4; ++c) {
            const float x = bf16_bits_to_float(ld_fresh(vp + c));
            if (!(fabsf(x) < INFINITY)) e[c] += x;
        }
    }
    return make_float4(e[0], e[1], e[2], e[3]);
}

template <int D, int NT>
__global__ void __launch_bounds__(DECODE_THREADS, 1) attention_decode_kernel(const __grid_constant__ Args a) {
    using C = DecodeCfg<D, NT>;
    constexpr int KS = D / 16;        // k steps of the first product, 16-row tiles of the second
    constexpr uint32_t CH = D / 8;    // 16-byte pieces of a row
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float2 meet_ml[DECODE_WARPS][C::ROWS];
    __shared__ uint32_t dirty, last_one;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    pdl_launch_dependents();
    pdl_wait_prior();
    const uint32_t group = a.group, per_block = C::ROWS / group;
    const bool split = a.parts != nullptr;

    // this CTA's share and where it begins
    Request mine = {}, other;
    auto cost_of = [&](uint32_t r, Request& x) -> uint64_t {
        if (r >= a.requests) return 0;
        x = request<true>(a, r);
        return (uint64_t)((x.n + per_block - 1u) / per_block) * (DECODE_ITEM_COST + x.len) * a.kv_heads;
    };
    const uint64_t cost = cost_of(lane, mine);
    uint64_t total = warp_sum(cost);
    for (uint32_t r0 = 32u; r0 < a.requests; r0 += 32u) total += warp_sum(cost_of(r0 + lane, other));
    const Shares shares(total, gridDim.x, UNIT);
    const uint64_t begin = shares.begin(blockIdx.x), end = shares.begin(blockIdx.x + 1u);
    if (begin == end) return;
    Place at;
    auto find = [&](auto cost_here, auto at_unit) {  // in 32 bits where the whole launch costs less than 2^32
        using U = decltype(at_unit);
        U before = 0;
        for (uint32_t r0 = 0;; r0 += 32u) {
            if (r0) cost_here = (U)cost_of(r0 + lane, mine);
            const U sum = a.requests == 1u ? cost_here : warp_prefix_sum(cost_here);
            const uint32_t past = __ballot_sync(0xFFFFFFFFu, r0 + lane < a.requests && before + sum > at_unit);
            if (past || r0 + 32u >= a.requests) {
                const uint32_t l = past ? __ffs(past) - 1u : 0u;  // there always is one
                before += __shfl_sync(0xFFFFFFFFu, sum - cost_here, l);
                at.r = r0 + l;
                at.x.q0 = __shfl_sync(0xFFFFFFFFu, mine.q0, l), at.x.n = __shfl_sync(0xFFFFFFFFu, mine.n, l);
                at.x.k0 = 0u, at.x.len = __shfl_sync(0xFFFFFFFFu, mine.len, l), at.x.before = __shfl_sync(0xFFFFFFFFu, mine.before, l);
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, sum, 31);
        }
        const U per_head = DECODE_ITEM_COST + at.x.len;
        const uint32_t item = small_quotient((U)(at_unit - before), per_head);
        at.start = before + item * per_head;
        at.block = item / a.kv_heads, at.head = item % a.kv_heads;
    };
    if (total >> 32) find(cost, begin);
    else find((uint32_t)cost, (uint32_t)begin);
    at.measure(per_block);
    at.more = true;
    at.cut(begin, end, split);
    if (at.unit >= at.stop) at.next(a, per_block, begin, end);
    if (!at.more) return;

    // ---- the ring: this warp's 16 keys of a unit, rows of D swizzled by 16-byte pieces
    const uint32_t ring = smem_addr(smem) + warp * (C::STAGES * 2 * C::TILE_BYTES);
    auto piece = [](uint32_t row, uint32_t c) { return row * (D * 2u) + ((c ^ (row & 7u)) << 4); };
    uint32_t absent = 0;  // of a stage's keys, a bit for each eight: no page
    auto fill = [&](const Place& p, uint32_t stage) {
        const uint32_t key0 = p.unit * UNIT + warp * TILE;
        const uint32_t kdst = ring + stage * 2u * C::TILE_BYTES, vdst = kdst + C::TILE_BYTES;
        const uint32_t mask = (1u << a.page_shift) - 1u;
        uint32_t pg[2];
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {  // a page holds a multiple of eight positions
            const uint32_t first = key0 + 8u * half;
            pg[half] = first < p.x.len ? (uint32_t)ld_fresh(a.table + (size_t)p.r * a.width + (first >> a.page_shift)) : a.pages;
        }
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
            const uint32_t first = key0 + 8u * half, in = first & mask;
            const bool known = pg[half] < a.pages;
            const uint32_t bit = 1u << (2u * stage + half);
            absent = known ? absent & ~bit : absent | bit;
            const uint32_t count = known ? p.x.len - first : 0u, number = known ? pg[half] : 0u;
            const uint32_t row0 = lane / CH, c = lane % CH;
            const uint16_t* kp = a.k + (int64_t)number * a.k_page + (int64_t)p.head * a.k_head + (int64_t)in * a.k_slot + 8u * c;
            const uint16_t* vp = a.v + (int64_t)number * a.v_page + (int64_t)p.head * a.v_head + (int64_t)in * a.v_slot + 8u * c;
#pragma unroll
            for (uint32_t i = 0; i < 8u * CH / 32u; ++i) {
                const uint32_t row = row0 + i * (32u / CH);
                const bool there = row < count;
                const uint32_t to = piece(8u * half + row, c);
                cp_async16(kdst + to, kp + (there ? (int64_t)row * a.k_slot : 0), there);
                cp_async16(vdst + to, vp + (there ? (int64_t)row * a.v_slot : 0), there);
            }
        }
    };
    uint32_t qf[NT][KS][2];
    float o[NT][KS][4], m[NT][2], l[NT][2];
    uint32_t sees[NT][2];  // positions that the lane's columns see
    uint32_t rows;
    auto begin_item = [&] {
        rows = min(per_block, at.x.n - at.block * per_block) * group;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t row = 8u * n + lane / 4u, i = at.block * per_block + row / group;
            const uint16_t* qp = a.q + (int64_t)(at.x.q0 + i) * a.q_token + (int64_t)(at.head * group + row % group) * a.q_head + 2u * (lane & 3u);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                qf[n][k][0] = row < rows ? ld_fresh(reinterpret_cast<const uint32_t*>(qp + 16 * k)) : 0u;
                qf[n][k][1] = row < rows ? ld_fresh(reinterpret_cast<const uint32_t*>(qp + 16 * k + 8)) : 0u;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][k][j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t col = 8u * n + 2u * (lane & 3u) + j;
                sees[n][j] = col < rows ? seen(a, at.x, at.block * per_block + col / group) : 0u;
                m[n][j] = -INFINITY, l[n][j] = 0.0f;
            }
        }
    };
    begin_item();  // its loads travel with the first keys'
    Place ahead = at;
    auto fill_next = [&](uint32_t stage) {
        if (ahead.more) {
            fill(ahead, stage);
            if (++ahead.unit == ahead.stop) ahead.next(a, per_block, begin, end);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (uint32_t s = 0; s < C::STAGES - 1u; ++s) fill_next(s);

    uint32_t stage = 0;
    if (threadIdx.x == 0) dirty = 0u;
    __syncthreads();
#pragma unroll 1
    do {
        // keys that some rows see and others do not: 0 * inf must not reach those that do not
        const uint32_t edge = first_edge_key(a, at.x);
        const bool whole = at.unit == 0u && at.stop == at.units;
#pragma unroll 1
        for (; at.unit < at.stop; ++at.unit) {
            asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
            __syncwarp();
            fill_next(stage == 0u ? C::STAGES - 1u : stage - 1u);  // the place read last is free
            const uint32_t kb = ring + stage * 2u * C::TILE_BYTES, vb = kb + C::TILE_BYTES, gone = absent >> (2u * stage) & 3u;
            stage = stage + 1u == C::STAGES ? 0u : stage + 1u;
            const uint32_t key0 = at.unit * UNIT + warp * TILE;
            if (key0 >= at.x.len) continue;
            if (key0 >= edge) {
                bool zeroed = false;
#pragma unroll 1
                for (uint32_t e = lane; e < TILE * CH; e += 32u) {
                    uint32_t w[4], z[4];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(vb + 16u * e) : "memory");
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[i] = finite_or_zero(w[i]), zeroed |= z[i] != w[i];
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(vb + 16u * e), "r"(z[0]), "r"(z[1]), "r"(z[2]), "r"(z[3]) : "memory");
                }
                if (zeroed) dirty = 1u;
                __syncwarp();
            }
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t f[4];
                ldmatrix4(f, kb + piece(lane & 15u, 2u * k + (lane >> 4)));
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816(s[n], f, qf[n][k][0], qf[n][k][1]);
            }
            if (gone) {  // no page: nobody sees these keys
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[n][j] = gone >> (j / 2) & 1u ? -INFINITY : s[n][j];
            }
            // The running maximum moves only when a score exceeds it by 2^8 (p grows up to 256 then): most tiles need neither the
            // maximum over the lanes nor a rescaled O.
            uint32_t pf[NT][2];
            const uint32_t key = key0 + lane / 4u;
            bool higher = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[n][j] = key + (j >= 2 ? 8u : 0u) < sees[n][j & 1] ? s[n][j] * a.scale_log2 : -INFINITY;
                    higher |= s[n][j] > m[n][j & 1] + 8.0f;
                }
            if (__any_sync(0xFFFFFFFFu, higher)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float top = fmaxf(m[n][j], fmaxf(s[n][j], s[n][j + 2]));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                        const float keep = top == -INFINITY ? 1.0f : exp2_fast(m[n][j] - top);
                        m[n][j] = top;
                        l[n][j] *= keep;
#pragma unroll
                        for (int k = 0; k < KS; ++k) o[n][k][j] *= keep, o[n][k][j + 2] *= keep;
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[n][j] = exp2_fast(s[n][j] - (m[n][j & 1] == -INFINITY ? 0.0f : m[n][j & 1]));
                const uint32_t low = pack_bf16(s[n][0], s[n][1]), high = pack_bf16(s[n][2], s[n][3]);
                add_bf16(l[n][0], l[n][1], low), add_bf16(l[n][0], l[n][1], high);
                pf[n][0] = movmatrix(low), pf[n][1] = movmatrix(high);
            }
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t f[4];
                // row of the stored tile: key; a quarter of the lanes each (keys 0-7 and 8-15) x (first and second eight dimensions)
                ldmatrix4_trans(f, vb + piece((lane & 7u) + 8u * (lane >> 4), 2u * k + ((lane >> 3) & 1u)));
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816(o[n][k], f, pf[n][0], pf[n][1]);
            }
        }

        // ---- the warps' parts meet in shared memory, eight rows at a time; an item of several CTAs goes on to the workspace
        const uint32_t first = whole ? blockIdx.x : shares.of(at.mark()), last = whole ? blockIdx.x : shares.of(at.last_mark());
        // two parts a CTA: of the item that its share begins in and of the one that it ends in
        float* const part = a.parts + (size_t)(2u * blockIdx.x + (first == blockIdx.x ? 1u : 0u)) * C::PART_FLOATS;
        float* const sum_o = reinterpret_cast<float*>(smem + C::RING);  // [warp][8][D], swizzled so that no two lanes of a store share a bank
        auto in_row = [](uint32_t row, uint32_t d) { return row * D + (d ^ ((row >> 1 & 3u) << 3)); };
        auto store = [&](uint32_t row, uint32_t d, float4 v, float l_all) {
            const float inv = l_all > 0.0f ? 1.0f / l_all : l_all == 0.0f ? 0.0f : l_all;  // no key: zeros; NaN stays
            const uint32_t i = at.block * per_block + row / group;
            v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            if (dirty) v = add_left_out(v, a, at, i, d);
            *reinterpret_cast<uint2*>(a.out + (int64_t)(at.x.q0 + i) * a.o_token + (int64_t)(at.head * group + row % group) * a.o_head + d) =
                make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        };
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float sum = l[n][j];
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
                if (lane < 4u) meet_ml[warp][8 * n + 2 * lane + j] = make_float2(m[n][j], sum);
            }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n > 0) {
                if (rows <= 8u * n) break;
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j)  // accumulator: row of the MMA = dimension, column = row of the item
                    sum_o[in_row(warp * 8u + 2u * (lane & 3u) + (j & 1u), 16u * k + lane / 4u + (j >= 2 ? 8u : 0u))] = o[n][k][j];
            __syncthreads();
#pragma unroll 1
            for (uint32_t e = threadIdx.x; e < 8u * D / 4u; e += DECODE_THREADS) {
                const uint32_t r8 = e / (D / 4u), row = 8u * n + r8, d = e % (D / 4u) * 4u;
                if (row >= rows) break;
                float top = -INFINITY, sum = 0.0f;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < DECODE_WARPS; ++w) top = fmaxf(top, meet_ml[w][row].x);
                const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
                for (int w = 0; w < DECODE_WARPS; ++w) {
                    const float2 ml = meet_ml[w][row];
                    const float f = exp2_fast(ml.x - from);
                    const float4 x = *reinterpret_cast<const float4*>(sum_o + in_row(w * 8u + r8, d));
                    sum = fmaf(ml.y, f, sum);
                    v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
                }
                if (whole) {
                    store(row, d, v, sum);
                } else {
                    *reinterpret_cast<float4*>(part + row * D + d) = v;
                    if (d == 0u) *reinterpret_cast<float2*>(part + C::ROWS * D + 2u * row) = make_float2(top, sum);
                }
            }
        }
        if (!whole) {
            __syncthreads();
            if (threadIdx.x == 0) {  // one arrival for the CTA; the upper half counts those that left values out
                const uint32_t arrival = dirty ? 0x10001u : 1u;
                uint32_t before;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(before) : "l"(a.counters + first), "r"(arrival) : "memory");
                last_one = (before & 0xFFFFu) == last - first;
                dirty = (before + arrival) >> 16;
                if (last_one) a.counters[first] = 0u;
            }
            __syncthreads();
            if (last_one) {
                constexpr uint32_t AT_ONCE = 8;  // parts whose loads travel together
#pragma unroll 1
                for (uint32_t e = threadIdx.x; e < rows * (D / 4u); e += DECODE_THREADS) {
                    const uint32_t row = e / (D / 4u), d = e % (D / 4u) * 4u;
                    float m_all = -INFINITY, l_all = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
                    for (uint32_t c0 = first; c0 <= last; c0 += AT_ONCE) {
                        float2 ml[AT_ONCE];
                        float4 x[AT_ONCE];
#pragma unroll
                        for (uint32_t i = 0; i < AT_ONCE; ++i) {  // beyond the last one: the last one again, with no weight
                            const uint32_t c = min(c0 + i, last);
                            const float* from_c = a.parts + (size_t)(2u * c + (c == first ? 1u : 0u)) * C::PART_FLOATS;
                            ml[i] = ld_fresh(reinterpret_cast<const float2*>(from_c + C::ROWS * D + 2u * row));
                            x[i] = ld_fresh(reinterpret_cast<const float4*>(from_c + row * D + d));
                        }
                        float top = m_all;
#pragma unroll
                        for (uint32_t i = 0; i < AT_ONCE; ++i) top = fmaxf(top, ml[i].x);
                        const float from = top == -INFINITY ? 0.0f : top, keep = exp2_fast(m_all - from);
                        m_all = top;
                        l_all *= keep, v.x *= keep, v.y *= keep, v.z *= keep, v.w *= keep;
#pragma unroll
                        for (uint32_t i = 0; i < AT_ONCE; ++i) {
                            if (c0 + i > last) break;
                            const float f = exp2_fast(ml[i].x - from);
                            l_all = fmaf(ml[i].y, f, l_all);
                            v.x = fmaf(x[i].x, f, v.x), v.y = fmaf(x[i].y, f, v.y), v.z = fmaf(x[i].z, f, v.z), v.w = fmaf(x[i].w, f, v.w);
                        }
                    }
                    store(row, d, v, l_all);
                }
            }
        }
        at.next(a, per_block, begin, end);
        if (at.more) begin_item();
        __syncthreads();  // the meeting's memory is free again
        if (threadIdx.x == 0) dirty = 0u;
        __syncthreads();
    } while (at.more);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

}  // namespace attention
}  // namespace miori_b200
