// Attention of a few new tokens per request over the paged cache: decoding, and drafted tokens that are checked together.
//
// HBM-bound: every cached key and value is read once, 4 * D bytes a position and key head, for 4 * D * rows operations.  What
// counts is bytes in flight and an even share for every SM.
//
// * An item has up to 8 or 16 rows (NT = 1, 2 columns of eight).  Keys are the MMA's 16 rows and the item's rows its 8 columns:
//   S^T = K Q^T, then O^T = V^T P^T, so that with up to eight rows no half of an MMA is padding.  K is the A operand as it lies
//   in shared memory (ldmatrix), V through ldmatrix.trans; P^T takes one movmatrix per eight keys and columns.
// * A warp owns 16 of a unit's 128 keys, with a ring of its own (STAGES tiles of 16 keys and values), its own running maximum, sum
//   and O: no barrier in the main loop.  cp.async fills the ring, so a page may be as short as 8 positions and strides are
//   free; what lies beyond the length arrives as zeros, never as what the page held before.
// * A CTA's share may begin and end inside an item.  The warps' parts meet in shared memory at the end of an item; an item
//   shared by several CTAs meets in the workspace: the CTA that arrives last adds the parts up in the order of the keys, so a
//   result does not depend on which one that is.
// * P is rounded to bf16 for the second product, as the values are; l sums the unrounded p.
#pragma once
#include "attention.cuh"

namespace miori_b200 {
namespace attention {

constexpr int DECODE_WARPS = 8, DECODE_THREADS = DECODE_WARPS * 32, TILE = 16, UNIT = DECODE_WARPS * TILE;

template <int D, int NT>
struct DecodeCfg {
    static constexpr int ROWS = 8 * NT;
    static constexpr int STAGES = D == 128 ? 3 : 6;
    static constexpr int TILE_BYTES = TILE * D * 2;                       // of keys, or of values
    static constexpr int RING = DECODE_WARPS * STAGES * 2 * TILE_BYTES;
    static constexpr int MEET = DECODE_WARPS * 8 * D * 4;                 // eight rows of every warp's O
    static constexpr int SMEM = RING + MEET;
    static constexpr int PART_FLOATS = ROWS * (D + 2) + 4;               // O, m, l and a flag; 16-byte multiple
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

// Where a share stands: an item (request, block of its tokens, key head) and a unit of its keys.
struct Place {
    Request x;
    uint32_t r, block, head, unit, units, blocks;
    __device__ __forceinline__ void enter(const Args& a, uint32_t request_id, uint32_t per_block) {
        r = request_id;
        x = request<true>(a, r);
        blocks = (x.n + per_block - 1u) / per_block;
        units = max((x.len + UNIT - 1u) / UNIT, 1u);
    }
    __device__ __forceinline__ bool next(const Args& a, uint32_t per_block) {  // true: another item now
        if (++unit < units) return false;
        unit = 0u;
        if (++head == a.kv_heads) {
            head = 0u;
            if (++block >= blocks) {
                block = 0u;
                do enter(a, r + 1u, per_block);
                while (blocks == 0u && r + 1u < a.requests);
            }
        }
        return true;
    }
};

template <int D, int NT>
__global__ void __launch_bounds__(DECODE_THREADS, 1) attention_decode_kernel(const Args a) {
    using C = DecodeCfg<D, NT>;
    constexpr int KS = D / 16;        // k steps of the first product, 16-row tiles of the second
    constexpr uint32_t CH = D / 8;    // 16-byte pieces of a row
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float meet_m[DECODE_WARPS][16], meet_l[DECODE_WARPS][16];
    __shared__ uint32_t dirty, last_one;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    pdl_launch_dependents();
    pdl_wait_prior();
    const uint32_t group = a.group, per_block = C::ROWS / group;

    // this CTA's share
    uint64_t total = 0;
    auto units_of = [&](uint32_t r) -> uint64_t {
        const Request x = request<true>(a, r);
        return (uint64_t)((x.n + per_block - 1u) / per_block) * max((x.len + UNIT - 1u) / UNIT, 1u) * a.kv_heads;
    };
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 32u) {
        uint64_t w = r0 + lane < a.requests ? units_of(r0 + lane) : 0u;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
        total += w;
    }
    const uint32_t shares = shares_of(total, gridDim.x);
    if (blockIdx.x >= shares) return;
    uint64_t item0;  // first unit of the item at hand
    auto locate = [&](uint64_t unit) {
        Place p;
        uint64_t before = 0;
        uint32_t found = 0;
        for (uint32_t r0 = 0; r0 < a.requests; r0 += 32u) {
            const uint64_t w = r0 + lane < a.requests ? units_of(r0 + lane) : 0u;
            uint64_t sum = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
                if (lane >= (uint32_t)o) sum += y;
            }
            const uint32_t past = __ballot_sync(0xFFFFFFFFu, before + sum > unit);
            if (past) {
                const uint32_t first = __ffs(past) - 1u;
                before += __shfl_sync(0xFFFFFFFFu, sum - w, first);
                found = r0 + first;
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, sum, 31);
        }
        p.enter(a, found, per_block);
        const uint64_t in = unit - before, per_head = p.units, per_tokens = per_head * a.kv_heads;
        p.block = (uint32_t)(in / per_tokens);
        p.head = (uint32_t)(in % per_tokens / per_head);
        p.unit = (uint32_t)(in % per_head);
        return p;
    };
    uint64_t begin = share_begin(total, blockIdx.x, shares), end = share_begin(total, blockIdx.x + 1u, shares);
    Place at = locate(begin);
    if (!a.parts) {  // items stay whole: those that begin in the share
        if (end < total) {
            const Place p = locate(end);
            if (p.unit) end += p.units - p.unit;
        }
        if (at.unit) {
            begin += at.units - at.unit;
            if (begin >= end) return;
            at.unit = at.units - 1u;
            at.next(a, per_block);
        }
    }
    item0 = begin - at.unit;

    // ---- the ring: this warp's 16 keys of a unit, rows of D swizzled by 16-byte pieces
    const uint32_t ring = smem_addr(smem) + warp * (C::STAGES * 2 * C::TILE_BYTES);
    auto piece = [](uint32_t row, uint32_t c) { return row * (D * 2u) + ((c ^ (row & 7u)) << 4); };
    auto fill = [&](const Place& p, uint32_t stage) {
        const uint32_t key0 = p.unit * UNIT + warp * TILE;
        const uint32_t kdst = ring + stage * 2u * C::TILE_BYTES, vdst = kdst + C::TILE_BYTES;
        const uint32_t mask = (1u << a.page_shift) - 1u;
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {  // a page holds a multiple of eight positions
            const uint32_t first = key0 + 8u * half;
            const uint32_t count = p.x.len > first ? p.x.len - first : 0u;
            uint32_t pg = count ? (uint32_t)ld_fresh(a.table + (size_t)p.r * a.width + (first >> a.page_shift)) : 0u;
            const bool known = pg < a.pages;
            if (!known) pg = 0u;
            const uint32_t in = first & mask;
            const uint16_t* kp = a.k + (int64_t)pg * a.k_page + (int64_t)p.head * a.k_head + (int64_t)in * a.k_slot;
            const uint16_t* vp = a.v + (int64_t)pg * a.v_page + (int64_t)p.head * a.v_head + (int64_t)in * a.v_slot;
#pragma unroll
            for (uint32_t i = 0; i < 8u * CH / 32u; ++i) {
                const uint32_t e = i * 32u + lane, row = e / CH, c = e % CH;
                const bool there = known && row < count;
                const uint32_t to = piece(8u * half + row, c);
                const int64_t ks = there ? (int64_t)row * a.k_slot + 8u * c : 0, vs = there ? (int64_t)row * a.v_slot + 8u * c : 0;
                cp_async16(kdst + to, kp + ks, there);
                cp_async16(vdst + to, vp + vs, there);
            }
        }
    };
    Place ahead = at;
    uint64_t filled = begin;
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) {
        if (filled < end) {
            fill(ahead, (uint32_t)s);
            if (++filled < end) ahead.next(a, per_block);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    uint32_t qf[NT][KS][2];
    float o[NT][KS][4], m[NT][2], l[NT][2];
    uint32_t sees[NT][2];  // positions that the lane's columns see
    bool zeroed = false;
    auto row_token = [&](uint32_t row) { return at.block * per_block + row / group; };
    auto begin_item = [&]() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t row = 8u * n + lane / 4u, i = row_token(row);
            const bool there = row < per_block * group && i < at.x.n;
            const uint16_t* qp = a.q + (int64_t)(at.x.q0 + (there ? i : 0u)) * a.q_token + (int64_t)(at.head * group + (there ? row % group : 0u)) * a.q_head;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint32_t c = 16u * k + 2u * (lane & 3u);
                qf[n][k][0] = there ? ld_fresh(reinterpret_cast<const uint32_t*>(qp + c)) : 0u;
                qf[n][k][1] = there ? ld_fresh(reinterpret_cast<const uint32_t*>(qp + c + 8u)) : 0u;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][k][j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t col = 8u * n + 2u * (lane & 3u) + j, ti = row_token(col);
                sees[n][j] = col < per_block * group && ti < at.x.n ? seen(a, at.x, ti) : 0u;
                m[n][j] = -INFINITY, l[n][j] = 0.0f;
            }
        }
        zeroed = false;
    };
    begin_item();
    if (threadIdx.x == 0) dirty = 0u;
    __syncthreads();

    uint64_t u = begin;
    uint32_t stage = 0;
    for (;;) {
        asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
        __syncwarp();
        // the stage read last is free: fill it before working on this one
        if (filled < end) {
            fill(ahead, (stage + C::STAGES - 1u) % C::STAGES);
            if (++filled < end) ahead.next(a, per_block);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");

        const uint32_t kb = ring + stage * 2u * C::TILE_BYTES, vb = kb + C::TILE_BYTES;
        const uint32_t key0 = at.unit * UNIT + warp * TILE;
        if (key0 < at.x.len) {
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
            uint32_t pf[NT][2];
            const uint32_t key = key0 + lane / 4u;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float p[4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float t0 = key < sees[n][j] ? s[n][j] * a.scale_log2 : -INFINITY;
                    const float t1 = key + 8u < sees[n][j] ? s[n][j + 2] * a.scale_log2 : -INFINITY;
                    float top = fmaxf(t0, t1);
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                    const float now = fmaxf(m[n][j], top), from = now == -INFINITY ? 0.0f : now;
                    const float keep = exp2_fast(m[n][j] - from);
                    m[n][j] = now;
                    p[j] = exp2_fast(t0 - from), p[j + 2] = exp2_fast(t1 - from);
                    l[n][j] = l[n][j] * keep + p[j] + p[j + 2];
#pragma unroll
                    for (int k = 0; k < KS; ++k) o[n][k][j] *= keep, o[n][k][j + 2] *= keep;
                }
                pf[n][0] = movmatrix(pack_bf16(p[0], p[1]));
                pf[n][1] = movmatrix(pack_bf16(p[2], p[3]));
            }
            // keys that some rows see and others do not: 0 * inf must not reach those that do not
            const bool edge = a.causal && at.x.n > 1u && key0 + TILE + at.x.n > at.x.len + 1u;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t f[4];
                // row of the stored tile: key; a quarter of the lanes each (keys 0-7 and 8-15) x (first and second eight dimensions)
                ldmatrix4_trans(f, vb + piece((lane & 7u) + 8u * (lane >> 4), 2u * k + ((lane >> 3) & 1u)));
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t w = finite_or_zero(f[j]);
                        zeroed |= w != f[j];
                        f[j] = w;
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816(o[n][k], f, pf[n][0], pf[n][1]);
            }
        }
        stage = stage + 1u == C::STAGES ? 0u : stage + 1u;
        const bool item_ends = at.unit + 1u == at.units, share_ends = u + 1u == end;
        if (!item_ends && !share_ends) {
            ++u, ++at.unit;
            continue;
        }

        // ---- the warps' parts meet: columns m and l first, then O eight rows at a time
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float sum = l[n][j];
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
                if (lane < 4u) meet_m[warp][8 * n + 2 * lane + j] = m[n][j], meet_l[warp][8 * n + 2 * lane + j] = sum;
            }
        if (zeroed) dirty = 1u;
        const uint32_t rows = min(per_block, at.x.n - at.block * per_block) * group;
        const uint64_t item_end = item0 + at.units;
        const uint32_t first = share_of(total, item0, shares), last = share_of(total, item_end - 1u, shares);
        const bool whole = !a.parts || first == last;
        // workspace: two parts a CTA, of the item that its share begins in and of the one that it ends in
        float* const mine = whole ? nullptr : a.parts + (size_t)(2u * blockIdx.x + (first == blockIdx.x ? 1u : 0u)) * C::PART_FLOATS;
        float* const sum_o = reinterpret_cast<float*>(smem + C::RING);  // [warp][8][D]
        auto store = [&](uint32_t row, uint32_t d, float4 v) {
            const uint32_t i = at.block * per_block + row / group;
            uint16_t* to = a.out + (int64_t)(at.x.q0 + i) * a.o_token + (int64_t)(at.head * group + row % group) * a.o_head + d;
            if (dirty) {  // values that are not finite, left out above, reach the rows that see them
                float e[4] = {v.x, v.y, v.z, v.w};
                const uint32_t stop = seen(a, at.x, i);
                const uint32_t start = at.x.len > at.x.n + TILE ? at.x.len - at.x.n - TILE : 0u;
                // the first key that an edge tile may hold, rounded down to a tile
                for (uint32_t j = start / TILE * TILE; j < stop; ++j) {
                    const uint32_t tile0 = j / TILE * TILE;
                    if (tile0 + TILE + at.x.n <= at.x.len + 1u) continue;  // not an edge tile: nothing was left out
                    const uint32_t pg = (uint32_t)ld_fresh(a.table + (size_t)at.r * a.width + (j >> a.page_shift));
                    if (pg >= a.pages) continue;
                    const uint16_t* vp = a.v + (int64_t)pg * a.v_page + (int64_t)at.head * a.v_head + (int64_t)(j & ((1u << a.page_shift) - 1u)) * a.v_slot + d;
                    for (int c = 0; c < 4; ++c) {
                        const float x = bf16_bits_to_float(ld_fresh(vp + c));
                        if (!(fabsf(x) < INFINITY)) e[c] += x;
                    }
                }
                v = make_float4(e[0], e[1], e[2], e[3]);
            }
            *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        };
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n > 0) __syncthreads();
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // accumulator: row of the MMA = dimension, column = row of the item
                    const uint32_t d = 16u * k + lane / 4u + (j >= 2 ? 8u : 0u), row = 2u * (lane & 3u) + (j & 1u);
                    sum_o[(warp * 8u + row) * D + d] = o[n][k][j];
                }
            __syncthreads();
            for (uint32_t e = threadIdx.x; e < 8u * D / 4u; e += DECODE_THREADS) {
                const uint32_t r8 = e / (D / 4u), row = 8u * n + r8, d = e % (D / 4u) * 4u;
                if (row >= rows) continue;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < DECODE_WARPS; ++w) top = fmaxf(top, meet_m[w][row]);
                const float from = top == -INFINITY ? 0.0f : top;
                float sum = 0.0f;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < DECODE_WARPS; ++w) {
                    const float f = exp2_fast(meet_m[w][row] - from);
                    const float4 x = *reinterpret_cast<const float4*>(sum_o + (w * 8u + r8) * D + d);
                    sum = fmaf(meet_l[w][row], f, sum);
                    v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
                }
                if (whole) {
                    const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;  // no key: zeros; NaN stays
                    store(row, d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                } else {
                    __stcg(reinterpret_cast<float4*>(mine + row * D + d), v);
                    if (d == 0u) __stcg(mine + C::ROWS * D + 2u * row, top), __stcg(mine + C::ROWS * D + 2u * row + 1u, sum);
                }
            }
        }
        if (!whole) {
            if (threadIdx.x == 0) __stcg(mine + C::ROWS * (D + 2), dirty ? 1.0f : 0.0f);
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                last_one = atomicAdd(a.counters + first, 1u) == last - first;
                if (last_one) a.counters[first] = 0u;
                __threadfence();
            }
            __syncthreads();
            if (last_one) {
                auto part = [&](uint32_t c) { return a.parts + (size_t)(2u * c + (c == first ? 1u : 0u)) * C::PART_FLOATS; };
                if (threadIdx.x == 0) {
                    uint32_t any = 0u;
                    for (uint32_t c = first; c <= last; ++c) any |= __ldcg(part(c) + C::ROWS * (D + 2)) != 0.0f;
                    dirty = any;
                }
                __syncthreads();
                for (uint32_t e = threadIdx.x; e < rows * (D / 4u); e += DECODE_THREADS) {
                    const uint32_t row = e / (D / 4u), d = e % (D / 4u) * 4u;
                    float top = -INFINITY;
                    for (uint32_t c = first; c <= last; ++c) top = fmaxf(top, __ldcg(part(c) + C::ROWS * D + 2u * row));
                    const float from = top == -INFINITY ? 0.0f : top;
                    float sum = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                    for (uint32_t c = first; c <= last; ++c) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(part(c) + C::ROWS * D + 2u * row));
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(part(c) + row * D + d));
                        const float f = exp2_fast(ml.x - from);
                        sum = fmaf(ml.y, f, sum);
                        v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
                    }
                    const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
                    store(row, d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                }
            }
        }
        if (share_ends) break;
        __syncthreads();  // the meeting's memory is free again
        if (threadIdx.x == 0) dirty = 0u;
        ++u;
        item0 = u;
        at.next(a, per_block);
        begin_item();
        __syncthreads();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

}  // namespace attention
}  // namespace miori_b200
