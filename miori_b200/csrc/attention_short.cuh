// Attention of few packed tokens: short prompts, where a launch's own latency is most of its time.
//
// The prompt kernel spends 6 us on setting up (shares, tensor memory, descriptors, some 20 KB of cold code) before its first
// product; this one is mma.sync on plain copies and little code.  Which of the two takes a call: takes_short in attention.cu.
//
// * A CTA of four warps has a block of 64 rows (tokens x the heads that share a key head), 16 rows a warp, and goes over all of
//   their keys, 64 at a time, two tiles in shared memory by cp.async.  Q stays in registers as the A operand, K and V are B operands
//   (ldmatrix, ldmatrix.trans), and the scores' accumulators are the probabilities' A operand as they lie.
// * Blocks are dealt by the grid: (block, key head), the host's bound on the blocks being tokens / tokens-a-block + requests.
// * What a row must not see: rows past the end arrive as zeros, values that are not finite are zeroed in every tile that some row
//   does not see as a whole and added at the end for the rows that see them.  P is rounded to bf16,
//   l sums the rounded p: see attention_decode.cuh.
//
// Latency-bound: one prompt of 77 tokens 6.5 us (the prompt kernel 10.0), 32 of 32 7.4 (12.0), 16 heads of 128 over 4, in a graph.
#pragma once
#include "attention.cuh"
#include "attention_decode.cuh"

namespace miori_b200 {
namespace attention {

constexpr int SHORT_THREADS = 128, SHORT_ROWS = 64, SHORT_KEYS = 64;
template <int D>
struct ShortCfg {
    static constexpr int TILE_BYTES = SHORT_KEYS * D * 2;
    static constexpr int SMEM = 4 * TILE_BYTES;  // two tiles of keys, two of values
};

template <int D>
__global__ void __launch_bounds__(SHORT_THREADS) attention_short_kernel(const __grid_constant__ Args a) {
    using C = ShortCfg<D>;
    constexpr int KS = D / 16, NK = SHORT_KEYS / 8;
    constexpr uint32_t CH = D / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, head = blockIdx.y, group = a.group, per_block = SHORT_ROWS / group;
    pdl_launch_dependents();
    pdl_wait_prior();

    // the block: request and first token
    Request x = {};
    uint32_t block = blockIdx.x;
    bool found = false;
    for (uint32_t r0 = 0; r0 < a.requests && !found; r0 += 32u) {
        Request mine = {};
        if (r0 + lane < a.requests) mine = request<false>(a, r0 + lane);
        const uint32_t blocks = (mine.n + per_block - 1u) / per_block, sum = warp_prefix_sum(blocks);
        const uint32_t past = __ballot_sync(0xFFFFFFFFu, sum > block);
        if (past) {
            const uint32_t l = __ffs(past) - 1u;
            block -= __shfl_sync(0xFFFFFFFFu, sum - blocks, l);
            x.q0 = __shfl_sync(0xFFFFFFFFu, mine.q0, l), x.n = __shfl_sync(0xFFFFFFFFu, mine.n, l);
            x.k0 = __shfl_sync(0xFFFFFFFFu, mine.k0, l), x.len = __shfl_sync(0xFFFFFFFFu, mine.len, l);
            x.before = __shfl_sync(0xFFFFFFFFu, mine.before, l);
            found = true;
        } else {
            block -= __shfl_sync(0xFFFFFFFFu, sum, 31);
        }
    }
    if (!found) return;
    const uint32_t token0 = block * per_block, tokens = min(per_block, x.n - token0);
    const uint32_t all_see = seen(a, x, token0), end = seen(a, x, token0 + tokens - 1u);  // positions that every row sees, that some row does

    const uint32_t base = smem_addr(smem);
    auto piece = [](uint32_t row, uint32_t c) { return row * (D * 2u) + ((c ^ (row & 7u)) << 4); };
    auto fill = [&](uint32_t tile) {
        const uint32_t kdst = base + (tile & 1u) * 2u * C::TILE_BYTES, vdst = kdst + C::TILE_BYTES, key0 = tile * SHORT_KEYS;
        const uint16_t* kp = a.k + (int64_t)(x.k0 + key0) * a.k_slot + (int64_t)head * a.k_head;
        const uint16_t* vp = a.v + (int64_t)(x.k0 + key0) * a.v_slot + (int64_t)head * a.v_head;
#pragma unroll
        for (uint32_t e = threadIdx.x; e < SHORT_KEYS * CH; e += SHORT_THREADS) {
            const uint32_t row = e / CH, c = e % CH;
            const bool there = key0 + row < x.len;
            cp_async16(kdst + piece(row, c), there ? kp + (int64_t)row * a.k_slot + 8u * c : a.k, there);
            cp_async16(vdst + piece(row, c), there ? vp + (int64_t)row * a.v_slot + 8u * c : a.v, there);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const uint32_t tiles = (end + SHORT_KEYS - 1u) / SHORT_KEYS;
    if (tiles > 0u) fill(0u);

    // rows lane / 4 and lane / 4 + 8 of the warp's sixteen
    uint32_t qf[KS][4], sees[2];
    float o[2 * KS][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {}, l_odd[2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t row = 16u * warp + lane / 4u + 8u * h, i = row / group;
        const bool there = i < tokens;
        sees[h] = there ? seen(a, x, token0 + i) : 0u;
        const uint16_t* qp = a.q + (int64_t)(x.q0 + token0 + (there ? i : 0u)) * a.q_token + (int64_t)(head * group + (there ? row % group : 0u)) * a.q_head + 2u * (lane & 3u);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qf[k][h] = there ? ld_fresh(reinterpret_cast<const uint32_t*>(qp + 16 * k)) : 0u;
            qf[k][2 + h] = there ? ld_fresh(reinterpret_cast<const uint32_t*>(qp + 16 * k + 8)) : 0u;
        }
    }
    uint32_t dirty_from = 0xFFFFFFFFu;  // first tile of values in which something was left out
#pragma unroll 1
    for (uint32_t tile = 0; tile < tiles; ++tile) {
        if (tile + 1u < tiles) fill(tile + 1u);
        else asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        const uint32_t kb = base + (tile & 1u) * 2u * C::TILE_BYTES, vb = kb + C::TILE_BYTES, key0 = tile * SHORT_KEYS;
        bool bad = false;
        if (key0 + SHORT_KEYS > all_see) {  // its own pieces, which the thread has waited for
#pragma unroll 4
            for (uint32_t e = threadIdx.x; e < SHORT_KEYS * CH; e += SHORT_THREADS) {
                uint32_t w[4], z[4];
                const uint32_t at = vb + piece(e / CH, e % CH);
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
                bool differs = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = finite_or_zero(w[i]), differs |= z[i] != w[i];
                if (differs) {
                    bad = true;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(z[0]), "r"(z[1]), "r"(z[2]), "r"(z[3]) : "memory");
                }
            }
        }
        if (__syncthreads_or(bad) && dirty_from == 0xFFFFFFFFu) dirty_from = tile;
        float s[NK][4];
        uint32_t p[NK][2];
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int n = 0; n < NK; n += 2) {
                uint32_t f[4];  // keys 8n .. 8n + 15: first and second eight dimensions of the first eight keys, then of the others
                ldmatrix4(f, kb + piece(8u * n + (lane & 7u) + 8u * (lane >> 4), 2u * k + ((lane >> 3) & 1u)));
                mma16816(s[n], qf[k], f[0], f[1]);
                mma16816(s[n + 1], qf[k], f[2], f[3]);
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < NK; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float& t = s[n][2 * h + j];
                    t = key0 + 8u * n + 2u * (lane & 3u) + j < sees[h] ? t * a.scale_log2 : -INFINITY;
                    top = fmaxf(top, t);
                }
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const float now = fmaxf(m[h], top), from = now == -INFINITY ? 0.0f : now, keep = exp2_fast(m[h] - from);
            m[h] = now;
            l[h] *= keep, l_odd[h] *= keep;
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                p[n][h] = pack_bf16(exp2_fast(s[n][2 * h] - from), exp2_fast(s[n][2 * h + 1] - from));
                add_bf16(l[h], l_odd[h], p[n][h]);
            }
#pragma unroll
            for (int d = 0; d < 2 * KS; ++d) o[d][2 * h] *= keep, o[d][2 * h + 1] *= keep;
        }
#pragma unroll
        for (int k = 0; k < NK / 2; ++k) {
            const uint32_t pa[4] = {p[2 * k][0], p[2 * k][1], p[2 * k + 1][0], p[2 * k + 1][1]};
#pragma unroll
            for (int d = 0; d < 2 * KS; d += 2) {
                uint32_t f[4];  // dimensions 8d .. 8d + 15 of sixteen keys
                ldmatrix4_trans(f, vb + piece(16u * k + (lane & 15u), d + (lane >> 4)));
                mma16816(o[d], pa, f[0], f[1]);
                mma16816(o[d + 1], pa, f[2], f[3]);
            }
        }
        __syncthreads();  // the tile is free
    }

#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float sum = l[h] + l_odd[h];
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
        const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;  // no key: zeros; NaN stays
        const uint32_t row = 16u * warp + lane / 4u + 8u * h, i = row / group;
        if (i >= tokens) continue;
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d) o[d][2 * h] *= inv, o[d][2 * h + 1] *= inv;
        if (dirty_from != 0xFFFFFFFFu) {  // values that are not finite, left out above, reach the rows that see them
#pragma unroll 1
            for (uint32_t key = max(dirty_from, all_see / SHORT_KEYS) * SHORT_KEYS; key < sees[h]; ++key) {
                const uint16_t* vp = a.v + (int64_t)(x.k0 + key) * a.v_slot + (int64_t)head * a.v_head + 2u * (lane & 3u);
#pragma unroll
                for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float v = bf16_bits_to_float(ld_fresh(vp + 8 * d + j));
                        if (!(fabsf(v) < INFINITY)) o[d][2 * h + j] += v;
                    }
            }
        }
        uint16_t* to = a.out + (int64_t)(x.q0 + token0 + i) * a.o_token + (int64_t)(head * group + row % group) * a.o_head + 2u * (lane & 3u);
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d) *reinterpret_cast<uint32_t*>(to + 8 * d) = pack_bf16(o[d][2 * h], o[d][2 * h + 1]);
    }
}

}  // namespace attention
}  // namespace miori_b200
