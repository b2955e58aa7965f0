// A whole layer of experts for the tokens of a decode step, 1..32 of them, in one launch:
//   l = R x;  p = softmax(l) or sigmoid(l);  the `top` experts of largest p (+ bias);  weights w = p [/ their sum] * factor
//   out[t] = sum_e w_e W_down,e (silu(g) * u),  [g; u] = W_up,e x[t]
//
// Bound by the chosen experts' weights, which are read once.  What a chain of launches pays on top is their hand-overs and the first trip to
// memory of each, so this is one cooperative kernel, one CTA an SM, clusters of four, with one meeting of the whole grid:
//   1  router: a cluster's CTAs take a quarter of K each, the partial logits meet through distributed shared memory.  Every CTA
//      chooses for itself (the same sums in the same order: the same choice), so that nothing waits for the grid;
//   2  gate and up: the rows of all chosen experts dealt evenly to the CTAs, eight gate and eight up rows an MMA tile; K over the
//      warps; the partial sums meet in shared memory, silu(g) * u goes to the workspace in fp32;
//   3  the grid meets; the first weights of 4 are on their way since before;
//   4  down: a cluster owns rows of the output.  The K axes of all experts, one behind the other, are dealt to the cluster's 64 warps, whose
//      sums, times w, meet per token: within a CTA, then over the cluster, always in the same order.
// Experts of more tokens than an MMA tile's columns (8, or 16 from nine tokens on) are listed once for every so many.
//
// Weights stream through a ring of cp.async stages that belongs to one warp: 16 rows x 128 of K and their scales, no CTA-wide wait.  They become
// fp16 without a rounding: 4-bit codes as subnormals in the bits of a half (see gemv_tma.cuh), e4m3 by conversion; products by mma.sync.m16n8k16,
// sums in fp32, times the scales after each group.  Activations, x and silu(g) * u, are fp16 times a power of two per token and 128 of K that
// puts the largest into [2^14, 2^15): for bf16 x no rounding down to 2^-27 of that largest (4 bits) or 2^-31; for silu(g) * u 2^-12 of a
// value, an eighth of what rounding it to bf16 costs where gate + up and down are two launches.
#pragma once
#include "common.cuh"

namespace miori_b200 {
namespace moe {

constexpr uint32_t MAX_TOKENS = 32, MAX_EXPERTS = 256, MAX_TOP = 16, MAX_ROWS = MAX_TOKENS * MAX_TOP;
constexpr uint32_t WARPS = 16, THREADS = WARPS * 32, CLUSTER = 4;
constexpr uint32_t UNIT = 128;  // of K: what a stage holds of 16 rows
constexpr uint32_t MAX_ENTRIES = MAX_EXPERTS + 32;
enum Format { GROUP64, GROUP32, E4M3 };

template <Format FMT>
struct Stage {
    static constexpr uint32_t WEIGHTS = FMT == E4M3 ? 2048 : 1024;
    static constexpr uint32_t SCALES = FMT == GROUP32 ? 256 : 128;
    static constexpr uint32_t BYTES = WEIGHTS + SCALES;
    static constexpr uint32_t DEPTH = FMT == E4M3 ? 4 : 6;
    static constexpr uint32_t RING = BYTES * DEPTH * WARPS;
};

struct Matrix {  // [experts][rows][K]
    const uint8_t* q;
    const uint8_t *s, *b;  // bf16 [experts][rows][K / group]; e4m3: s fp32 [experts][ceil(rows / 128)][ceil(K / 128)]
    uint32_t rows, K, units;
};
struct Args {
    const uint16_t *x, *router;
    const float* bias;
    Matrix up, down;
    void* out;
    float* h;            // [rows][F], rows: the (expert, token) pairs in the experts' order
    uint32_t* counters;  // arrived, left
    float factor;
    uint32_t tokens, experts, top, H, F;
    uint32_t sigmoid, norm, bf16;
    uint32_t slices;   // warps over K in 2, a power of two
    uint32_t area;     // bytes of partial sums
    uint32_t tiles_at_once;  // row tiles of a pass of 4
};

struct Tables {
    uint32_t mask[MAX_EXPERTS];       // tokens that chose the expert
    uint16_t entry_of[MAX_EXPERTS];   // its first entry
    uint16_t entry_expert[MAX_ENTRIES], entry_row[MAX_ENTRIES + 1];
    uint8_t row_token[MAX_ROWS];
    float row_weight[MAX_ROWS];
    int16_t chosen[MAX_ROWS];         // [token][place], -1: nobody
    float weight[MAX_ROWS];
    uint32_t entries;
    uint32_t given_up;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two e4m3 as two fp16, exactly.
__device__ __forceinline__ uint32_t e4m3_half(uint16_t pair) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(pair));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float remote_f32(uint32_t addr, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// Where K lies in a thread's fragments.  Thread (g, t) of a warp, g = lane / 4, holds of a unit 32 elements, the same of rows g and g + 8 of the weights
// and of column g of the activations, so that one MMA, whose k axis runs over t, stays inside a scale group.  Piece i (8 elements, word i of 4-bit codes):
template <Format FMT>
__device__ __forceinline__ uint32_t piece_k(uint32_t t, uint32_t i) {
    if (FMT == GROUP64) return (i >> 1) * 64u + t * 16u + (i & 1u) * 8u;
    if (FMT == GROUP32) return i * 32u + t * 8u;
    return t * 32u + i * 8u;
}
// 4-bit stages: a row's 64 bytes are four 16-byte chunks, fetched by the four threads of the row; chunk c of row g lies at slot c ^ (this), so that the
// words that a warp's threads read next lie in different banks.
template <Format FMT>
__device__ __forceinline__ uint32_t chunk_swizzle(uint32_t g) { return FMT == GROUP64 ? (g & 2u) : (g >> 1) & 3u; }

// The stage of one tile: row_lo, row_hi the thread's two rows of the matrix of expert `e`.
template <Format FMT>
__device__ __forceinline__ void issue(uint32_t stage, const Matrix& m, uint32_t e, uint32_t row_lo, uint32_t row_hi, uint32_t unit, uint32_t lane) {
    const uint32_t g = lane >> 2, t = lane & 3u;
    const size_t base = (size_t)e * m.rows;
    if constexpr (FMT == E4M3) {
#pragma unroll
        for (uint32_t r = 0; r < 2u; ++r) {
            const uint8_t* row = m.q + (base + (r ? row_hi : row_lo)) * m.K;
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c) {
                const uint32_t k = unit * UNIT + t * 32u + c * 16u;
                const bool there = k < m.K;
                cp16(stage + ((r * 2u + c) * 32u + lane) * 16u, row + (there ? k : 0u), there);
            }
        }
        if (lane < 2u) {
            const uint32_t row_blocks = (m.rows + 127u) / 128u, row = lane ? row_hi : row_lo;  // lanes 0 and 1 have g = 0: the tile's first rows
            cp4(stage + 2048u + lane * 4u, m.s + (((size_t)e * row_blocks + row / 128u) * m.units + unit) * 4u);
        }
    } else {
        constexpr uint32_t GROUP = FMT == GROUP64 ? 64 : 32;
        const uint32_t slot = (g * 4u + (t ^ chunk_swizzle<FMT>(g))) * 16u;
        const size_t at = (size_t)unit * 64u + t * 16u;
        cp16(stage + slot, m.q + (base + row_lo) * (m.K / 2u) + at, true);
        cp16(stage + 512u + slot, m.q + (base + row_hi) * (m.K / 2u) + at, true);
        // thread t of a row fetches its s, its partner's s, its b, its partner's b
        const uint8_t* from = t < 2u ? m.s : m.b;
        const size_t row = base + (t & 1u ? row_hi : row_lo);
        if constexpr (FMT == GROUP64) cp4(stage + 1024u + lane * 4u, from + (row * (m.K / GROUP) + unit * 2u) * 2u);
        else cp8(stage + 1024u + lane * 8u, from + (row * (m.K / GROUP) + unit * 4u) * 2u);
    }
}

// Activations of one unit as B fragments of up to NT tiles of eight columns.
template <Format FMT, int NT>
struct Frag {
    static constexpr int GROUPS = FMT == GROUP64 ? 2 : FMT == GROUP32 ? 4 : 1;
    uint32_t b[NT][16];
    float scale[NT][2];                                   // of the columns 2 t, 2 t + 1 whose sums this thread gets
    float sum[NT][FMT == E4M3 ? 1 : GROUPS][2];           // theirs, times 2^-22: what the biases multiply
};

// v: the thread's 32 elements of column g, in pieces.
template <Format FMT, int NT>
__device__ __forceinline__ void make_frag(Frag<FMT, NT>& f, int n, const float (&v)[32], uint32_t lane) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 32; ++i) m = fmaxf(m, fabsf(v[i]));
    m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    // 2^(14 - exponent of m), no further than where its reciprocal is still a normal number
    const uint32_t field = min(268u - (__float_as_uint(m) >> 23), 253u);
    const float up = __uint_as_float(field << 23), down = __uint_as_float((254u - field) << 23);
    const uint32_t c0 = (lane & 3u) * 8u, c1 = c0 + 4u;  // a lane of each of the two columns
    if constexpr (FMT == E4M3) {
#pragma unroll
        for (int i = 0; i < 16; ++i) f.b[n][i] = pack_half(v[2 * i] * up, v[2 * i + 1] * up);
        f.scale[n][0] = __shfl_sync(0xFFFFFFFFu, down, c0);
        f.scale[n][1] = __shfl_sync(0xFFFFFFFFu, down, c1);
    } else {
        // word i, codes 0..7: codes (0, 4) and (2, 6) are taken as multiples of 2^-22, (1, 5) and (3, 7) of 2^-18
        const float up16 = up * 0.0625f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f.b[n][4 * i] = pack_half(v[8 * i] * up, v[8 * i + 4] * up);
            f.b[n][4 * i + 1] = pack_half(v[8 * i + 1] * up16, v[8 * i + 5] * up16);
            f.b[n][4 * i + 2] = pack_half(v[8 * i + 2] * up, v[8 * i + 6] * up);
            f.b[n][4 * i + 3] = pack_half(v[8 * i + 3] * up16, v[8 * i + 7] * up16);
        }
        // The sums are those of the rounded values, so that a rounding counts times the weight and not times the code; by MMAs with rows of
        // 2^-22 and 2^-18, which leave them with the threads that need them.
        constexpr int G = Frag<FMT, NT>::GROUPS, PIECES = 4 / G;
#pragma unroll
        for (int q = 0; q < G; ++q) {
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = q * PIECES * 2; i < (q + 1) * PIECES * 2; ++i) mma_f16(s, 0x00040004u, 0x00040004u, 0x00400040u, 0x00400040u, f.b[n][2 * i], f.b[n][2 * i + 1]);
            f.sum[n][q][0] = s[0], f.sum[n][q][1] = s[1];
        }
        const float whole = down * 4194304.0f;  // 2^22
        f.scale[n][0] = __shfl_sync(0xFFFFFFFFu, whole, c0);
        f.scale[n][1] = __shfl_sync(0xFFFFFFFFu, whole, c1);
    }
}

// One stage times one unit of activations: out[n] = (row g, column 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1), scales applied.
template <Format FMT, int NT>
__device__ __forceinline__ void multiply(uint32_t stage, const Frag<FMT, NT>& f, uint32_t tiles, float (&out)[NT][4], uint32_t lane) {
    const uint32_t g = lane >> 2, t = lane & 3u;
    if constexpr (FMT == E4M3) {
        float acc[NT][4] = {};
        const uint2 sc = lds64(stage + 2048u);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint4 lo = lds128(stage + (c * 32u + lane) * 16u), hi = lds128(stage + ((2u + c) * 32u + lane) * 16u);
            const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a0 = e4m3_half((uint16_t)wl[i]), a2 = e4m3_half((uint16_t)(wl[i] >> 16));
                const uint32_t a1 = e4m3_half((uint16_t)wh[i]), a3 = e4m3_half((uint16_t)(wh[i] >> 16));
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    if (n == 0 || (uint32_t)n < tiles) mma_f16(acc[n], a0, a1, a2, a3, f.b[n][c * 8 + i * 2], f.b[n][c * 8 + i * 2 + 1]);
            }
        }
        const float sl = __uint_as_float(sc.x), sh = __uint_as_float(sc.y);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            out[n][0] = acc[n][0] * sl * f.scale[n][0], out[n][1] = acc[n][1] * sl * f.scale[n][1];
            out[n][2] = acc[n][2] * sh * f.scale[n][0], out[n][3] = acc[n][3] * sh * f.scale[n][1];
        }
    } else {
        constexpr int G = Frag<FMT, NT>::GROUPS, PIECES = 4 / G;
        // scales and biases of rows g and g + 8, a pair of groups a word: s lo, s hi, b lo, b hi (twice as wide in groups of 32)
        uint32_t words[4 * (G / 2)];
        if constexpr (FMT == GROUP64) {
            const uint4 w = lds128(stage + 1024u + g * 16u);
            words[0] = w.x, words[1] = w.y, words[2] = w.z, words[3] = w.w;
        } else {
            const uint4 w = lds128(stage + 1024u + g * 32u), z = lds128(stage + 1024u + g * 32u + 16u);
            words[0] = w.x, words[1] = w.y, words[2] = w.z, words[3] = w.w, words[4] = z.x, words[5] = z.y, words[6] = z.z, words[7] = z.w;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) out[n][0] = out[n][1] = out[n][2] = out[n][3] = 0.0f;
#pragma unroll
        for (int q = 0; q < G; ++q) {
            uint32_t lo[PIECES], hi[PIECES];
            if constexpr (FMT == GROUP64) {
                const uint32_t at = stage + (g * 4u + ((t >> 1) + 2u * q ^ chunk_swizzle<FMT>(g))) * 16u + (t & 1u) * 8u;
                const uint2 l = lds64(at), h = lds64(at + 512u);
                lo[0] = l.x, lo[1] = l.y, hi[0] = h.x, hi[1] = h.y;
            } else {
                const uint32_t at = stage + (g * 4u + ((uint32_t)q ^ chunk_swizzle<FMT>(g))) * 16u + t * 4u;
                lo[0] = lds32(at), hi[0] = lds32(at + 512u);
            }
            float acc[NT][4] = {};
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const uint32_t l2 = lo[p] << 2, l6 = lo[p] >> 6, h2 = hi[p] << 2, h6 = hi[p] >> 6;
                const int at = (q * PIECES + p) * 4;
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    if (n == 0 || (uint32_t)n < tiles) {
                        mma_f16(acc[n], l2 & 0x003C003Cu, h2 & 0x003C003Cu, l2 & 0x03C003C0u, h2 & 0x03C003C0u, f.b[n][at], f.b[n][at + 1]);
                        mma_f16(acc[n], l6 & 0x003C003Cu, h6 & 0x003C003Cu, l6 & 0x03C003C0u, h6 & 0x03C003C0u, f.b[n][at + 2], f.b[n][at + 3]);
                    }
            }
            const int pair = G / 2, at = q >> 1;
            auto value = [&](int which) { return q & 1 ? bf16hi(words[which * pair + at]) : bf16lo(words[which * pair + at]); };
            const float sl = value(0), sh = value(1), bl = value(2), bh = value(3);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                out[n][0] = __fmaf_rn(sl, acc[n][0], __fmaf_rn(bl, f.sum[n][q][0], out[n][0]));
                out[n][1] = __fmaf_rn(sl, acc[n][1], __fmaf_rn(bl, f.sum[n][q][1], out[n][1]));
                out[n][2] = __fmaf_rn(sh, acc[n][2], __fmaf_rn(bh, f.sum[n][q][0], out[n][2]));
                out[n][3] = __fmaf_rn(sh, acc[n][3], __fmaf_rn(bh, f.sum[n][q][1], out[n][3]));
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
            out[n][0] *= f.scale[n][0], out[n][1] *= f.scale[n][1], out[n][2] *= f.scale[n][0], out[n][3] *= f.scale[n][1];
    }
}

// A score as a number that grows with it; 1 for NaN, below every score.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) return 1u;
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// 1: logits of all experts for all tokens, in every CTA, [token][expert] at the start of the area.
__device__ __forceinline__ void route_logits(const Args& a, uint32_t area, uint32_t rank, uint32_t warp, uint32_t lane) {
    const uint32_t g = lane >> 2, t = lane & 3u;
    uint32_t wide = 1;  // tiles of 16 experts, up to a power of two
    while (wide * 16u < a.experts) wide *= 2u;
    const uint32_t split = WARPS / wide, tile = warp % wide, slice = warp / wide;
    const uint32_t units = (a.H + UNIT - 1u) / UNIT, u0 = rank * units / CLUSTER, u1 = (rank + 1u) * units / CLUSTER;
    const uint32_t columns = (a.tokens + 7u) / 8u;
    const uint32_t e_lo = tile * 16u + g, e_hi = e_lo + 8u;
    float acc[MAX_TOKENS / 8][4] = {};
    for (uint32_t u = u0 + slice; u < u1; u += split) {
        const uint32_t k = u * UNIT + t * 32u;
        uint4 lo[4], hi[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const bool there = k + i * 8u < a.H;
            lo[i] = hi[i] = make_uint4(0u, 0u, 0u, 0u);
            if (there && e_lo < a.experts) lo[i] = ld_fresh(reinterpret_cast<const uint4*>(a.router + (size_t)e_lo * a.H + k + i * 8u));
            if (there && e_hi < a.experts) hi[i] = ld_fresh(reinterpret_cast<const uint4*>(a.router + (size_t)e_hi * a.H + k + i * 8u));
        }
#pragma unroll
        for (uint32_t n = 0; n < MAX_TOKENS / 8u; ++n) {
            if (n >= columns) break;
            const uint32_t token = n * 8u + g;
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (token < a.tokens && k + i * 8u < a.H) x = ld_fresh(reinterpret_cast<const uint4*>(a.x + (size_t)token * a.H + k + i * 8u));
                mma_bf16(acc[n], lo[i].x, hi[i].x, lo[i].y, hi[i].y, x.x, x.y);
                mma_bf16(acc[n], lo[i].z, hi[i].z, lo[i].w, hi[i].w, x.z, x.w);
            }
        }
    }
    // [slice][token][expert of the tiles], then the CTA's sums over the slices, then the cluster's over the CTAs
    const uint32_t width = wide * 16u, plane = a.tokens * width;
    float* part = nullptr;
    asm volatile("{\n\t.reg .u64 p;\n\tcvt.u64.u32 p, %1;\n\tcvta.shared.u64 %0, p;\n\t}" : "=l"(part) : "r"(area));
#pragma unroll
    for (uint32_t n = 0; n < MAX_TOKENS / 8u; ++n) {
        const uint32_t token = n * 8u + 2u * t;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
            if (token + (i & 1u) < a.tokens) part[slice * plane + (token + (i & 1u)) * width + (i < 2u ? e_lo : e_hi)] = acc[n][i];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < plane; i += THREADS) {
        float s = part[i];
        for (uint32_t p = 1; p < split; ++p) s += part[p * plane + i];
        part[i] = s;
    }
    cluster_barrier();
    // behind the partial sums, which the other CTAs still read
    for (uint32_t i = threadIdx.x; i < plane; i += THREADS) {
        float s = remote_f32(area + i * 4u, 0);
#pragma unroll
        for (uint32_t r = 1; r < CLUSTER; ++r) s += remote_f32(area + i * 4u, r);
        part[split * plane + i] = s;
    }
    cluster_barrier();
}

// The choice of one token by one warp.  logits: [expert] in shared memory.
__device__ __forceinline__ void choose(const Args& a, Tables& tb, const float* logits, uint32_t token, uint32_t lane) {
    constexpr int PER = MAX_EXPERTS / 32;
    float p[PER];
    uint32_t key[PER];
    float most = -INFINITY, total = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t e = j * 32u + lane;
        p[j] = e < a.experts ? logits[e] : -INFINITY;
        key[j] = e < a.experts ? order_key(p[j]) : 0u;
        most = fmaxf(most, p[j]);
    }
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < PER; ++j) p[j] = 1.0f / (1.0f + expf(-p[j]));
    } else {
#pragma unroll
        for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            p[j] = j * 32u + lane < a.experts ? expf(p[j] - most) : 0.0f;
            total += p[j];
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
#pragma unroll
        for (int j = 0; j < PER; ++j) p[j] = p[j] / total;
    }
    if (a.bias) {  // without one the order is that of the logits, which no exponential has rounded
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t e = j * 32u + lane;
            if (e < a.experts) {
                const float b = ld_fresh(a.bias + e);
                key[j] = b == -INFINITY ? 0u : order_key(p[j] + b);
            }
        }
    }
    float mine = 0.0f, sum = 0.0f;  // lane j: the j-th choice
    int expert = -1;
    for (uint32_t place = 0; place < a.top; ++place) {
        uint32_t best = 0, best_e = 0xFFFFFFFFu;
        float best_p = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (key[j] > best) best = key[j], best_e = j * 32u + lane, best_p = p[j];
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
        if (top == 0u) break;
        const uint32_t e = __reduce_min_sync(0xFFFFFFFFu, best == top ? best_e : 0xFFFFFFFFu);
        const float w = __shfl_sync(0xFFFFFFFFu, best_p, e & 31u);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j * 32u + lane == e) key[j] = 0u;
        sum += w;
        if (lane == place) mine = w, expert = (int)e;
    }
    if (lane < a.top) {
        tb.chosen[token * a.top + lane] = (int16_t)expert;
        tb.weight[token * a.top + lane] = (a.norm ? mine / sum : mine) * a.factor;
        if (expert >= 0) atomicOr(&tb.mask[expert], 1u << token);
    }
}

// Entries: the chosen experts in order, one for every `columns` of their tokens.  By one warp.
__device__ __forceinline__ void list_entries(const Args& a, Tables& tb, uint32_t columns, uint32_t lane) {
    uint32_t entry = 0, row = 0;
    for (uint32_t e0 = 0; e0 < a.experts; e0 += 32u) {
        const uint32_t e = e0 + lane, count = e < a.experts ? __popc(tb.mask[e]) : 0u, mine = (count + columns - 1u) / columns;
        uint32_t before = mine << 16 | count;  // both prefix sums in one
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, before, d);
            if (lane >= (uint32_t)d) before += v;
        }
        const uint32_t all = __shfl_sync(0xFFFFFFFFu, before, 31);
        const uint32_t my_entry = entry + (before >> 16) - mine, my_row = row + (before & 0xFFFFu) - count;
        if (e < a.experts) tb.entry_of[e] = (uint16_t)my_entry;
        for (uint32_t i = 0; i < mine; ++i) {
            tb.entry_expert[my_entry + i] = (uint16_t)e;
            tb.entry_row[my_entry + i] = (uint16_t)(my_row + i * columns);
        }
        entry += all >> 16, row += all & 0xFFFFu;
    }
    if (lane == 0) tb.entries = entry, tb.entry_row[entry] = (uint16_t)row;
}

template <Format FMT, int NT>
__global__ void __launch_bounds__(THREADS, 1)
moe_kernel(const Args a) {
    using S = Stage<FMT>;
    constexpr uint32_t COLUMNS = 8u * NT, CELL = NT * 512u;  // a tile's partial sums: NT float4 a thread
    constexpr int DEPTH = S::DEPTH;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Tables tb;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t rank = blockIdx.x % CLUSTER, cluster = blockIdx.x / CLUSTER, clusters = gridDim.x / CLUSTER;
    const uint32_t ring = smem_addr(smem) + warp * (S::BYTES * DEPTH), area = smem_addr(smem) + S::RING;
    float* const cells = reinterpret_cast<float*>(smem + S::RING);

    // ---- 1
    for (uint32_t e = threadIdx.x; e < MAX_EXPERTS; e += THREADS) tb.mask[e] = 0u;
    if (threadIdx.x == 0) tb.given_up = 0u;
    route_logits(a, area, rank, warp, lane);
    {
        uint32_t wide = 1;
        while (wide * 16u < a.experts) wide *= 2u;
        const float* logits = cells + WARPS / wide * (a.tokens * wide * 16u);
        for (uint32_t token = warp; token < a.tokens; token += WARPS) choose(a, tb, logits + token * wide * 16u, token, lane);
    }
    __syncthreads();
    if (warp == 0) list_entries(a, tb, COLUMNS, lane);
    __syncthreads();
    if (threadIdx.x < a.tokens * a.top) {
        const int e = tb.chosen[threadIdx.x];
        if (e >= 0) {
            const uint32_t token = threadIdx.x / a.top;
            const uint32_t row = tb.entry_row[tb.entry_of[e]] + __popc(tb.mask[e] & ((1u << token) - 1u));
            tb.row_token[row] = (uint8_t)token;
            tb.row_weight[row] = tb.weight[threadIdx.x];
        }
    }
    __syncthreads();
    const uint32_t entries = tb.entries;

    // ---- 2
    const uint32_t f_tiles = a.F / 8u;
    {
        const uint64_t items = (uint64_t)entries * f_tiles;
        const uint32_t i0 = (uint32_t)(items * blockIdx.x / gridDim.x), i1 = (uint32_t)(items * (blockIdx.x + 1u) / gridDim.x);
        const uint32_t slices = a.slices, groups = WARPS / slices, slice = warp % slices, group = warp / slices;
        const uint32_t per_round = a.area / (slices * CELL) / groups * groups;  // items
        // the order in which this warp goes through its stages: rounds, units of its slice, items of its group
        struct Walk {
            uint32_t first, unit, item;
        };
        auto begin = [&](uint32_t first) { return Walk{first, slice, first + group}; };
        auto valid = [&](const Walk& w) { return w.first < i1; };
        auto settle = [&](Walk& w) {  // to the next stage there is
            while (w.first < i1) {
                if (w.unit >= a.up.units) w = begin(w.first + per_round);
                else if (w.item >= min(i1, w.first + per_round)) w.unit += slices, w.item = w.first + group;
                else break;
            }
        };
        Walk ahead = begin(i0);
        settle(ahead);
        uint32_t put = 0, got = 0;
        auto fill = [&]() {
            if (valid(ahead)) {
                const uint32_t entry = ahead.item / f_tiles, row = (ahead.item - entry * f_tiles) * 8u + g;
                issue<FMT>(ring + put * S::BYTES, a.up, tb.entry_expert[entry], row, a.F + row, ahead.unit, lane);
                ahead.item += groups;
                settle(ahead);
            }
            cp_commit();
            if (++put == (uint32_t)DEPTH) put = 0u;
        };
        for (int i = 0; i < DEPTH - 1; ++i) fill();
        for (uint32_t first = i0; first < i1; first += per_round) {
            const uint32_t last = min(i1, first + per_round);
            for (uint32_t unit = slice; unit < a.up.units; unit += slices) {
                Frag<FMT, NT> f;
                uint32_t have = 0xFFFFFFFFu, tiles = 1;
                for (uint32_t item = first + group; item < last; item += groups) {
                    const uint32_t entry = item / f_tiles;
                    if (entry != have) {
                        have = entry;
                        const uint32_t row0 = tb.entry_row[entry], count = tb.entry_row[entry + 1u] - row0;
                        tiles = (count + 7u) / 8u;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (n && (uint32_t)n >= tiles) break;
                            float v[32];
                            const bool there = n * 8u + g < count;
                            const uint16_t* x = a.x + (size_t)(there ? tb.row_token[row0 + n * 8u + g] : 0u) * a.H;
#pragma unroll
                            for (uint32_t i = 0; i < 4u; ++i) {
                                const uint32_t k = unit * UNIT + piece_k<FMT>(t, i);
                                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                                if (there && k < a.H) w = ld_fresh(reinterpret_cast<const uint4*>(x + k));
                                v[8 * i] = bf16lo(w.x), v[8 * i + 1] = bf16hi(w.x), v[8 * i + 2] = bf16lo(w.y), v[8 * i + 3] = bf16hi(w.y);
                                v[8 * i + 4] = bf16lo(w.z), v[8 * i + 5] = bf16hi(w.z), v[8 * i + 6] = bf16lo(w.w), v[8 * i + 7] = bf16hi(w.w);
                            }
                            make_frag(f, n, v, lane);
                        }
                    }
                    cp_wait<DEPTH - 2>();
                    __syncwarp();
                    float o[NT][4];
                    multiply<FMT, NT>(ring + got * S::BYTES, f, tiles, o, lane);
                    __syncwarp();
                    if (++got == (uint32_t)DEPTH) got = 0u;
                    fill();
                    float4* cell = reinterpret_cast<float4*>(cells) + (((item - first) * slices + slice) * NT) * 32u + lane;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (n && (uint32_t)n >= tiles) break;
                        float4 s = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
                        if (unit != slice) {
                            const float4 p = cell[n * 32];
                            s.x += p.x, s.y += p.y, s.z += p.z, s.w += p.w;
                        }
                        cell[n * 32] = s;
                    }
                }
            }
            __syncthreads();
            const uint32_t used = min(slices, a.up.units);
            for (uint32_t i = threadIdx.x; i < (last - first) * CELL / 16u; i += THREADS) {
                const uint32_t at = i / (NT * 32u), n = i / 32u % NT, entry = (first + at) / f_tiles;
                const uint32_t row0 = tb.entry_row[entry], count = tb.entry_row[entry + 1u] - row0, column = n * 8u + 2u * t;
                if (column >= count) continue;
                const float4* from = reinterpret_cast<const float4*>(cells) + (at * slices * NT + n) * 32u + lane;
                float4 s = from[0];
                for (uint32_t p = 1; p < used; ++p) {
                    const float4 v = from[p * NT * 32u];
                    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
                }
                float* to = a.h + (size_t)(row0 + column) * a.F + (first + at - entry * f_tiles) * 8u + g;
                to[0] = s.x / (1.0f + expf(-s.x)) * s.z;
                if (column + 1u < count) to[a.F] = s.y / (1.0f + expf(-s.y)) * s.w;
            }
            __syncthreads();
        }
    }
    cp_wait<0>();

    // ---- 3 and 4
    const uint32_t row_tiles = a.H / 16u, r0 = (uint32_t)((uint64_t)row_tiles * cluster / clusters), r1 = (uint32_t)((uint64_t)row_tiles * (cluster + 1u) / clusters);
    const uint32_t worker = rank * WARPS + warp, all_units = entries * a.down.units;
    const uint32_t u0 = (uint32_t)((uint64_t)all_units * worker / (CLUSTER * WARPS)), u1 = (uint32_t)((uint64_t)all_units * (worker + 1u) / (CLUSTER * WARPS));
    struct Walk {
        uint32_t first, unit, tile;
    } ahead = {r0, u0, r0};
    uint32_t put = 0, got = 0;
    auto fill = [&]() {
        if (ahead.first < r1 && u0 < u1) {
            const uint32_t entry = ahead.unit / a.down.units, row = ahead.tile * 16u + g;
            issue<FMT>(ring + put * S::BYTES, a.down, tb.entry_expert[entry], row, row + 8u, ahead.unit - entry * a.down.units, lane);
            if (++ahead.tile >= min(r1, ahead.first + a.tiles_at_once)) {
                if (++ahead.unit >= u1) ahead.first += a.tiles_at_once, ahead.unit = u0;
                ahead.tile = ahead.first;
            }
        }
        cp_commit();
        if (++put == (uint32_t)DEPTH) put = 0u;
    };
    for (int i = 0; i < DEPTH - 1; ++i) fill();

    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(&a.counters[0], 1u);
        const long long began = clock64();
        uint32_t seen;
        for (;;) {
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(a.counters) : "memory");
            if (seen >= gridDim.x) break;
            if (clock64() - began > WAIT_LIMIT_CYCLES) {
                tb.given_up = 1u;
                device_error(0x6F01u, blockIdx.x, seen);
                break;
            }
        }
        __threadfence();
    }
    __syncthreads();
    pdl_launch_dependents();
    const bool given_up = tb.given_up != 0u;  // the cluster barriers below are reached all the same

    for (uint32_t first = r0; first < r1; first += a.tiles_at_once) {
        const uint32_t last = min(r1, first + a.tiles_at_once), plane = (last - first) * a.tokens * 16u;
        float* mine = cells + warp * (a.tiles_at_once * a.tokens * 16u);  // [tile][token][16 rows]
        for (uint32_t i = lane; i < plane; i += 32u) mine[i] = 0.0f;
        __syncwarp();
        for (uint32_t unit = u0; unit < u1 && !given_up; ++unit) {
            const uint32_t entry = unit / a.down.units, k0 = (unit - entry * a.down.units) * UNIT;
            const uint32_t row0 = tb.entry_row[entry], count = tb.entry_row[entry + 1u] - row0, tiles = (count + 7u) / 8u;
            Frag<FMT, NT> f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n && (uint32_t)n >= tiles) break;
                float v[32];
                const bool there = n * 8u + g < count;
                const float* h = a.h + (size_t)(row0 + (there ? n * 8u + g : 0u)) * a.F;
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) {
                    const uint32_t k = k0 + piece_k<FMT>(t, i);
                    float4 p = make_float4(0.0f, 0.0f, 0.0f, 0.0f), q = p;
                    if (there && k < a.F) p = ld_fresh(reinterpret_cast<const float4*>(h + k)), q = ld_fresh(reinterpret_cast<const float4*>(h + k + 4u));
                    v[8 * i] = p.x, v[8 * i + 1] = p.y, v[8 * i + 2] = p.z, v[8 * i + 3] = p.w, v[8 * i + 4] = q.x, v[8 * i + 5] = q.y, v[8 * i + 6] = q.z, v[8 * i + 7] = q.w;
                }
                make_frag(f, n, v, lane);
            }
            // where the sums of this thread's columns go, and their weights
            uint32_t to[NT][2];
            float w[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (uint32_t c = 0; c < 2u; ++c) {
                    const uint32_t column = n * 8u + 2u * t + c;
                    to[n][c] = column < count ? tb.row_token[row0 + column] * 16u + g : 0xFFFFFFFFu;
                    w[n][c] = column < count ? tb.row_weight[row0 + column] : 0.0f;
                }
            for (uint32_t tile = first; tile < last; ++tile) {
                cp_wait<DEPTH - 2>();
                __syncwarp();
                float o[NT][4];
                multiply<FMT, NT>(ring + got * S::BYTES, f, tiles, o, lane);
                __syncwarp();
                if (++got == (uint32_t)DEPTH) got = 0u;
                fill();
                float* at = mine + (tile - first) * (a.tokens * 16u);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (uint32_t c = 0; c < 2u; ++c)
                        if (to[n][c] != 0xFFFFFFFFu) {
                            at[to[n][c]] = __fmaf_rn(w[n][c], o[n][c], at[to[n][c]]);
                            at[to[n][c] + 8u] = __fmaf_rn(w[n][c], o[n][2u + c], at[to[n][c] + 8u]);
                        }
            }
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < plane; i += THREADS) {
            float s = cells[i];
#pragma unroll
            for (uint32_t p = 1; p < WARPS; ++p) s += cells[p * (a.tiles_at_once * a.tokens * 16u) + i];
            cells[i] = s;
        }
        cluster_barrier();
        const uint32_t share0 = plane / 16u * rank / CLUSTER * 16u, share1 = plane / 16u * (rank + 1u) / CLUSTER * 16u;
        for (uint32_t i = share0 + threadIdx.x; i < share1; i += THREADS) {
            float s = remote_f32(area + i * 4u, 0);
#pragma unroll
            for (uint32_t r = 1; r < CLUSTER; ++r) s += remote_f32(area + i * 4u, r);
            const uint32_t tile = i / (a.tokens * 16u), token = i / 16u % a.tokens, row = (first + tile) * 16u + i % 16u;
            const size_t at = (size_t)token * a.H + row;
            if (given_up) continue;
            if (a.bf16) static_cast<uint16_t*>(a.out)[at] = (uint16_t)pack_bf16(s, 0.0f);
            else static_cast<float*>(a.out)[at] = s;
        }
        cluster_barrier();
    }
    cp_wait<0>();
    // the last to leave puts the counters back to zero
    if (threadIdx.x == 0 && !given_up) {
        __threadfence();
        if (atomicAdd(&a.counters[1], 1u) == gridDim.x - 1u) {
            a.counters[0] = 0u;
            a.counters[1] = 0u;
        }
    }
}

}  // namespace moe
}  // namespace miori_b200
