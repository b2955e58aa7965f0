// A whole layer of experts for the tokens of a decode step, 1..32 of them:
//   l = R x;  p = softmax(l) or sigmoid(l);  the `top` experts of largest p (+ bias);  weights w = p [/ their sum] * factor
//   out[t] = sum_e w_e W_down,e (silu(g) * u),  [g; u] = W_up,e x[t]
//
// Bound by the chosen experts' weights, which are read once.  Three launches, each of which begins while the one before drains:
//   moe_router  logits, 16 experts a CTA, K over its warps;
//   moe_up      every CTA chooses for itself from the logits (the same sums in the same order: the same choice); the rows of all chosen experts'
//               gate and up are dealt evenly to the CTAs, eight of each an MMA tile, K over the warps, whose partial sums meet in
//               shared memory; silu(g) * u goes to the workspace in fp32.  At its end a CTA asks L2 for its share of the down weights;
//   moe_down    a cluster of four CTAs owns rows of the output.  The K axes of all experts, one behind the other, are dealt to its 64 warps,
//               whose sums meet by token, times w, in a CTA and then over the cluster, always in the same order.
// (As one cooperative launch with a meeting of the grid between the products the layer took 23 us for a token where this takes 11: such a
// meeting costs 2.6 us, what it saves of a launch 0.7, and clusters of a whole SM's shared memory leave 16 SMs out.)
// Experts of more tokens than an MMA tile's columns (8, or 16 from nine tokens on) are listed once for every so many.
//
// Weights stream through a ring of cp.async stages that belongs to one warp: 16 rows x 128 of K and their scales, no CTA-wide wait.  They become
// fp16 without a rounding: 4-bit codes as subnormals in the bits of a half, e4m3 by conversion; products by mma.sync.m16n8k16, sums in fp32, times
// the scales after each group.  Activations, x and silu(g) * u, are fp16 times a power of two per token and 128 of K that puts the largest into
// [2^14, 2^15): for bf16 x no rounding down to 2^-27 of that largest (4 bits) or 2^-31; for silu(g) * u 2^-11 of a value at most, an
// eighth of what rounding it to bf16 costs where gate + up and down are two calls.
#pragma once
#include "common.cuh"

namespace miori_b200 {
namespace moe {

constexpr uint32_t MAX_TOKENS = 32, MAX_EXPERTS = 256, MAX_TOP = 16, MAX_ROWS = MAX_TOKENS * MAX_TOP;
constexpr uint32_t WARPS = 16, THREADS = WARPS * 32, CLUSTER = 4;
constexpr uint32_t UNIT = 128;  // of K: what a stage holds of 16 rows
constexpr uint32_t MAX_ENTRIES = MAX_EXPERTS + 32;
constexpr size_t PREFETCH = 192 * 1024;  // bytes of down weights that a CTA of moe_up asks L2 for
enum Format { GROUP64, GROUP32, E4M3 };

template <Format FMT>
struct Stage {
    static constexpr uint32_t WEIGHTS = FMT == E4M3 ? 2048 : 1024;
    static constexpr uint32_t SCALES = FMT == GROUP32 ? 256 : 128;
    static constexpr uint32_t BYTES = WEIGHTS + SCALES;
    static constexpr uint32_t DEPTH = FMT == E4M3 ? 4 : 5;
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
    float* logits;  // [tokens][experts]
    float* h;       // [rows][F], rows: the (expert, token) pairs in the experts' order
    float factor;
    uint32_t tokens, experts, top, H, F;
    uint32_t sigmoid, norm, bf16, ahead;  // ahead: weights may be read before the launch before is done
    uint32_t slices;   // moe_up: warps over K, a power of two
    uint32_t area;     // bytes of partial sums
    uint32_t per;      // moe_down: row tiles of a cluster
};

struct Tables {
    uint32_t mask[MAX_EXPERTS];       // tokens that chose the expert
    uint16_t entry_of[MAX_EXPERTS];   // its first entry
    uint16_t entry_expert[MAX_ENTRIES], entry_row[MAX_ENTRIES + 1];
    uint8_t row_token[MAX_ROWS];
    int16_t chosen[MAX_ROWS];         // [token][place], -1: nobody
    uint16_t slot[MAX_ROWS];          // of a place: entry * 16 + column of the entry
    float weight[MAX_ROWS];
    uint32_t entries;
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
// Warps may come here from loops that their threads leave at different times: not the aligned form.
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
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

// Activations of one unit as B fragments of up to NT tiles of eight columns.
template <Format FMT, int NT>
struct Frag {
    static constexpr int GROUPS = FMT == GROUP64 ? 2 : FMT == GROUP32 ? 4 : 1;
    uint32_t b[NT][16];
    float scale[NT][2];                                   // of the columns 2 t, 2 t + 1 whose sums this thread gets
    float sum[NT][FMT == E4M3 ? 1 : GROUPS][2];           // theirs, times 2^-24: what the biases multiply
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
        // word i, codes 0..7: codes (0, 4) and (2, 6) are taken as multiples of 2^-24, (1, 5) and (3, 7) of 2^-20
        const float up16 = up * 0.0625f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f.b[n][4 * i] = pack_half(v[8 * i] * up, v[8 * i + 4] * up);
            f.b[n][4 * i + 1] = pack_half(v[8 * i + 1] * up16, v[8 * i + 5] * up16);
            f.b[n][4 * i + 2] = pack_half(v[8 * i + 2] * up, v[8 * i + 6] * up);
            f.b[n][4 * i + 3] = pack_half(v[8 * i + 3] * up16, v[8 * i + 7] * up16);
        }
        // The sums are those of the rounded values, so that a rounding counts times the weight and not times the code; by MMAs with rows of
        // 2^-24 and 2^-20, which leave them with the threads that need them.
        constexpr int G = Frag<FMT, NT>::GROUPS, PIECES = 4 / G;
#pragma unroll
        for (int q = 0; q < G; ++q) {
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = q * PIECES * 2; i < (q + 1) * PIECES * 2; ++i) mma_f16(s, 0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u, f.b[n][2 * i], f.b[n][2 * i + 1]);
            f.sum[n][q][0] = s[0], f.sum[n][q][1] = s[1];
        }
        const float whole = down * 16777216.0f;  // 2^24
        f.scale[n][0] = __shfl_sync(0xFFFFFFFFu, whole, c0);
        f.scale[n][1] = __shfl_sync(0xFFFFFFFFu, whole, c1);
    }
}

// One stage times one unit of activations, COUNT tiles of columns: out[n] = (row g, column 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1), scales
// applied.
template <Format FMT, int NT, int COUNT>
__device__ __forceinline__ void multiply(uint32_t stage, const Frag<FMT, NT>& f, float (&out)[NT][4], uint32_t lane) {
    const uint32_t g = lane >> 2, t = lane & 3u;
    if constexpr (FMT == E4M3) {
        float acc[COUNT][4] = {};
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
                for (int n = 0; n < COUNT; ++n)
                    mma_f16(acc[n], a0, a1, a2, a3, f.b[n][c * 8 + i * 2], f.b[n][c * 8 + i * 2 + 1]);
            }
        }
        const float sl = __uint_as_float(sc.x), sh = __uint_as_float(sc.y);
#pragma unroll
        for (int n = 0; n < COUNT; ++n) {
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
        for (int n = 0; n < COUNT; ++n) out[n][0] = out[n][1] = out[n][2] = out[n][3] = 0.0f;
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
            float acc[COUNT][4] = {};
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const uint32_t l = lo[p], h = hi[p], l8 = l >> 8, h8 = h >> 8;
                const int at = (q * PIECES + p) * 4;
#pragma unroll
                for (int n = 0; n < COUNT; ++n) {
                    mma_f16(acc[n], l & 0x000F000Fu, h & 0x000F000Fu, l & 0x00F000F0u, h & 0x00F000F0u, f.b[n][at], f.b[n][at + 1]);
                    mma_f16(acc[n], l8 & 0x000F000Fu, h8 & 0x000F000Fu, l8 & 0x00F000F0u, h8 & 0x00F000F0u, f.b[n][at + 2], f.b[n][at + 3]);
                }
            }
            const int pair = G / 2, at = q >> 1;
            auto value = [&](int which) { return q & 1 ? bf16hi(words[which * pair + at]) : bf16lo(words[which * pair + at]); };
            const float sl = value(0), sh = value(1), bl = value(2), bh = value(3);
#pragma unroll
            for (int n = 0; n < COUNT; ++n) {
                out[n][0] = __fmaf_rn(sl, acc[n][0], __fmaf_rn(bl, f.sum[n][q][0], out[n][0]));
                out[n][1] = __fmaf_rn(sl, acc[n][1], __fmaf_rn(bl, f.sum[n][q][1], out[n][1]));
                out[n][2] = __fmaf_rn(sh, acc[n][2], __fmaf_rn(bh, f.sum[n][q][0], out[n][2]));
                out[n][3] = __fmaf_rn(sh, acc[n][3], __fmaf_rn(bh, f.sum[n][q][1], out[n][3]));
            }
        }
#pragma unroll
        for (int n = 0; n < COUNT; ++n)
            out[n][0] *= f.scale[n][0], out[n][1] *= f.scale[n][1], out[n][2] *= f.scale[n][0], out[n][3] *= f.scale[n][1];
    }
}

// A score as a number that grows with it; 1 for NaN, below every score.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) return 1u;
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Logits [token][expert]: a CTA has 16 experts, its warps share K.
__global__ void __launch_bounds__(THREADS)
moe_router_kernel(const Args a) {
    __shared__ float part[WARPS / 2][MAX_TOKENS][16];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t units = (a.H + UNIT - 1u) / UNIT, columns = (a.tokens + 7u) / 8u;
    const uint32_t e_lo = blockIdx.x * 16u + g, e_hi = e_lo + 8u;
    uint4 lo[4], hi[4];
    auto weights = [&](uint32_t u) {
        const uint32_t k = u * UNIT + t * 32u;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const bool there = u < units && k + i * 8u < a.H;
            lo[i] = hi[i] = make_uint4(0u, 0u, 0u, 0u);
            if (there && e_lo < a.experts) lo[i] = ld_fresh(reinterpret_cast<const uint4*>(a.router + (size_t)e_lo * a.H + k + i * 8u));
            if (there && e_hi < a.experts) hi[i] = ld_fresh(reinterpret_cast<const uint4*>(a.router + (size_t)e_hi * a.H + k + i * 8u));
        }
    };
    pdl_launch_dependents();
    if (a.ahead) weights(warp);
    pdl_wait_prior();
    float acc[MAX_TOKENS / 8][4] = {};
    for (uint32_t u = warp; u < units; u += WARPS) {
        if (u != warp || !a.ahead) weights(u);
        const uint32_t k = u * UNIT + t * 32u;
#pragma unroll
        for (uint32_t n = 0; n < MAX_TOKENS / 8u; ++n) {
            if (n >= columns) break;
            const uint32_t token = n * 8u + g;
            uint4 x[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (token < a.tokens && k + i * 8u < a.H) x[i] = ld_fresh(reinterpret_cast<const uint4*>(a.x + (size_t)token * a.H + k + i * 8u));
            }
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                mma_bf16(acc[n], lo[i].x, hi[i].x, lo[i].y, hi[i].y, x[i].x, x[i].y);
                mma_bf16(acc[n], lo[i].z, hi[i].z, lo[i].w, hi[i].w, x[i].z, x[i].w);
            }
        }
    }
    // the upper half of the warps hands its sums to the lower half, then one thread adds up an output
    for (int half = 1; half >= 0; --half) {
        if ((warp >= WARPS / 2) == (half == 1)) {
#pragma unroll
            for (uint32_t n = 0; n < MAX_TOKENS / 8u; ++n) {
                const uint32_t token = n * 8u + 2u * t;
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i)
                    if (token + (i & 1u) < a.tokens) {
                        float& p = part[warp % (WARPS / 2)][token + (i & 1u)][g + (i < 2u ? 0u : 8u)];
                        p = half ? acc[n][i] : p + acc[n][i];
                    }
            }
        }
        __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < a.tokens * 16u; i += THREADS) {
        const uint32_t token = i / 16u, e = blockIdx.x * 16u + i % 16u;
        float s = part[0][token][i % 16u];
#pragma unroll
        for (uint32_t p = 1; p < WARPS / 2; ++p) s += part[p][token][i % 16u];
        if (e < a.experts) a.logits[token * a.experts + e] = s;
    }
}

// The choice of one token by one warp.
__device__ __forceinline__ void choose(const Args& a, Tables& tb, uint32_t token, uint32_t lane) {
    constexpr int PER = MAX_EXPERTS / 32;
    const float* logits = a.logits + token * a.experts;
    float l[PER], r[PER];
    uint32_t key[PER];
    float most = -INFINITY, total = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (j * 32u >= a.experts) break;
        const uint32_t e = j * 32u + lane;
        l[j] = e < a.experts ? ld_fresh(logits + e) : -INFINITY;
        r[j] = a.bias && e < a.experts ? ld_fresh(a.bias + e) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (j * 32u < a.experts) most = fmaxf(most, l[j]);
    if (!a.sigmoid) {
#pragma unroll
        for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j * 32u < a.experts) total += j * 32u + lane < a.experts ? expf(l[j] - most) : 0.0f;
#pragma unroll
        for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
    }
    auto score = [&](float v) { return a.sigmoid ? 1.0f / (1.0f + expf(-v)) : expf(v - most) / total; };
    // without a bias the order is that of the logits, which no exponential has rounded
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        key[j] = 0u;
        if (j * 32u < a.experts) key[j] = j * 32u + lane >= a.experts || r[j] == -INFINITY ? 0u : order_key(a.bias ? score(l[j]) + r[j] : l[j]);
    }
    float mine = 0.0f;  // lane j: the j-th choice's logit
    int expert = -1;
    for (uint32_t place = 0; place < a.top; ++place) {
        uint32_t best = key[0], best_e = lane;
        float best_l = l[0];
#pragma unroll
        for (int j = 1; j < PER; ++j)
            if (key[j] > best) best = key[j], best_e = j * 32u + lane, best_l = l[j];
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
        if (top == 0u) break;
        const uint32_t e = __reduce_min_sync(0xFFFFFFFFu, best == top ? best_e : 0xFFFFFFFFu);
        const float w = __shfl_sync(0xFFFFFFFFu, best_l, e & 31u);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j * 32u + lane == e) key[j] = 0u;
        if (lane == place) mine = w, expert = (int)e;
    }
    const float p = expert >= 0 ? score(mine) : 0.0f;
    float sum = p;
#pragma unroll
    for (int d = 8; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (lane < a.top) {
        tb.chosen[token * a.top + lane] = (int16_t)expert;
        tb.weight[token * a.top + lane] = (a.norm ? p / sum : p) * a.factor;
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

// Who works on what, in every CTA the same.
__device__ __forceinline__ void make_tables(const Args& a, Tables& tb, uint32_t columns, uint32_t warp, uint32_t lane) {
    for (uint32_t e = threadIdx.x; e < a.experts; e += THREADS) tb.mask[e] = 0u;
    __syncthreads();
    for (uint32_t token = warp; token < a.tokens; token += WARPS) choose(a, tb, token, lane);
    __syncthreads();
    if (warp == 0) list_entries(a, tb, columns, lane);
    __syncthreads();
    if (threadIdx.x < a.tokens * a.top) {
        const int e = tb.chosen[threadIdx.x];
        if (e >= 0) {
            const uint32_t token = threadIdx.x / a.top, at = __popc(tb.mask[e] & ((1u << token) - 1u)), first = tb.entry_of[e];
            tb.row_token[tb.entry_row[first] + at] = (uint8_t)token;
            tb.slot[threadIdx.x] = (uint16_t)((first + at / columns) * 16u + at % columns);
        }
    }
    __syncthreads();
}

// One warp's stages: a run of tiles whose rows lie evenly apart, of one expert and one unit of K.
template <Format FMT>
struct Run {
    const uint8_t *q, *s;   // this thread's piece of the next tile
    uint32_t left = 0;      // tiles
    bool hi_there, lo_there;  // e4m3: whether the pieces lie within K

    // row: the tile's first; part: what its second eight rows lie behind the first
    __device__ __forceinline__ void begin(const Matrix& m, uint32_t e, uint32_t row, uint32_t part, uint32_t unit, uint32_t tiles, uint32_t lane) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        const size_t base = (size_t)e * m.rows + row + g;
        left = tiles;
        if constexpr (FMT == E4M3) {
            const uint32_t k = unit * UNIT + t * 32u;
            lo_there = k < m.K, hi_there = k + 16u < m.K;
            q = m.q + base * m.K + k;
            // lanes 0 and 1 fetch the scales of the tile's two halves, whose rows lie within a block each
            const uint32_t blocks = (m.rows + 127u) / 128u;
            s = m.s + (((size_t)e * blocks) * m.units + unit) * 4u;
        } else {
            constexpr uint32_t GROUP = FMT == GROUP64 ? 64 : 32;
            q = m.q + base * (m.K / 2u) + unit * 64u + t * 16u;
            // thread t of a row fetches its s, its partner's s, its b, its partner's b
            s = (t < 2u ? m.s : m.b) + ((base + (t & 1u ? part : 0u)) * (m.K / GROUP) + unit * (UNIT / GROUP)) * 2u;
        }
    }
    // row: of the tile, for the scales of e4m3; then on by `step` rows
    __device__ __forceinline__ void fetch(uint32_t stage, const Matrix& m, uint32_t row, uint32_t part, uint32_t step, uint32_t lane) {
        const uint32_t g = lane >> 2, t = lane & 3u;
        if constexpr (FMT == E4M3) {
            const uint8_t* second = q + (size_t)part * m.K;
            cp16(stage + lane * 16u, lo_there ? q : m.q, lo_there);
            cp16(stage + 512u + lane * 16u, hi_there ? q + 16 : m.q, hi_there);
            cp16(stage + 1024u + lane * 16u, lo_there ? second : m.q, lo_there);
            cp16(stage + 1536u + lane * 16u, hi_there ? second + 16 : m.q, hi_there);
            if (lane < 2u) cp4(stage + 2048u + lane * 4u, s + (size_t)((row + (lane ? part : 0u)) / 128u) * m.units * 4u);
            q += (size_t)step * m.K;
        } else {
            const uint32_t slot = (g * 4u + (t ^ chunk_swizzle<FMT>(g))) * 16u;
            constexpr uint32_t GROUP = FMT == GROUP64 ? 64 : 32;
            cp16(stage + slot, q, true);
            cp16(stage + 512u + slot, q + (size_t)part * (m.K / 2u), true);
            if constexpr (FMT == GROUP64) cp4(stage + 1024u + lane * 4u, s);
            else cp8(stage + 1024u + lane * 8u, s);
            q += (size_t)step * (m.K / 2u);
            s += (size_t)step * (m.K / GROUP) * 2u;
        }
        --left;
    }
};

template <Format FMT, int NT>
__global__ void __launch_bounds__(THREADS, 1)
moe_up_kernel(const Args a) {
    using S = Stage<FMT>;
    constexpr uint32_t COLUMNS = 8u * NT, CELL = NT * 512u;  // a tile's partial sums: NT float4 a thread
    constexpr int DEPTH = S::DEPTH;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Tables tb;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t ring = smem_addr(smem) + warp * (S::BYTES * DEPTH);
    float4* const cells = reinterpret_cast<float4*>(smem + S::RING);

    pdl_wait_prior();
    pdl_launch_dependents();  // not sooner: moe_down reads the logits before its wait
    make_tables(a, tb, COLUMNS, warp, lane);
    const uint32_t f_tiles = a.F / 8u;
    const uint64_t items = (uint64_t)tb.entries * f_tiles;
    const uint32_t i0 = (uint32_t)(items * blockIdx.x / gridDim.x), i1 = (uint32_t)(items * (blockIdx.x + 1u) / gridDim.x);
    const uint32_t slices = a.slices, groups = WARPS / slices, slice = warp % slices, group = warp / slices;
    const uint32_t per_round = a.area / (slices * CELL) / groups * groups;  // items
    // A warp goes through rounds, units of its slice, entries, items of its group.  Where the next stage to be asked for is:
    uint32_t n_first = i0, n_unit = slice, n_item = i0 + group, n_row = 0;
    Run<FMT> run;
    uint32_t put = ring, got = ring;
    const uint32_t ring_end = ring + S::BYTES * DEPTH;
    auto seek = [&]() {  // to the next run, where there is one
        while (n_first < i1) {
            const uint32_t last = min(i1, n_first + per_round);
            if (n_unit >= a.up.units) {
                n_first += per_round, n_unit = slice, n_item = n_first + group;
            } else if (n_item >= last) {
                n_unit += slices, n_item = n_first + group;
            } else {
                const uint32_t entry = n_item / f_tiles, end = min(last, (entry + 1u) * f_tiles);
                n_row = (n_item - entry * f_tiles) * 8u;
                run.begin(a.up, tb.entry_expert[entry], n_row, a.F, n_unit, (end - n_item + groups - 1u) / groups, lane);
                n_item += run.left * groups;
                return;
            }
        }
    };
    auto fill = [&]() {
        if (run.left == 0u && n_first < i1) seek();
        if (run.left) {
            run.fetch(put, a.up, n_row, a.F, groups * 8u, lane);
            n_row += groups * 8u;
        }
        cp_commit();
        put += S::BYTES;
        if (put == ring_end) put = ring;
    };
    for (int i = 0; i < DEPTH - 1; ++i) fill();
    for (uint32_t first = i0; first < i1; first += per_round) {
        const uint32_t last = min(i1, first + per_round);
        for (uint32_t unit = slice; unit < a.up.units; unit += slices) {
            for (uint32_t item = first + group; item < last;) {
                const uint32_t entry = item / f_tiles, end = min(last, (entry + 1u) * f_tiles);
                const uint32_t row0 = tb.entry_row[entry], count = tb.entry_row[entry + 1u] - row0, tiles = (count + 7u) / 8u;
                Frag<FMT, NT> f;
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
                float4* cell = cells + (((item - first) * slices + slice) * NT) * 32u + lane;
                for (; item < end; item += groups, cell += groups * slices * NT * 32u) {
                    cp_wait<DEPTH - 2>();
                    __syncwarp();
                    float o[NT][4];
                    if (NT == 1 || tiles == 1u) multiply<FMT, NT, 1>(got, f, o, lane);
                    else multiply<FMT, NT, NT>(got, f, o, lane);
                    got += S::BYTES;
                    if (got == ring_end) got = ring;
                    fill();
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
        }
        if (last == i1 && warp == 0 && lane == 0) {
            // this CTA's share of the down weights, on their way to L2 while the sums meet: whole experts' bytes, in pieces
            const size_t expert = (size_t)a.down.rows * a.down.K / (FMT == E4M3 ? 1u : 2u), all = expert * tb.entries;
            size_t at = all * blockIdx.x / gridDim.x & ~(size_t)15, to = all * (blockIdx.x + 1u) / gridDim.x & ~(size_t)15;
            if (to - at > PREFETCH) to = at + PREFETCH;
            while (at < to) {
                const size_t entry = at / expert, offset = at - entry * expert;
                const uint32_t bytes = (uint32_t)min((size_t)16384, min(to - at, expert - offset));
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.down.q + tb.entry_expert[entry] * expert + offset), "r"(bytes) : "memory");
                at += bytes;
            }
        }
        __syncthreads();
        const uint32_t used = min(slices, a.up.units);
        for (uint32_t i = threadIdx.x; i < (last - first) * CELL / 16u; i += THREADS) {
            const uint32_t at = i / (NT * 32u), n = i / 32u % NT, entry = (first + at) / f_tiles;
            const uint32_t row0 = tb.entry_row[entry], count = tb.entry_row[entry + 1u] - row0, column = n * 8u + 2u * t;
            if (column >= count) continue;
            const float4* from = cells + (at * slices * NT + n) * 32u + lane;
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
    cp_wait<0>();
}

template <Format FMT, int NT>
__global__ void __launch_bounds__(THREADS, 1)
moe_down_kernel(const Args a) {
    using S = Stage<FMT>;
    constexpr uint32_t COLUMNS = 8u * NT, WORKERS = CLUSTER * WARPS;
    constexpr int DEPTH = S::DEPTH;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Tables tb;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t rank = blockIdx.x % CLUSTER, cluster = blockIdx.x / CLUSTER;
    const uint32_t ring = smem_addr(smem) + warp * (S::BYTES * DEPTH), area = smem_addr(smem) + S::RING;
    float4* const cells = reinterpret_cast<float4*>(smem + S::RING);

    pdl_launch_dependents();
    make_tables(a, tb, COLUMNS, warp, lane);  // the logits are those of a launch that was done before moe_up let this one start
    const uint32_t units = a.down.units, all_units = tb.entries * units;
    const uint32_t r0 = cluster * a.per, r1 = min(a.H / 16u, r0 + a.per);
    // warp w of the cluster has the units [all w / 64, all (w + 1) / 64)
    const uint32_t worker = rank * WARPS + warp, u0 = all_units * worker / WORKERS, u1 = all_units * (worker + 1u) / WORKERS;
    // partial sums: a cell for each entry that a warp meets and each row tile of a pass
    const uint32_t segments = ((all_units + WORKERS - 1u) / WORKERS + units - 2u) / units + 1u;
    const uint32_t out_tile = a.tokens * 64u;  // bytes of the CTA's sums of a row tile, [token][16 rows]
    const uint32_t at_once = min(a.per, a.area / (WARPS * segments * NT * 512u + out_tile));
    float* const sums = reinterpret_cast<float*>(cells);  // in front of the cells
    float4* const mine = cells + at_once * out_tile / 16u + warp * (segments * at_once * NT * 32u) + lane;

    uint32_t n_first = r0, n_unit = u0, n_row = 0;
    Run<FMT> run;
    uint32_t put = ring, got = ring;
    const uint32_t ring_end = ring + S::BYTES * DEPTH;
    auto fill = [&]() {
        if (run.left == 0u && n_first < r1 && u0 < u1) {
            const uint32_t entry = n_unit / units;
            n_row = n_first * 16u;
            run.begin(a.down, tb.entry_expert[entry], n_row, 8u, n_unit - entry * units, min(at_once, r1 - n_first), lane);
            if (++n_unit == u1) n_unit = u0, n_first += at_once;
        }
        if (run.left) {
            run.fetch(put, a.down, n_row, 8u, 16u, lane);
            n_row += 16u;
        }
        cp_commit();
        put += S::BYTES;
        if (put == ring_end) put = ring;
    };
    for (int i = 0; i < DEPTH - 1; ++i) fill();
    pdl_wait_prior();

    for (uint32_t first = r0; first < r1; first += at_once) {
        const uint32_t last = min(r1, first + at_once);
        uint32_t segment = 0;
        for (uint32_t unit = u0; unit < u1; ++unit) {
            const uint32_t entry = unit / units, k0 = (unit - entry * units) * UNIT;
            const uint32_t row0 = tb.entry_row[entry], count = tb.entry_row[entry + 1u] - row0, tiles = (count + 7u) / 8u;
            const bool fresh = unit == u0 || k0 == 0u;  // the first unit of its entry here
            if (fresh && unit != u0) ++segment;
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
            float4* cell = mine + segment * (at_once * NT * 32u);
            for (uint32_t tile = first; tile < last; ++tile, cell += NT * 32u) {
                cp_wait<DEPTH - 2>();
                __syncwarp();
                float o[NT][4];
                if (NT == 1 || tiles == 1u) multiply<FMT, NT, 1>(got, f, o, lane);
                else multiply<FMT, NT, NT>(got, f, o, lane);
                got += S::BYTES;
                if (got == ring_end) got = ring;
                fill();
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (n && (uint32_t)n >= tiles) break;
                    float4 s = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
                    if (!fresh) {
                        const float4 p = cell[n * 32];
                        s.x += p.x, s.y += p.y, s.z += p.z, s.w += p.w;
                    }
                    cell[n * 32] = s;
                }
            }
        }
        __syncthreads();
        // a token's places, and of each the warps of this CTA that had units of its entry
        const uint32_t outputs = (last - first) * a.tokens * 16u;
        const float* const parts = reinterpret_cast<const float*>(cells + at_once * out_tile / 16u);
        for (uint32_t i = threadIdx.x; i < outputs; i += THREADS) {
            const uint32_t row = i & 15u, rest = i >> 4, tile = rest / a.tokens, token = rest - tile * a.tokens;
            float total = 0.0f;
            for (uint32_t place = 0; place < a.top; ++place) {
                const uint32_t at = token * a.top + place;
                if (tb.chosen[at] < 0) continue;
                const uint32_t entry = tb.slot[at] >> 4, column = tb.slot[at] & 15u, begin = entry * units, end = begin + units;
                // the warp that has unit u is ((u + 1) 64 - 1) / all
                const uint32_t w0 = ((begin + 1u) * WORKERS - 1u) / all_units, w1 = (end * WORKERS - 1u) / all_units;
                const uint32_t lo = max(w0, rank * WARPS), hi = min(w1, rank * WARPS + WARPS - 1u);
                float s = 0.0f;
                for (uint32_t w = lo; w <= hi && w0 <= w1; ++w) {
                    const uint32_t from = all_units * w / WORKERS;
                    if (from == all_units * (w + 1u) / WORKERS) continue;  // no units
                    const uint32_t seg = entry - from / units;
                    s += parts[(((((w - rank * WARPS) * segments + seg) * at_once + tile) * NT + column / 8u) * 32u + (row & 7u) * 4u + (column & 7u) / 2u) * 4u + (column & 1u) +
                               (row >> 3) * 2u];
                }
                total = __fmaf_rn(tb.weight[at], s, total);
            }
            sums[i] = total;
        }
        cluster_barrier();
        const uint32_t pieces = outputs / 16u, share0 = pieces * rank / CLUSTER * 16u, share1 = pieces * (rank + 1u) / CLUSTER * 16u;
        for (uint32_t i = share0 + threadIdx.x; i < share1; i += THREADS) {
            float s = remote_f32(area + i * 4u, 0);
#pragma unroll
            for (uint32_t r = 1; r < CLUSTER; ++r) s += remote_f32(area + i * 4u, r);
            const uint32_t rest = i >> 4, tile = rest / a.tokens, token = rest - tile * a.tokens;
            const size_t at = (size_t)token * a.H + (first + tile) * 16u + (i & 15u);
            if (a.bf16) static_cast<uint16_t*>(a.out)[at] = (uint16_t)pack_bf16(s, 0.0f);
            else static_cast<float*>(a.out)[at] = s;
        }
        cluster_barrier();
    }
    cp_wait<0>();
}

}  // namespace moe
}  // namespace miori_b200
