// A whole layer of experts for the tokens of a decode step, 1..32 of them:
//   l = R x;  p = softmax(l) or sigmoid(l);  the `top` experts of largest p (+ bias);  weights w = p [/ their sum] * factor
//   out[t] = sum_e w_e W_down,e (silu(g) * u),  [g; u] = W_up,e x[t]
//
// Bound by the chosen experts' weights, which are read once.  Three launches, each of which begins while the one before drains:
//   moe_router  one cluster: logits, K over its CTAs and warps, the choice of each token, and the lists that the others work from;
//   moe_up      the rows of all chosen experts' gate and up are dealt evenly to the CTAs, eight of each an MMA tile, and a CTA's tiles times K
//               evenly to its warps; a tile that several warps share meets in shared memory.  silu(g) * u goes to the workspace
//               in fp32, the largest of each row beside it;
//   moe_down    a cluster of four CTAs owns rows of the output.  The K axes of all experts, one behind the other, are dealt to its 64 warps,
//               whose sums meet by token, times w, in a CTA and then over the cluster, always in the same order.
// (As one cooperative launch with a meeting of the grid between the products, every CTA choosing for itself, a token took 23 us: such a meeting
// costs 2.6, a launch's hand-over 0.7, a choice 2.  Weights asked of L2 ahead of their kernel, up's before the choice or down's at the end of moe_up, are nobody's gain:
// a token took 18.0 us without, 18.6 with.)
// An MMA tile has eight columns: moe_up's are eight tokens, moe_down's four, each twice (below).  An expert of more tokens is listed, and read, once for every
// eight or four of them; L2 serves the further readings.
//
// Weights stream through a ring of cp.async stages that belongs to one warp: 16 rows x 128 bytes and their scales, no CTA-wide wait.  They become
// fp16 without a rounding: 4-bit codes as subnormals in the bits of a half, e4m3 by conversion; products by mma.sync.m16n8k16, sums in fp32, times
// the scales after each group.  Experts of 2048 x 1536 in 4 bits and groups of 64, 4 of 32 a token: 18.5 us for one token, of which 3.3 are the bytes' and the rest latency; 61 to 64 for 32 (25.6); in
// groups of 32 20 and 77 (3.6 and 28.4); in e4m3, 8 of 64 of 2048 x 768, 4 tokens: 39 to 40 (19).  What bounds the stream of many tokens is less HBM than the number of instructions a stage takes: B fragments are made once
// a CTA and expert (moe_up) or once for several row tiles (moe_down), a row of activations has one power of two.
// Activations, x and silu(g) * u, are fp16 times a power of two per row that puts its largest into [2^14, 2^15): bf16 x is not rounded down to
// 2^-27 of that largest (4 bits) or 2^-31.  silu(g) * u, fp32, is a pair of fp16, a value and what it has beyond that, in two columns of one tile: 2^-22 of a value at most, where one
// fp16 would be off by 2^-11 and the result by 3e-4 of its size (now 4e-6 in 4 bits, 4e-7 in e4m3).  It costs a second reading where an expert has more than four tokens: 55 us for 32 tokens
// with one fp16, 61 to 64 with the pair; one token 18.0 and 18.5.
#pragma once
#include "common.cuh"

namespace miori_b200 {
namespace moe {

constexpr uint32_t MAX_TOKENS = 32, MAX_EXPERTS = 256, MAX_TOP = 16, MAX_ROWS = MAX_TOKENS * MAX_TOP, MAX_HIDDEN = 7168, MAX_FF = 65536;
constexpr uint32_t WARPS = 16, THREADS = WARPS * 32, CLUSTER = 4, ROUTER_CLUSTER = 8;
// Tokens of an entry: the columns of an MMA tile, of which moe_down takes two a token.
constexpr uint32_t UP_ENTRY = 8, DOWN_ENTRY = 4;
constexpr uint32_t most_entries(uint32_t of) { return MAX_EXPERTS + (MAX_ROWS - MAX_EXPERTS) / of; }  // every expert one, and one more for every `of` rows beyond
constexpr uint32_t MAX_UP_ENTRIES = most_entries(UP_ENTRY), MAX_DOWN_ENTRIES = most_entries(DOWN_ENTRY);
constexpr uint32_t WORKERS = CLUSTER * WARPS;  // warps of moe_down that share the entries' units
// The most entries that one of them meets: its units are neighbours, and may begin with an entry's last.
__host__ __device__ constexpr uint32_t segments_of(uint32_t all_units, uint32_t units) {
    const uint32_t mine = (all_units + WORKERS - 1u) / WORKERS;
    return ((mine ? mine : 1u) + units - 2u) / units + 1u;
}
enum Format { GROUP64, GROUP32, E4M3 };

// A unit of K is what 128 bytes of a row hold; a stage is a unit of 16 rows.
template <Format FMT>
struct Stage {
    static constexpr uint32_t UNIT = FMT == E4M3 ? 128 : 256;
    static constexpr uint32_t CHUNK = UNIT / 8;             // elements in 16 bytes
    static constexpr int HALVES = UNIT / 128;               // B fragments are made for 128 of K
    static constexpr int GROUPS = FMT == GROUP64 ? 2 : FMT == GROUP32 ? 4 : 1;  // scale groups of a half
    static constexpr uint32_t SCALES = FMT == GROUP32 ? 512 : FMT == GROUP64 ? 256 : 128;
    static constexpr uint32_t BYTES = 2048 + SCALES;
    static constexpr int UP = 3, DOWN = 4;                  // stages of a warp's ring in moe_up and moe_down
    __host__ __device__ static constexpr uint32_t ring(int depth) { return BYTES * depth * WARPS; }
    // B fragments of a half in shared memory: four planes of 16 bytes a thread, and the sums [group][column]
    static constexpr uint32_t HALF = 2048 + (FMT == E4M3 ? 0 : GROUPS * 32);
    static constexpr uint32_t FRAG = HALVES * HALF;
};

struct Matrix {  // [experts][rows][K]
    const uint8_t* q;
    const uint8_t *s, *b;  // bf16 [experts][rows][K / group]; e4m3: s fp32 [experts][ceil(rows / 128)][ceil(K / 128)]
    uint32_t rows, K, units;
    Div by_units;
    uint32_t pitch, scale_pitch;  // bytes of a row of q, of a row of s and b
    uint32_t whole;               // rows are whole units
};
// What moe_router tells the products.
struct alignas(16) UpTables {
    uint16_t entry_expert[MAX_UP_ENTRIES], entry_row[MAX_UP_ENTRIES + 2];
    uint8_t row_token[MAX_ROWS];
    uint32_t x_top[MAX_TOKENS];       // the largest |x| of a token, as bits
    uint32_t entries;
};
struct alignas(16) DownTables {
    uint16_t entry_expert[MAX_DOWN_ENTRIES], entry_row[MAX_DOWN_ENTRIES + 2];
    int32_t chosen[MAX_ROWS];         // [token][place], -1: nobody
    float weight[MAX_ROWS];
    uint16_t slot[MAX_ROWS];          // of a place: entry * 4 + its token's number in the entry
    uint32_t entries;
};
struct Tables {
    UpTables up;
    DownTables down;
};

struct Args {
    const uint16_t *x, *router;
    const float* bias;
    Matrix up, down;
    void* out;
    Tables* tables;  // the workspace: tables, h_top, h
    uint32_t* h_top;  // the largest |h| of a row, as bits
    float* h;         // [rows][F], rows: the (expert, token) pairs in the experts' order
    float factor;
    uint32_t tokens, experts, top, H, F;
    uint32_t sigmoid, norm, bf16, ahead;  // ahead: weights may be read before the launch before is done
    Div by_tokens, by_tiles, by_ctas;  // tokens, F / 8, CTAs of moe_up
    uint32_t slots;    // moe_up: entries whose B fragments shared memory takes
    uint32_t area;     // moe_down: bytes of partial sums
    uint32_t per;      // moe_down: row tiles of a cluster
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(there ? 8u : 0u) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool there = true) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4u : 0u) : "memory");
}
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
// The first of a chain: its sum begins at zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
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

// Where K lies in a thread's fragments.  Thread (g, t) of a warp, g = lane / 4, holds of 128 of K 32 elements, the same of rows g and g + 8 of the
// weights and of column g of the activations, so that one MMA, whose k axis runs over t, stays inside a scale group.  Piece i (8 elements):
template <Format FMT>
__device__ __forceinline__ uint32_t piece_k(uint32_t t, uint32_t i) {
    return FMT == GROUP32 ? i * 32u + t * 8u : (i >> 1) * 64u + t * 16u + (i & 1u) * 8u;
}
// Chunk c (16 bytes) of row r of a stage lies at c ^ swizzle(r % 8), so that what a warp's threads read at once lies in different banks: 8 bytes of a
// quarter of the chunks and 4 rows, 4 bytes of a chunk and 8 rows, or 16 bytes of half the chunks and 2 rows.
template <Format FMT>
__device__ __forceinline__ uint32_t swizzle(uint32_t r) { return FMT == E4M3 ? (r & 1u) << 2 | r >> 1 : (r & 3u) << 1 | r >> 2; }

// What a product with 4-bit codes lacks, which are taken as multiples of 2^-24: half of its exponent goes to the sums and half to their row's power of two, whose
// exponent alone has no room for all of it where the row's largest is 2^118 or more.
template <Format FMT>
constexpr float WHOLE_ROOT = FMT == E4M3 ? 1.0f : 4096.0f;

// 2^(14 - exponent of the largest), as far as its reciprocal is a normal number; and the reciprocal.
__device__ __forceinline__ uint32_t scale_field(uint32_t top) { return min(268u - (top >> 23), 253u); }
__device__ __forceinline__ float scale_up(uint32_t top) { return __uint_as_float(scale_field(top) << 23); }
__device__ __forceinline__ float scale_down(uint32_t top) { return __uint_as_float((254u - scale_field(top)) << 23); }

// Two numbers as fp16, or what they have beyond that: exactly, before it is rounded itself.  Not two paths: a warp's lanes want both.
__device__ __forceinline__ uint32_t pack_part(float lo, float hi, bool rest) {
    const uint32_t w = pack_half(lo, hi);
    float l, h;
    asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(l), "=f"(h) : "r"(w));
    const uint32_t r = pack_half(lo - l, hi - h);
    return rest ? r : w;
}
// B fragments of eight columns and one unit.  v: the thread's 32 elements of column g, in pieces; up: the column's power of two; pack: makes fp16 of two.
template <Format FMT, class P>
__device__ __forceinline__ void make_frag(uint32_t (&b)[16], const float (&v)[32], float up, P pack) {
    if constexpr (FMT == E4M3) {
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = pack(v[2 * i] * up, v[2 * i + 1] * up);
    } else {
        // word i, codes 0..7: codes (0, 4) and (2, 6) are taken as multiples of 2^-24, (1, 5) and (3, 7) of 2^-20
        const float up16 = up * 0.0625f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            b[4 * i] = pack(v[8 * i] * up, v[8 * i + 4] * up);
            b[4 * i + 1] = pack(v[8 * i + 1] * up16, v[8 * i + 5] * up16);
            b[4 * i + 2] = pack(v[8 * i + 2] * up, v[8 * i + 6] * up);
            b[4 * i + 3] = pack(v[8 * i + 3] * up16, v[8 * i + 7] * up16);
        }
    }
}
// The columns' sums over each scale group, which the biases multiply: of the rounded values, so that a rounding counts times the weight and not
// times the code; by MMAs with rows of 1 and 16, which leave the sums of columns 2 t and 2 t + 1 with thread (g, t).  Rows of 2^-24 and 2^-20, as codes
// are, would lose what is less than 2^-19 of a column's largest, since an MMA lines up products by the exponents of normal numbers; these lose nothing to 2^-23 (measured).
template <Format FMT>
__device__ __forceinline__ void make_sums(float (&sum)[Stage<FMT>::GROUPS][2], const uint32_t (&b)[16]) {
    constexpr int G = Stage<FMT>::GROUPS, PIECES = 4 / G;
#pragma unroll
    for (int q = 0; q < G; ++q) {
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = q * PIECES * 2; i < (q + 1) * PIECES * 2; ++i) mma_f16(s, 0x3C003C00u, 0x3C003C00u, 0x4C004C00u, 0x4C004C00u, b[2 * i], b[2 * i + 1]);
        sum[q][0] = s[0] * 5.9604644775390625e-8f, sum[q][1] = s[1] * 5.9604644775390625e-8f;  // 2^-24
    }
}

// What a thread adds to a stage's address, made once: where its first chunk lies (others by exclusive or, since stages begin on 128-byte boundaries), its
// rows' scales, and where it puts what it fetches.
template <Format FMT>
struct Places {
    uint32_t chunk, scale, d0, d1;
    __device__ __forceinline__ explicit Places(uint32_t lane) {
        const uint32_t g = lane >> 2, t = lane & 3u, r = lane >> 3, c = lane & 7u;
        chunk = g * 128u + (FMT == GROUP64 ? (((t >> 1) ^ swizzle<FMT>(g)) << 4) + (t & 1u) * 8u : FMT == GROUP32 ? (swizzle<FMT>(g) << 4) + t * 4u : (t ^ swizzle<FMT>(g)) << 4);
        scale = 2048u + (FMT == E4M3 ? 0u : g * (FMT == GROUP64 ? 32u : 64u));
        d0 = r * 128u + ((c ^ swizzle<FMT>(r)) << 4), d1 = r * 128u + 512u + ((c ^ swizzle<FMT>(r + 4u)) << 4);
    }
};

// One stage times one unit of eight columns, added to tot = (row g, column 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1).
// frag(half, b, sum): the B fragments of a half.
template <Format FMT, class F>
__device__ __forceinline__ void multiply(uint32_t stage, const Places<FMT>& places, float (&tot)[4], F frag) {
    using S = Stage<FMT>;
    const uint32_t chunk = stage + places.chunk, scale = stage + places.scale;
    uint32_t b[16];
    float sum[S::GROUPS][2];
    if constexpr (FMT == E4M3) {
        float acc[2][4];
        const uint2 sc = lds64(scale);
        frag(0, b, sum);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t at = chunk ^ (c * 64u);
            const uint4 lo = lds128(at), hi = lds128(at + 1024u);
            const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a0 = e4m3_half((uint16_t)wl[i]), a1 = e4m3_half((uint16_t)wh[i]), a2 = e4m3_half((uint16_t)(wl[i] >> 16)), a3 = e4m3_half((uint16_t)(wh[i] >> 16));
                if (i == 0) mma_f16_first(acc[c], a0, a1, a2, a3, b[c * 8], b[c * 8 + 1]);
                else mma_f16(acc[c], a0, a1, a2, a3, b[c * 8 + i * 2], b[c * 8 + i * 2 + 1]);
            }
        }
        const float sl = __uint_as_float(sc.x), sh = __uint_as_float(sc.y);
        tot[0] = __fmaf_rn(sl, acc[0][0] + acc[1][0], tot[0]), tot[1] = __fmaf_rn(sl, acc[0][1] + acc[1][1], tot[1]);
        tot[2] = __fmaf_rn(sh, acc[0][2] + acc[1][2], tot[2]), tot[3] = __fmaf_rn(sh, acc[0][3] + acc[1][3], tot[3]);
    } else {
        constexpr int G = S::GROUPS, PIECES = 4 / G;
        // rows g and g + 8: scales, scales, biases, biases, a pair of groups a word
        uint32_t words[4][G];
        if constexpr (FMT == GROUP64) {
            const uint4 w = lds128(scale), z = lds128(scale + 16u);
            words[0][0] = w.x, words[0][1] = w.y, words[1][0] = w.z, words[1][1] = w.w, words[2][0] = z.x, words[2][1] = z.y, words[3][0] = z.z, words[3][1] = z.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 w = lds128(scale + i * 16u);
                words[i][0] = w.x, words[i][1] = w.y, words[i][2] = w.z, words[i][3] = w.w;
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            frag(half, b, sum);
            uint32_t lo[4], hi[4];
#pragma unroll
            for (int q = 0; q < G; ++q) {
                if constexpr (FMT == GROUP64) {
                    const uint32_t at = chunk ^ (half * 64u + q * 32u);
                    const uint2 l = lds64(at), h = lds64(at + 1024u);
                    lo[2 * q] = l.x, lo[2 * q + 1] = l.y, hi[2 * q] = h.x, hi[2 * q + 1] = h.y;
                } else {
                    const uint32_t at = chunk ^ (half * 64u + q * 16u);
                    lo[q] = lds32(at), hi[q] = lds32(at + 1024u);
                }
            }
            float acc[G][4];
            // the groups' chains of MMAs take turns
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int q = 0; q < G; ++q) {
                    const uint32_t l = lo[q * PIECES + p], h = hi[q * PIECES + p], l8 = l >> 8, h8 = h >> 8;
                    const int at = (q * PIECES + p) * 4;
                    if (p == 0) mma_f16_first(acc[q], l & 0x000F000Fu, h & 0x000F000Fu, l & 0x00F000F0u, h & 0x00F000F0u, b[at], b[at + 1]);
                    else mma_f16(acc[q], l & 0x000F000Fu, h & 0x000F000Fu, l & 0x00F000F0u, h & 0x00F000F0u, b[at], b[at + 1]);
                    mma_f16(acc[q], l8 & 0x000F000Fu, h8 & 0x000F000Fu, l8 & 0x00F000F0u, h8 & 0x00F000F0u, b[at + 2], b[at + 3]);
                }
#pragma unroll
            for (int q = 0; q < G; ++q) {
                const int group = half * G + q;
                auto value = [&](int which) { return group & 1 ? bf16hi(words[which][group >> 1]) : bf16lo(words[which][group >> 1]); };
                const float sl = value(0), sh = value(1), bl = value(2), bh = value(3);
                tot[0] = __fmaf_rn(sl, acc[q][0], __fmaf_rn(bl, sum[q][0], tot[0]));
                tot[1] = __fmaf_rn(sl, acc[q][1], __fmaf_rn(bl, sum[q][1], tot[1]));
                tot[2] = __fmaf_rn(sh, acc[q][2], __fmaf_rn(bh, sum[q][0], tot[2]));
                tot[3] = __fmaf_rn(sh, acc[q][3], __fmaf_rn(bh, sum[q][1], tot[3]));
            }
        }
    }
}

// A score as a number that grows with it; 1 for NaN, below every score.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) return 1u;
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t remote(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}

// What only moe_router works with.
struct Lists {
    Tables to;
    uint32_t mask[MAX_EXPERTS];      // tokens that chose the expert
    uint16_t entry_of[MAX_EXPERTS];  // its first entry of moe_down
};
// The choice of one token by one warp.  logit(e): the token's logit of expert e.  The results go to the lists of the cluster's first CTA.
// PER: experts of a lane.
template <int PER, class L>
__device__ __forceinline__ void choose(const Args& a, Lists& lists, uint32_t token, uint32_t lane, L logit) {
    float l[PER], r[PER];
    uint32_t key[PER];
    float most = -INFINITY, total = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (j * 32u >= a.experts) break;
        const uint32_t e = j * 32u + lane;
        r[j] = a.bias && e < a.experts ? ld_fresh(a.bias + e) : 0.0f;
        l[j] = e < a.experts ? logit(e) : -INFINITY;
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
    float p = expert >= 0 ? score(mine) : 0.0f, sum = 1.0f;
    if (a.norm) {  // as shares of the largest chosen one, e^(l - m) [/ (1 + e^l)]: scores that underflow have a sum all the same
        float m = expert >= 0 ? mine : -INFINITY;
#pragma unroll
        for (int d = 8; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
        if (expert >= 0) p = a.sigmoid ? expf(fminf(mine, 0.0f) - fminf(m, 0.0f)) / (1.0f + expf(-fabsf(mine))) : total == total ? expf(mine - m) : total;
        sum = p;
#pragma unroll
        for (int d = 8; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    }
    if (lane < a.top) {
        const uint32_t at = token * a.top + lane;
        asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(remote(smem_addr(&lists.to.down.chosen[at]), 0)), "r"(expert) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(smem_addr(&lists.to.down.weight[at]), 0)), "f"(p / sum * a.factor) : "memory");
        if (expert >= 0) asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(remote(smem_addr(&lists.mask[expert]), 0)), "r"(1u << token) : "memory");
    }
}

// Entries: the chosen experts in order, one for every eight of their tokens (moe_up) and every four (moe_down).  By one warp.
__device__ __forceinline__ void list_entries(const Args& a, Lists& lists, uint32_t lane) {
    UpTables& up = lists.to.up;
    DownTables& down = lists.to.down;
    uint32_t up_entry = 0, down_entry = 0, row = 0;
    for (uint32_t e0 = 0; e0 < a.experts; e0 += 32u) {
        const uint32_t e = e0 + lane, count = e < a.experts ? __popc(lists.mask[e]) : 0u;
        const uint32_t my_up = (count + UP_ENTRY - 1u) / UP_ENTRY, my_down = (count + DOWN_ENTRY - 1u) / DOWN_ENTRY;
        uint32_t before = my_up << 22 | my_down << 12 | count;  // three prefix sums in one: 32 experts have up to 128 and 256 entries and 512 rows
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, before, d);
            if (lane >= (uint32_t)d) before += v;
        }
        const uint32_t all = __shfl_sync(0xFFFFFFFFu, before, 31);
        const uint32_t at_up = up_entry + (before >> 22) - my_up, at_down = down_entry + (before >> 12 & 0x3FFu) - my_down, my_row = row + (before & 0xFFFu) - count;
        if (e < a.experts) lists.entry_of[e] = (uint16_t)at_down;
        for (uint32_t i = 0; i < my_down; ++i) {
            down.entry_expert[at_down + i] = (uint16_t)e;
            down.entry_row[at_down + i] = (uint16_t)(my_row + i * DOWN_ENTRY);
        }
        for (uint32_t i = 0; i < my_up; ++i) {
            up.entry_expert[at_up + i] = (uint16_t)e;
            up.entry_row[at_up + i] = (uint16_t)(my_row + i * UP_ENTRY);
        }
        up_entry += all >> 22, down_entry += all >> 12 & 0x3FFu, row += all & 0xFFFu;
    }
    if (lane == 0) up.entries = up_entry, up.entry_row[up_entry] = (uint16_t)row, down.entries = down_entry, down.entry_row[down_entry] = (uint16_t)row;
}

// Logits and choices: one cluster, whose CTAs have a share of K each for all tokens and experts, and then each their tokens.
template <int PER>
__global__ void __launch_bounds__(THREADS)
moe_router_kernel(const Args a) {
    constexpr uint32_t WIDE = PER * 2, REST = WARPS / WIDE, WIDTH = PER * 32;  // tiles of 16 experts; warps of each; experts of a plane
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Lists lists;
    float* const part = reinterpret_cast<float*>(smem);  // [slice][token][expert]
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u, rank = blockIdx.x;
    const uint32_t columns = (a.tokens + 7u) / 8u, plane = a.tokens * WIDTH;
    // a tile's warps are dealt to the tiles of eight tokens, and what is left of them to K
    const uint32_t spread = min(columns > 2u ? 4u : columns, REST), split = REST / spread;
    const uint32_t tile = warp % WIDE, turn = warp / WIDE % spread, slice = warp / WIDE / spread;
    const uint32_t units = (a.H + 127u) / 128u, u0 = rank * units / ROUTER_CLUSTER, u1 = (rank + 1u) * units / ROUTER_CLUSTER;
    const uint32_t e_lo = tile * 16u + g, e_hi = e_lo + 8u;
    uint4 lo[4], hi[4];
    auto weights = [&](uint32_t u) {
        const uint32_t k = u * 128u + t * 32u;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const bool there = u < u1 && k + i * 8u < a.H;
            lo[i] = hi[i] = make_uint4(0u, 0u, 0u, 0u);
            if (there && e_lo < a.experts) lo[i] = ld_fresh(reinterpret_cast<const uint4*>(a.router + (size_t)e_lo * a.H + k + i * 8u));
            if (there && e_hi < a.experts) hi[i] = ld_fresh(reinterpret_cast<const uint4*>(a.router + (size_t)e_hi * a.H + k + i * 8u));
        }
    };
    pdl_launch_dependents();
    if (a.ahead) weights(u0 + slice);
    uint32_t* const x_top = lists.to.up.x_top;
    for (uint32_t e = threadIdx.x; e < MAX_EXPERTS; e += THREADS) lists.mask[e] = 0u;
    if (threadIdx.x < MAX_TOKENS) x_top[threadIdx.x] = 0u;
    __syncthreads();
    pdl_wait_prior();
    if (rank == 0u && threadIdx.x < a.tokens * a.top) a.h_top[threadIdx.x] = 0u;
    for (uint32_t n = turn; n < columns; n += spread) {
        const uint32_t token = n * 8u + g, in = min(token, a.tokens - 1u);  // those behind the last are computed and not stored
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t most = 0u;
        for (uint32_t u = u0 + slice; u < u1; u += split) {
            if (n != turn || u != u0 + slice || !a.ahead) weights(u);
            const uint32_t k = u * 128u + t * 32u;
            uint4 x[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (k + i * 8u < a.H) x[i] = ld_fresh(reinterpret_cast<const uint4*>(a.x + (size_t)in * a.H + k + i * 8u));
            }
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                mma_bf16(acc, lo[i].x, hi[i].x, lo[i].y, hi[i].y, x[i].x, x[i].y);
                mma_bf16(acc, lo[i].z, hi[i].z, lo[i].w, hi[i].w, x[i].z, x[i].w);
                // magnitudes of bf16 are ordered as their bits are: the larger of each half of the words
                most = __vmaxu2(__vmaxu2(most, __vmaxu2(x[i].x & 0x7FFF7FFFu, x[i].y & 0x7FFF7FFFu)), __vmaxu2(x[i].z & 0x7FFF7FFFu, x[i].w & 0x7FFF7FFFu));
            }
        }
        if (tile == 0u) {
            most = max(most & 0xFFFFu, most >> 16) << 16;
            most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
            most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
            if (t == 0u && token < a.tokens) atomicMax(&x_top[token], most);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t of = n * 8u + 2u * t + (i & 1u);
            if (of < a.tokens) part[slice * plane + of * WIDTH + (i < 2u ? e_lo : e_hi)] = acc[i];
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < plane; i += THREADS) {
        float s = part[i];
        for (uint32_t p = 1; p < split; ++p) s += part[p * plane + i];
        part[i] = s;
    }
    cluster_barrier();
    if (rank == 0u && threadIdx.x < a.tokens) {
        uint32_t m = x_top[threadIdx.x];
#pragma unroll
        for (uint32_t r = 1; r < ROUTER_CLUSTER; ++r) m = max(m, __float_as_uint(remote_f32(smem_addr(&x_top[threadIdx.x]), r)));
        x_top[threadIdx.x] = m;
    }
    for (uint32_t token = rank + ROUTER_CLUSTER * warp; token < a.tokens; token += ROUTER_CLUSTER * WARPS)
        choose<PER>(a, lists, token, lane, [&](uint32_t e) {
            const uint32_t at = smem_addr(part + token * WIDTH + e);
            float v[ROUTER_CLUSTER], s = 0.0f;
#pragma unroll
            for (uint32_t r = 0; r < ROUTER_CLUSTER; ++r) v[r] = remote_f32(at, r);
#pragma unroll
            for (uint32_t r = 0; r < ROUTER_CLUSTER; ++r) s += v[r];
            return s;
        });
    cluster_barrier();
    if (rank) return;
    if (warp == 0) list_entries(a, lists, lane);
    __syncthreads();
    if (threadIdx.x < a.tokens * a.top) {
        const int e = lists.to.down.chosen[threadIdx.x];
        if (e >= 0) {
            const uint32_t token = threadIdx.x / a.top, at = __popc(lists.mask[e] & ((1u << token) - 1u)), first = lists.entry_of[e];
            lists.to.up.row_token[lists.to.down.entry_row[first] + at] = (uint8_t)token;
            lists.to.down.slot[threadIdx.x] = (uint16_t)(first * DOWN_ENTRY + at);
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < sizeof(Tables) / 16u; i += THREADS) reinterpret_cast<uint4*>(a.tables)[i] = reinterpret_cast<const uint4*>(&lists.to)[i];
}

template <class T>
__device__ __forceinline__ void read_tables(const T* from, T& to) {
    static_assert(sizeof(T) % 16 == 0, "copied by 16 bytes");
#pragma unroll
    for (uint32_t i = threadIdx.x; i < sizeof(T) / 16u; i += THREADS) reinterpret_cast<uint4*>(&to)[i] = ld_fresh(reinterpret_cast<const uint4*>(from) + i);
    __syncthreads();
}

// Where a warp's next stages come from: a run of them that lie evenly apart, of one expert.
template <Format FMT>
struct Run {
    using S = Stage<FMT>;
    const uint8_t *q, *s;  // this thread's piece of the next one
    uint32_t left = 0;     // stages
    uint32_t k;            // where the unit begins

    // row: the tile's first; part: what its second eight rows lie behind the first
    __device__ __forceinline__ void begin(const Matrix& m, uint32_t e, uint32_t row, uint32_t part, uint32_t unit, uint32_t stages, uint32_t lane) {
        const size_t base = (size_t)e * m.rows + row;
        left = stages;
        k = unit * S::UNIT;
        // a fetch takes four rows, eight threads a row
        q = m.q + (base + (lane >> 3)) * m.pitch + unit * 128u + (lane & 7u) * 16u;
        if constexpr (FMT == E4M3) {
            // lanes 0 and 1 fetch the scales of the tile's halves, each of which lies within a block
            const uint32_t blocks = (m.rows + 127u) / 128u;
            s = m.s + (((size_t)e * blocks + (row + (lane ? part : 0u)) / 128u) * m.units + unit) * 4u;
        } else {
            // thread (g, t): s of row g, s of its partner, b of row g, b of its partner
            const uint32_t g = lane >> 2, t = lane & 3u;
            s = (t < 2u ? m.s : m.b) + (base + g + (t & 1u ? part : 0u)) * m.scale_pitch + unit * (S::SCALES / 32u);
        }
    }
    // part: bytes from a row to its partner; then on by so many bytes, and elements of K
    __device__ __forceinline__ void fetch(uint32_t stage, const Places<FMT>& places, const Matrix& m, size_t part, uint32_t q_step, uint32_t s_step, uint32_t k_step, uint32_t lane) {
        const uint32_t d0 = stage + places.d0, d1 = stage + places.d1, to = stage + 2048u + lane * (S::SCALES / 32u);
        const uint32_t four = m.pitch * 4u;
        if (m.whole) {
            cp16(d0, q, true);
            cp16(d1, q + four, true);
            cp16(d0 + 1024u, q + part, true);
            cp16(d1 + 1024u, q + part + four, true);
            if constexpr (FMT == GROUP64) cp8(to, s, true);
            if constexpr (FMT == GROUP32) cp16(to, s, true);
        } else {  // rows may end inside the unit
            const bool there = k + (lane & 7u) * S::CHUNK < m.K;
            const uint8_t *first = there ? q : m.q, *second = there ? q + part : m.q;
            cp16(d0, first, there);
            cp16(d1, there ? first + four : first, there);
            cp16(d0 + 1024u, second, there);
            cp16(d1 + 1024u, there ? second + four : second, there);
            // the biases behind K have to be numbers: they are multiplied by sums that are zero
            const bool more = k + 128u < m.K;
            if constexpr (FMT == GROUP64) cp4(to, s), cp4(to + 4u, more ? s + 4 : s, more);
            if constexpr (FMT == GROUP32) cp8(to, s, true), cp8(to + 8u, more ? s + 8 : s, more);
            k += k_step;
        }
        if constexpr (FMT == E4M3)
            if (lane < 2u) cp4(stage + 2048u + lane * 4u, s);
        q += q_step, s += s_step;
        --left;
    }
};

// The 32 elements of 128 of K that a thread's B fragments hold of a row of x, bf16, or of h, fp32.  K, a multiple of 16, may end among them.
template <Format FMT>
__device__ __forceinline__ void read_x(float (&v)[32], const uint16_t* x, bool there, uint32_t k0, uint32_t K, uint32_t t) {
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t k = k0 + piece_k<FMT>(t, i);
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (there && k < K) w = ld_fresh(reinterpret_cast<const uint4*>(x + k));
        v[8 * i] = bf16lo(w.x), v[8 * i + 1] = bf16hi(w.x), v[8 * i + 2] = bf16lo(w.y), v[8 * i + 3] = bf16hi(w.y);
        v[8 * i + 4] = bf16lo(w.z), v[8 * i + 5] = bf16hi(w.z), v[8 * i + 6] = bf16lo(w.w), v[8 * i + 7] = bf16hi(w.w);
    }
}
template <Format FMT>
__device__ __forceinline__ void read_h(float (&v)[32], const float* h, bool there, uint32_t k0, uint32_t K, uint32_t t) {
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t k = k0 + piece_k<FMT>(t, i);
        float4 p = make_float4(0.0f, 0.0f, 0.0f, 0.0f), q = p;
        if (there && k < K) p = ld_fresh(reinterpret_cast<const float4*>(h + k)), q = ld_fresh(reinterpret_cast<const float4*>(h + k + 4u));
        v[8 * i] = p.x, v[8 * i + 1] = p.y, v[8 * i + 2] = p.z, v[8 * i + 3] = p.w, v[8 * i + 4] = q.x, v[8 * i + 5] = q.y, v[8 * i + 6] = q.z, v[8 * i + 7] = q.w;
    }
}

template <Format FMT, int DEPTH>
__global__ void __launch_bounds__(THREADS, 1)
moe_up_kernel(const Args a) {
    using S = Stage<FMT>;
    constexpr uint32_t CELL = 512u, RING = S::ring(DEPTH);  // a tile's partial sums: a float4 a thread
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ UpTables tb;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t ring = smem_addr(smem) + warp * (S::BYTES * DEPTH), ring_end = ring + S::BYTES * DEPTH;
    float4* const cells = reinterpret_cast<float4*>(smem + RING);  // two a warp
    const uint32_t frags = smem_addr(smem) + RING + 2u * WARPS * CELL;

    pdl_wait_prior();
    pdl_launch_dependents();  // not sooner: moe_down reads the tables before its wait
    read_tables(&a.tables->up, tb);
    const uint32_t f_tiles = a.F / 8u, units = a.up.units, items = tb.entries * f_tiles;
    const uint32_t i0 = a.by_ctas(items * blockIdx.x), i1 = a.by_ctas(items * (blockIdx.x + 1u));
    // A pass: as many entries as have room for their B fragments (one token: all, since theirs are the same).  Its tiles times units are
    // dealt to the warps.
    const uint32_t slots = a.tokens == 1u ? 0x10000u : a.slots;
    auto pass_end = [&](uint32_t from) { return min(i1, (a.by_tiles(from) + slots) * f_tiles); };
    auto share = [&](uint32_t from, uint32_t w) { return (pass_end(from) - from) * units * w / WARPS; };

    uint32_t n_from = i0, n_stage = 0, n_end = 0;  // the pass, stages of it to be asked for
    if (i0 < i1) n_stage = share(i0, warp), n_end = share(i0, warp + 1u);
    Run<FMT> run;
    const Places<FMT> places(lane);
    uint32_t got = ring;
    const size_t part = (size_t)a.F * a.up.pitch;
    auto fill = [&](uint32_t put) {
        if (run.left == 0u) {
            while (n_from < i1 && n_stage == n_end) {
                n_from = pass_end(n_from);
                if (n_from < i1) n_stage = share(n_from, warp), n_end = share(n_from, warp + 1u);
            }
            if (n_from < i1) {
                const uint32_t in_pass = a.up.by_units(n_stage), unit = n_stage - in_pass * units, item = n_from + in_pass, entry = a.by_tiles(item);
                run.begin(a.up, tb.entry_expert[entry], (item - entry * f_tiles) * 8u, a.F, unit, min(units - unit, n_end - n_stage), lane);
                n_stage += run.left;
            }
        }
        if (run.left) run.fetch(put, places, a.up, part, 128u, FMT == E4M3 ? 4u : S::SCALES / 32u, S::UNIT, lane);
        cp_commit();
    };
#pragma unroll 1
    for (uint32_t put = ring; put < ring_end; put += S::BYTES) fill(put);

    // silu(g) * u of a tile, whose sums are whole
    auto finish = [&](uint32_t item, const float (&tot)[4]) {
        const uint32_t entry = a.by_tiles(item), row0 = tb.entry_row[entry], count = tb.entry_row[entry + 1u] - row0;
#pragma unroll
        for (uint32_t c = 0; c < 2u; ++c) {
            const uint32_t column = 2u * t + c;
            uint32_t most = 0u;
            if (column < count) {
                const float down = scale_down(tb.x_top[tb.row_token[row0 + column]]) * WHOLE_ROOT<FMT>;
                const float gate = tot[c] * WHOLE_ROOT<FMT> * down, up = tot[2u + c] * WHOLE_ROOT<FMT> * down, h = gate / (1.0f + expf(-gate)) * up;
                a.h[(size_t)(row0 + column) * a.F + (item - entry * f_tiles) * 8u + g] = h;
                most = __float_as_uint(fabsf(h));
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
            if (g == 0u && column < count) atomicMax(a.h_top + row0 + column, most);
        }
    };

    for (uint32_t from = i0; from < i1; from = pass_end(from)) {
        const uint32_t to = pass_end(from), entry0 = a.by_tiles(from), entry1 = a.tokens == 1u ? entry0 + 1u : a.by_tiles(to - 1u) + 1u;
        for (uint32_t task = warp; task < (entry1 - entry0) * units * S::HALVES; task += WARPS) {
            const uint32_t half = task % S::HALVES, at = task / S::HALVES, slot = a.up.by_units(at), unit = at - slot * units;
            const uint32_t row0 = tb.entry_row[entry0 + slot], count = tb.entry_row[entry0 + slot + 1u] - row0;
            const uint32_t token = g < count ? tb.row_token[row0 + g] : 0u;
            float v[32];
            read_x<FMT>(v, a.x + (size_t)token * a.H, g < count, unit * S::UNIT + half * 128u, a.H, t);
            uint32_t b[16];
            make_frag<FMT>(b, v, scale_up(tb.x_top[token]), pack_half);
            const uint32_t dst = frags + task * S::HALF;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + i * 512u + lane * 16u), "r"(b[4 * i]), "r"(b[4 * i + 1]), "r"(b[4 * i + 2]), "r"(b[4 * i + 3]) : "memory");
            if constexpr (FMT != E4M3) {
                float sum[S::GROUPS][2];
                make_sums<FMT>(sum, b);
                if (g == 0u) {
#pragma unroll
                    for (int q = 0; q < S::GROUPS; ++q) asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(dst + 2048u + q * 32u + t * 8u), "f"(sum[q][0]), "f"(sum[q][1]) : "memory");
                }
            }
        }
        __syncthreads();
        const uint32_t s0 = share(from, warp), s1 = share(from, warp + 1u);
        const uint32_t t0 = a.up.by_units(s0), t1 = a.up.by_units(s1);  // its first tile of the pass, and the one that the next warp begins in
        uint32_t item = from + t0, unit = s0 - t0 * units;
        bool whole = unit == 0u, first = true;  // this warp has the tile from its first unit on; it is the warp's first
        float tot[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t stage = s0; stage < s1;) {
            const uint32_t count = min(units - unit, s1 - stage);
            uint32_t at = frags + ((a.tokens == 1u ? 0u : a.by_tiles(item) - entry0) * units + unit) * S::FRAG + lane * 16u;  // B fragments of the next unit
#pragma unroll 1
            for (uint32_t i = 0; i < count; ++i) {
                cp_wait<DEPTH - 1>();
                __syncwarp();
                multiply<FMT>(got, places, tot, [&](int half, uint32_t (&b)[16], float (&sum)[S::GROUPS][2]) {
                    const uint32_t src = at + half * S::HALF;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 w = lds128(src + i * 512u);
                        b[4 * i] = w.x, b[4 * i + 1] = w.y, b[4 * i + 2] = w.z, b[4 * i + 3] = w.w;
                    }
                    if constexpr (FMT != E4M3) {
                        const uint32_t sums = src + (2048u + t * 8u - lane * 16u);
#pragma unroll
                        for (int q = 0; q < S::GROUPS; ++q) {
                            const uint2 w = lds64(sums + q * 32u);
                            sum[q][0] = __uint_as_float(w.x), sum[q][1] = __uint_as_float(w.y);
                        }
                    }
                });
                at += S::FRAG;
                __syncwarp();  // everybody has read the stage
                fill(got);
                got += S::BYTES;
                if (got == ring_end) got = ring;
            }
            stage += count, unit += count;
            if (unit == units && whole) finish(item, tot);
            else cells[(warp * 2u + (first ? 0u : 1u)) * 32u + lane] = make_float4(tot[0], tot[1], tot[2], tot[3]);
            first = false;
            tot[0] = tot[1] = tot[2] = tot[3] = 0.0f;
            if (unit == units) ++item, unit = 0u, whole = true;
        }
        __syncthreads();
        // a tile that goes on beyond the end of the warp that began it: that warp adds up the others' cells, their first ones
        if (const uint32_t begin = t1 * units; begin >= s0 && begin < s1) {
            {
                const float4 own = cells[(warp * 2u + (t0 == t1 ? 0u : 1u)) * 32u + lane];
                tot[0] = own.x, tot[1] = own.y, tot[2] = own.z, tot[3] = own.w;
                for (uint32_t w = warp + 1u; w < WARPS && share(from, w) < begin + units; ++w) {
                    if (share(from, w) == share(from, w + 1u)) continue;
                    const float4 v = cells[w * 64u + lane];
                    tot[0] += v.x, tot[1] += v.y, tot[2] += v.z, tot[3] += v.w;
                }
                finish(from + t1, tot);
            }
        }
    }
    cp_wait<0>();
}

template <Format FMT>
__global__ void __launch_bounds__(THREADS, 1)
moe_down_kernel(const Args a) {
    using S = Stage<FMT>;
    constexpr uint32_t REST = DOWN_ENTRY / 2u * 4u;  // floats of a cell from a column to that of the rest: a float4 holds two
    constexpr int DEPTH = S::DOWN;
    constexpr uint32_t RING = S::ring(DEPTH);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ DownTables tb;
    __shared__ __align__(8) uint64_t arrived;  // the cluster's sums of this CTA's tiles
    __shared__ volatile uint32_t abort_flag;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t rank = blockIdx.x % CLUSTER, cluster = blockIdx.x / CLUSTER;
    const uint32_t ring = smem_addr(smem) + warp * (S::BYTES * DEPTH), ring_end = ring + S::BYTES * DEPTH, area = smem_addr(smem) + RING;
    float4* const cells = reinterpret_cast<float4*>(smem + RING);

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        abort_flag = 0u;
        mbar_init(smem_addr(&arrived), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    read_tables(&a.tables->down, tb);  // of a launch that was done before moe_up let this one start
    const uint32_t units = a.down.units, all_units = tb.entries * units;
    const uint32_t r0 = cluster * a.per, r1 = min(a.H / 16u, r0 + a.per);
    // warp w of the cluster has the units [all w / 64, all (w + 1) / 64)
    const uint32_t worker = rank * WARPS + warp, u0 = all_units * worker / WORKERS, u1 = all_units * (worker + 1u) / WORKERS;
    // partial sums: a cell for each entry that a warp meets and each row tile of a pass
    const uint32_t segments = segments_of(all_units, units);
    const uint32_t out_tile = a.tokens * 64u;  // bytes of a CTA's sums of a row tile, [token][16 rows]
    // in front of the cells: the four CTAs' sums of this one's tiles, every fourth of a pass
    uint32_t at_once = min(a.per, a.area / (WARPS * segments * 512u + out_tile));
    while ((at_once + CLUSTER - 1u) / CLUSTER * CLUSTER * out_tile + at_once * (WARPS * segments * 512u) > a.area) --at_once;
    const uint32_t own = (at_once + CLUSTER - 1u) / CLUSTER, front = own * CLUSTER * out_tile;
    float4* const mine = cells + front / 16u + warp * (segments * at_once * 32u) + lane;

    uint32_t n_first = r0, n_unit = u0, n_row = 0;
    Run<FMT> run;
    const Places<FMT> places(lane);
    uint32_t got = ring;
    const size_t part = (size_t)8 * a.down.pitch;
    const uint32_t q_step = 16u * a.down.pitch, s_step = FMT == E4M3 ? 0u : 16u * a.down.scale_pitch;
    auto fill = [&](uint32_t put) {
        if (run.left == 0u && n_first < r1 && u0 < u1) {
            const uint32_t entry = a.down.by_units(n_unit);
            n_row = n_first * 16u;
            run.begin(a.down, tb.entry_expert[entry], n_row, 8u, n_unit - entry * units, min(at_once, r1 - n_first), lane);
            if (++n_unit == u1) n_unit = u0, n_first += at_once;
        }
        if (run.left) {
            run.fetch(put, places, a.down, part, q_step, s_step, 0u, lane);
            if (FMT == E4M3) {  // the next block's scales every eighth tile
                n_row += 16u;
                if ((n_row & 127u) == 0u) run.s += units * 4u;
            }
        }
        cp_commit();
    };
#pragma unroll 1
    for (uint32_t put = ring; put < ring_end; put += S::BYTES) fill(put);
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    pdl_wait_prior();
    asm volatile("barrier.cluster.wait;" ::: "memory");  // the cluster's barriers exist
    // In place of a place's expert: this CTA's first warp that had units of its entry, the entry's number there, how many warps.  In place of its
    // weight that times the row's power of two.
    if (threadIdx.x < a.tokens * a.top) {
        uint32_t what = 0;
        if (tb.chosen[threadIdx.x] >= 0) {
            const uint32_t entry = tb.slot[threadIdx.x] / DOWN_ENTRY, column = tb.slot[threadIdx.x] % DOWN_ENTRY, begin = entry * units;
            // the warp that has unit u is ((u + 1) 64 - 1) / all
            const uint32_t w0 = ((begin + 1u) * WORKERS - 1u) / all_units, w1 = ((begin + units) * WORKERS - 1u) / all_units;
            const uint32_t lo = max(w0, rank * WARPS), hi = min(w1, rank * WARPS + WARPS - 1u);
            if (lo <= hi) what = (lo - rank * WARPS) | (entry - all_units * lo / WORKERS / units) << 8 | (hi - lo + 1u) << 16;
            tb.weight[threadIdx.x] *= scale_down(ld_fresh(a.h_top + tb.entry_row[entry] + column)) * WHOLE_ROOT<FMT>;
        }
        tb.chosen[threadIdx.x] = (int)what;
    }

    uint32_t parity = 0u;
    for (uint32_t first = r0; first < r1; first += at_once) {
        const uint32_t last = min(r1, first + at_once);
        uint32_t segment = 0;
        if (u0 == u1) {  // fewer units than warps: nothing to add, but it is added
            for (uint32_t i = 0; i < last - first; ++i) mine[i * 32u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        for (uint32_t unit = u0; unit < u1; ++unit) {
            const uint32_t entry = a.down.by_units(unit), k0 = (unit - entry * units) * S::UNIT;
            const uint32_t row0 = tb.entry_row[entry], count = tb.entry_row[entry + 1u] - row0;
            const bool fresh = unit == u0 || k0 == 0u;  // the first unit of its entry here
            if (fresh && unit != u0) ++segment;
            uint32_t b[S::HALVES][16];
            float sum[S::HALVES][S::GROUPS][2];
            {
                // columns 0..3: the tokens' activations as fp16; 4..7: what they have beyond that, nothing where a row has an infinity
                const uint32_t token = g % DOWN_ENTRY, row = row0 + (token < count ? token : 0u), top = ld_fresh(a.h_top + row);
                const bool rest = g >= DOWN_ENTRY, there = token < count && !(rest && top >= 0x7F800000u);
                const float up = scale_up(top);
#pragma unroll
                for (int half = 0; half < S::HALVES; ++half) {
                    float v[32];
                    read_h<FMT>(v, a.h + (size_t)row * a.F, there, k0 + half * 128u, a.F, t);
                    make_frag<FMT>(b[half], v, up, [rest](float lo, float hi) { return pack_part(lo, hi, rest); });
                    if constexpr (FMT != E4M3) make_sums<FMT>(sum[half], b[half]);
                }
            }
            float4* cell = mine + segment * (at_once * 32u);
#pragma unroll 1
            for (uint32_t tile = first; tile < last; ++tile, cell += 32u) {
                cp_wait<DEPTH - 1>();
                __syncwarp();
                float tot[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (!fresh) {
                    const float4 p = *cell;
                    tot[0] = p.x, tot[1] = p.y, tot[2] = p.z, tot[3] = p.w;
                }
                multiply<FMT>(got, places, tot, [&](int half, uint32_t (&to)[16], float (&sums_to)[S::GROUPS][2]) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) to[i] = b[half][i];
#pragma unroll
                    for (int q = 0; q < S::GROUPS; ++q) sums_to[q][0] = sum[half][q][0], sums_to[q][1] = sum[half][q][1];
                });
                *cell = make_float4(tot[0], tot[1], tot[2], tot[3]);
                __syncwarp();  // everybody has read the stage
                fill(got);
                got += S::BYTES;
                if (got == ring_end) got = ring;
            }
        }
        __syncthreads();
        // A row of a token's sums in all tiles of the pass: its places, and of each the warps of this CTA that had units of its entry, all but the first
        // of which began with it.  Few tokens' are eight threads' work each.  The sums go straight to the CTA that owns the tile.
        const uint32_t tiles = last - first, lanes = a.tokens <= 4u ? 8u : 1u, warp_floats = segments * at_once * 128u;
        const uint32_t mine_now = (tiles + CLUSTER - 1u - rank) / CLUSTER;  // of the tiles, those that are this CTA's
        const float* const parts = reinterpret_cast<const float*>(cells + front / 16u);
        if (threadIdx.x == 0) mbar_expect_tx(smem_addr(&arrived), mine_now * CLUSTER * out_tile);
        for (uint32_t i = threadIdx.x / lanes; i < a.tokens * 16u; i += THREADS / lanes) {
            const uint32_t row = i & 15u, token = i >> 4, w0 = threadIdx.x & (lanes - 1u);
            for (uint32_t t0 = 0; t0 < tiles; t0 += CLUSTER) {
                float total[CLUSTER] = {};
                for (uint32_t at = token * a.top; at < (token + 1u) * a.top; ++at) {
                    const uint32_t what = (uint32_t)tb.chosen[at], warps = what >> 16, column = tb.slot[at] % DOWN_ENTRY;
                    const float* from = parts + (what & 0xFFu) * warp_floats + (t0 * 32u + (row & 7u) * 4u + column / 2u) * 4u + (column & 1u) + (row >> 3) * 2u;
                    const float weight = tb.weight[at];
                    float s[CLUSTER] = {};
                    for (uint32_t w = w0; w < warps; w += lanes) {
                        const float* p = from + w * warp_floats + (w == 0u ? (what >> 8 & 0xFFu) * (at_once * 128u) : 0u);
#pragma unroll
                        for (uint32_t j = 0; j < CLUSTER; ++j)
                            if (t0 + j < tiles) s[j] += p[j * 128u] + p[j * 128u + REST];
                    }
                    if (warps) {
#pragma unroll
                        for (uint32_t j = 0; j < CLUSTER; ++j) total[j] = __fmaf_rn(weight, s[j] * WHOLE_ROOT<FMT>, total[j]);
                    }
                }
                if (lanes == 8u) {  // whole warps: 16 rows a token
#pragma unroll
                    for (uint32_t d = 1; d < 8u; d *= 2u)
#pragma unroll
                        for (uint32_t j = 0; j < CLUSTER; ++j) total[j] += __shfl_xor_sync(0xFFFFFFFFu, total[j], d);
                }
                if (w0 == 0u) {
#pragma unroll
                    for (uint32_t j = 0; j < CLUSTER; ++j)
                        if (t0 + j < tiles)
                            asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];"
                                         ::"r"(remote(area + ((rank * own + t0 / CLUSTER) * a.tokens * 16u + i) * 4u, j)), "r"(__float_as_uint(total[j])), "r"(remote(smem_addr(&arrived), j)) : "memory");
                }
            }
        }
        // No CTA leaves, or sends a next pass's sums, before all have come this far; on the last pass that is said before they are waited for.
        if (last >= r1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
        if (mine_now) {
            const bool ok = mbar_wait<true, Order::CLUSTER>(smem_addr(&arrived), parity, &abort_flag, 0x81);
            for (uint32_t i = threadIdx.x; ok && i < mine_now * a.tokens * 16u; i += THREADS) {
                const uint32_t rest = i >> 4, q = a.by_tokens(rest), token = rest - q * a.tokens;
                float v = 0.0f;
#pragma unroll
                for (uint32_t r = 0; r < CLUSTER; ++r) {
                    const float w = reinterpret_cast<const float*>(cells)[r * own * a.tokens * 16u + i];
                    v = r ? v + w : w;
                }
                const size_t at = (size_t)token * a.H + (first + q * CLUSTER + rank) * 16u + (i & 15u);
                if (a.bf16) static_cast<uint16_t*>(a.out)[at] = (uint16_t)pack_bf16(v, 0.0f);
                else static_cast<float*>(a.out)[at] = v;
            }
        }
        parity ^= 1u;
        if (last < r1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait;" ::: "memory");
    }
    cp_wait<0>();
}

}  // namespace moe
}  // namespace miori_b200
