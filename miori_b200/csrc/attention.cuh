// What the attention kernels share: their arguments, how a launch's work is dealt out, and how parts of it meet again.
//
//   o[i] = sum_j softmax_j(scale * q_i . k_j) * v_j     over the positions j <= length - n + i that token i of n sees
//
// The kernels (attention_decode.cuh, attention_prompt.cuh, attention_short.cuh) go over the keys once with the running maximum m and sum l of a
// softmax, fp32: with t = scale * log2(e) * q . k, m' = max(m, t), l' = l * 2^(m - m') + sum 2^(t - m'), and o likewise.  A
// row's keys may be split over CTAs: parts (m, l, o) of a row join as o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p.
//
// An item is a block of a request's tokens with one key head: all the query heads that share the head are rows of the item
// (row = token * group + head), so keys and values are read once for all of them.  An item's work is known on the device alone
// (lengths live there: a recorded graph serves every step), so the decode and the prompt kernel are a fixed number of CTAs, and each
// finds its share by the same arithmetic: an item costs the positions that it goes over and a constant more for its beginning and
// end, and share k of G is units [k * size, (k + 1) * size) of all items' costs, in order, with size = ceil(total / G) and a tile of keys
// at least.  The last shares may be shorter or empty.  That needs no list and no counter.  Without a workspace an item stays whole and belongs
// to the share that holds its first tile.  The short kernel is dealt by its grid.
#pragma once
#include "common.cuh"

namespace miori_b200 {
namespace attention {

struct Args {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    const int32_t *cu, *lens, *table;  // lens: positions of each request (paged) or first position of each (cu_k, packed)
    int64_t q_token, q_head, o_token, o_head;
    int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;  // packed: slot is the token's stride, page unused
    uint32_t requests, heads, kv_heads, group, tokens, keys;   // tokens, keys: rows of q and of packed k
    uint32_t width, page_shift, pages;                           // of the table; page size as a power of two
    uint32_t causal;
    float scale_log2;  // scale * log2(e)
    // workspace, all null without one: then items are not split
    uint32_t* counters;  // of CTAs that are done with an item (decode)
    uint4* joins;        // what is to be added up behind the prompt kernel
    float* parts;
};

__device__ __forceinline__ float exp2_fast(float x) {  // 2^x, 2 ulp, 0 for x = -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A pair of bf16 added up in fp32 without being unpacked: the lower to x and the upper to y, or both to one sum.
__device__ __forceinline__ void add_bf16(float& x, float& y, uint32_t pair) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tadd.rn.f32.bf16 %0, lo, %0;\n\tadd.rn.f32.bf16 %1, hi, %1;\n\t}" : "+f"(x), "+f"(y) : "r"(pair));
}
__device__ __forceinline__ float add_bf16(float sum, uint32_t pair) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tadd.rn.f32.bf16 %0, lo, %0;\n\tadd.rn.f32.bf16 %0, hi, %0;\n\t}" : "+f"(sum) : "r"(pair));
    return sum;
}
// Bits of a pair of bf16 with those halves zero that are not finite.
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t pair) {
    if ((pair & 0x7F80u) == 0x7F80u) pair &= 0xFFFF0000u;
    if ((pair & 0x7F800000u) == 0x7F800000u) pair &= 0x0000FFFFu;
    return pair;
}

// A request as the kernels see it.  Lengths that contradict one another are cut off to what is there: no row of q or k beyond
// the tensors, no column beyond the table is ever read.  Where its tokens stand is another matter: that follows from the
// lengths as they were given, or the tokens that are there would see positions that are not theirs.
struct Request {
    uint32_t q0, n;   // first token in q, number of tokens
    uint32_t k0, len;  // first row of packed k (0 where paged), number of positions
    int32_t before;     // positions in front of the first token (n > 0)
};
template <bool PAGED>
__device__ __forceinline__ Request request(const Args& a, uint32_t r) {
    Request x;
    const int32_t q0 = ld_fresh(a.cu + r), q1 = ld_fresh(a.cu + r + 1);
    x.q0 = min((uint32_t)max(q0, 0), a.tokens);
    x.n = min((uint32_t)max(q1, 0), a.tokens);
    x.n = x.n > x.q0 ? x.n - x.q0 : 0u;
    if constexpr (PAGED) {
        x.k0 = 0u;
        const uint64_t room = (uint64_t)a.width << a.page_shift;
        x.len = (uint32_t)max(ld_fresh(a.lens + r), 0);
        x.before = (int32_t)(x.len - (uint32_t)max(q1, 0) + x.q0);  // 2^32 drops off: where n > 0 it is within -2^31 .. 2^31
        if ((uint64_t)x.len > room) x.len = (uint32_t)room;
    } else {
        const uint32_t k0 = (uint32_t)max(ld_fresh(a.lens + r), 0), k1 = (uint32_t)max(ld_fresh(a.lens + r + 1), 0);
        x.before = (int32_t)((k1 > k0 ? k1 - k0 : 0u) - (uint32_t)max(q1, 0) + x.q0);
        x.k0 = min(k0, a.keys);
        x.len = min(k1, a.keys);
        x.len = x.len > x.k0 ? x.len - x.k0 : 0u;
    }
    return x;
}
// Positions that token i of the request sees.
__device__ __forceinline__ uint32_t seen(const Args& a, const Request& x, uint32_t i) {
    if (!a.causal) return x.len;
    const int64_t s = (int64_t)x.before + (int64_t)i + 1;
    return s <= 0 ? 0u : min((uint32_t)s, x.len);
}

// `total` units cut into shares of the same length, at least `least` and no more of them than CTAs; the last one may be shorter.
// None before it is empty: whoever adds parts up counts on every CTA between the first and the last of an item.
struct Shares {
    uint64_t total, size;
    __device__ __forceinline__ Shares(uint64_t total_, uint32_t ctas, uint32_t least) : total(total_) {
        // both branches, since a division of 64 bits costs a few hundred cycles
        if (total >> 32) size = (total + ctas - 1u) / ctas;
        else size = ((uint32_t)total + (uint64_t)ctas - 1u) >> 32 ? (total + ctas - 1u) / ctas : ((uint32_t)total + ctas - 1u) / ctas;
        size = max(size, (uint64_t)least);
    }
    __device__ __forceinline__ uint64_t begin(uint32_t k) const { return min(k * size, total); }
    __device__ __forceinline__ uint32_t of(uint64_t unit) const { return (uint32_t)(unit / size); }
};
// a / b where the result is small: no division of 64 bits.
template <class U>
__device__ __forceinline__ uint32_t small_quotient(U a, U b) {
    uint32_t q = (uint32_t)__fdividef((float)a, (float)b);  // off by one at most below 2^20
    while ((uint64_t)q * b > a) --q;
    while (a - q * b >= b) ++q;
    return q;
}
// Sum over a warp of numbers below 2^51.
__device__ __forceinline__ uint64_t warp_sum(uint64_t x) {
    return __reduce_add_sync(0xFFFFFFFFu, (uint32_t)x & 0xFFFFFFu) + ((uint64_t)__reduce_add_sync(0xFFFFFFFFu, (uint32_t)(x >> 24)) << 24);
}
template <class U>
__device__ __forceinline__ U warp_prefix_sum(U x) {  // inclusive
#pragma unroll
    for (uint32_t o = 1; o < 32u; o <<= 1) {
        const U y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if ((threadIdx.x & 31u) >= o) x += y;
    }
    return x;
}

}  // namespace attention
}  // namespace miori_b200
