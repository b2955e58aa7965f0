// Entries of the attention operators: argument checks, tensor maps, and which kernel takes a call.
//   attention_paged   queries of a step against the page cache   (reference, one request at a time over a contiguous cache:
//                     attn_decode, attn_decode_split + attn_combine, shaders/ops.metal:392-436,635-710)
//   attention_prompt  packed prompts against their own keys         (reference, 16 heads of gemm_naive, softmax_prefill and
//                     gemm_naive per layer: src/engine.cpp:582-601)
#include "attention.cuh"
#include "attention_decode.cuh"
#include "attention_prompt.cuh"
#include "attention_short.cuh"

#include <cmath>

namespace miori_b200 {
namespace attention {

// Rows of an item (new tokens x heads that share a key head) up to which the decode kernel takes a call, by the size of a head.  us in a
// graph, decode against prompt kernel.  16 rows of 128: a request of 1000 positions 11.8, 14.4; 8 of 1000 13.1, 18.5; 32 of 4000 52.3, 62.2, with
// heads that share nothing 93.2, 105.  32 rows of 64: 8 of 1000 17.0, 18.7; 9 of 3000 25.4, 29.6; 32 of 4000 76.7, 94.1.  With 32 rows
// of 128 the decode kernel has no registers left (32 of 4000: 115 when it was tried, 69).
constexpr uint32_t DECODE_ROWS_128 = 16, DECODE_ROWS_64 = 32;
// Packed calls that the short kernel takes: up to 512 tokens (and keys), or up to 2048 of prompts of 64 on average.  us in a graph, short
// against prompt kernel, 16 heads of 128 over 4: one prompt of 77 6.5, 10.0, of 256 10.7, 17.2, of 448 17.6, 19.2, of 512 21, 19 (where 2 of 256
// are 12.5, 18.2: the host knows the sum only), of 1024 39, 24.5; 32 of 32 7.4, 12.0; 32 of 64 13.2, 13.4; 2 of 512 22.3, 21.5.  32 heads of
// 64 over 8: one of 512 18.3, 17.1; 32 of 64 14.4, 16.8.  16 heads of 64 that share nothing: one of 512 14.8, 15.7; 32 of 64 9.9, 23.4.
static bool takes_short(uint32_t tokens, uint32_t keys, uint32_t requests) {
    const uint32_t most = tokens > keys ? tokens : keys;
    return most <= 512u || (most <= 2048u && most <= 64u * requests);
}
constexpr size_t COUNTER_BYTES = 4096, JOIN_BYTES = 12288;  // for up to 768 SMs
static size_t part_bytes() { return 2u * (size_t)sm_count() * PromptCfg<128>::PART_FLOATS * 4u; }

static int make_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const int64_t* strides, const uint32_t* box) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(MIORI_E_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
    cuuint64_t d[4], s[3];
    cuuint32_t b[4], e[4];
    for (int i = 0; i < rank; ++i) d[i] = dims[i], b[i] = box[i], e[i] = 1;
    for (int i = 0; i + 1 < rank; ++i) s[i] = (cuuint64_t)strides[i] * 2u;
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), d, s, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? MIORI_OK : fail(MIORI_E_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

// What both entries ask of their arguments.
static int check_common(const char* fn, const void* q, const void* k, const void* v, const void* out, const int64_t* strides, int n_strides,
                        uint32_t requests, uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t dim, float scale, const void* workspace,
                        size_t workspace_bytes) {
    if (requests == 0 || tokens == 0 || heads == 0 || kv_heads == 0)
        return fail(MIORI_E_INVALID, "%s: empty shape (requests=%u tokens=%u heads=%u kv_heads=%u)", fn, requests, tokens, heads, kv_heads);
    if (!q || !k || !v || !out || !strides) return fail(MIORI_E_INVALID, "%s: null pointer", fn);
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return fail(MIORI_E_INVALID, "%s: pointers must be 16-byte aligned", fn);
    if (requests > 65535u || tokens > 0x3FFFFFFFu) return fail(MIORI_E_INVALID, "%s: at most 65535 requests and 2^30 tokens", fn);
    if (dim != 64 && dim != 128) return fail(MIORI_E_INVALID, "%s: heads of 64 or 128, got %u", fn, dim);
    if (heads % kv_heads) return fail(MIORI_E_INVALID, "%s: %u heads do not share %u key heads evenly", fn, heads, kv_heads);
    if (heads / kv_heads > 64u) return fail(MIORI_E_INVALID, "%s: at most 64 heads share a key head, got %u", fn, heads / kv_heads);
    if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(MIORI_E_INVALID, "%s: the scale must be positive and finite", fn);
    for (int i = 0; i < n_strides; ++i)
        if (strides[i] <= 0 || strides[i] % 8 || strides[i] >= (1ll << 38))
            return fail(MIORI_E_INVALID, "%s: strides must be positive multiples of 8 elements below 2^38, got %lld", fn, (long long)strides[i]);
    if (workspace && (!aligned16(workspace) || workspace_bytes < miori_attention_workspace_bytes()))
        return fail(MIORI_E_INVALID, "%s: a workspace of %zu bytes, 16-byte aligned, is needed", fn, miori_attention_workspace_bytes());
    return MIORI_OK;
}

static void use_workspace(Args& a, void* workspace) {
    if (!workspace) return;
    a.counters = (uint32_t*)workspace;
    a.joins = (uint4*)((char*)workspace + COUNTER_BYTES);
    a.parts = (float*)((char*)workspace + COUNTER_BYTES + JOIN_BYTES);
}

// No kernel here reads or writes anything ahead of its wait for the launch before, so every launch may begin beside that one, whatever the flags
// say (one stream's decode 10.2 us a call without).
template <int D, bool PAGED>
static int launch_prompt(const Args& a, bool may_split, cudaStream_t stream) {
    CUtensorMap mq, mk, mv;
    const uint32_t per_tile = ROW_TILE / a.group;
    {
        const uint64_t d[3] = {(uint64_t)D, a.heads, a.tokens};
        const int64_t s[2] = {a.q_head, a.q_token};
        const uint32_t b[3] = {64, a.group, per_tile};
        if (const int rc = make_map(&mq, a.q, 3, d, s, b)) return rc;
    }
    for (int i = 0; i < 2; ++i) {
        CUtensorMap* m = i ? &mv : &mk;
        const void* base = i ? a.v : a.k;
        const int64_t slot = i ? a.v_slot : a.k_slot, head = i ? a.v_head : a.k_head, page = i ? a.v_page : a.k_page;
        int rc;
        if (PAGED) {
            const uint64_t d[4] = {(uint64_t)D, 1ull << a.page_shift, a.kv_heads, a.pages};
            const int64_t s[3] = {slot, head, page};
            const uint32_t b[4] = {64, (1u << a.page_shift) < (uint32_t)KEYS ? 1u << a.page_shift : (uint32_t)KEYS, 1, 1};
            rc = make_map(m, base, 4, d, s, b);
        } else {
            const uint64_t d[3] = {(uint64_t)D, a.kv_heads, a.keys};
            const int64_t s[2] = {head, slot};
            const uint32_t b[3] = {64, 1, (uint32_t)KEYS};
            rc = make_map(m, base, 3, d, s, b);
        }
        if (rc) return rc;
    }
    const uint32_t G = (uint32_t)sm_count();
    cudaError_t e = launch(attention_prompt_kernel<D, PAGED>, dim3(G), dim3(PROMPT_THREADS), PromptCfg<D>::SMEM, stream, true, mq, mk, mv, a);
    if (e != cudaSuccess) return cuda_fail(e, "attention_prompt launch");
    if (a.parts && may_split) {
        e = launch(attention_join_kernel<D>, dim3(G, 2 * ROW_TILE / JOIN_ROWS), dim3(JOIN_THREADS), 0, stream, true, a);
        if (e != cudaSuccess) return cuda_fail(e, "attention_join launch");
    }
    return MIORI_OK;
}

template <int D>
static int launch_decode(const Args& a, uint32_t rows, cudaStream_t stream) {
    const dim3 grid((uint32_t)sm_count()), block(DECODE_THREADS);
    cudaError_t e = cudaSuccess;
    if (rows <= 8u) e = launch(attention_decode_kernel<D, 1>, grid, block, DecodeCfg<D, 1>::SMEM, stream, true, a);
    else if (rows <= 16u) e = launch(attention_decode_kernel<D, 2>, grid, block, DecodeCfg<D, 2>::SMEM, stream, true, a);
    else if constexpr (D == 64) e = launch(attention_decode_kernel<D, 4>, grid, block, DecodeCfg<D, 4>::SMEM, stream, true, a);
    return e == cudaSuccess ? MIORI_OK : cuda_fail(e, "attention_decode launch");
}

template <int D>
static int launch_short(const Args& a, cudaStream_t stream) {
    const uint32_t per_block = SHORT_ROWS / a.group;
    const dim3 grid((a.tokens + per_block - 1u) / per_block + a.requests, a.kv_heads);
    const cudaError_t e = launch(attention_short_kernel<D>, grid, dim3(SHORT_THREADS), ShortCfg<D>::SMEM, stream, true, a);
    return e == cudaSuccess ? MIORI_OK : cuda_fail(e, "attention_short launch");
}

}  // namespace attention
}  // namespace miori_b200

using namespace miori_b200;

MIORI_API size_t miori_attention_workspace_bytes(void) { return attention::COUNTER_BYTES + attention::JOIN_BYTES + attention::part_bytes(); }

MIORI_API int miori_attention_paged(const void* q, const void* k_cache, const void* v_cache, void* out, const int64_t* strides,
                                    const int32_t* table, const int32_t* lens, const int32_t* cu, uint32_t requests, uint32_t tokens,
                                    uint32_t width, uint32_t pages, uint32_t page, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                                    uint32_t max_new, float scale, uint32_t flags, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace attention;
    if (const int rc = check_common("attention_paged", q, k_cache, v_cache, out, strides, 10, requests, tokens, heads, kv_heads, dim, scale, workspace, workspace_bytes))
        return rc;
    if (!table || !lens || !cu) return fail(MIORI_E_INVALID, "attention_paged: null pointer");
    if (width == 0 || pages == 0) return fail(MIORI_E_INVALID, "attention_paged: empty table or cache (width=%u pages=%u)", width, pages);
    if (page < 8 || (page & (page - 1)) || page > 65536) return fail(MIORI_E_INVALID, "attention_paged: pages of a power of two from 8 to 65536 positions, got %u", page);
    if (pages > 0x7FFFFFFFu) return fail(MIORI_E_INVALID, "attention_paged: too many pages");
    if ((uint64_t)width * page > 0x7FFFFF00ull) return fail(MIORI_E_INVALID, "attention_paged: a table of 2^31 positions or more");
    Args a = {};
    a.q = (const uint16_t*)q, a.k = (const uint16_t*)k_cache, a.v = (const uint16_t*)v_cache, a.out = (uint16_t*)out;
    a.cu = cu, a.lens = lens, a.table = table;
    a.q_token = strides[0], a.q_head = strides[1], a.o_token = strides[2], a.o_head = strides[3];
    a.k_page = strides[4], a.k_head = strides[5], a.k_slot = strides[6], a.v_page = strides[7], a.v_head = strides[8], a.v_slot = strides[9];
    a.requests = requests, a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.tokens = tokens, a.width = width, a.pages = pages;
    while ((1u << a.page_shift) < page) ++a.page_shift;
    a.causal = (flags & MIORI_ATTENTION_FULL) == 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    use_workspace(a, workspace);
    const uint64_t rows = (uint64_t)(max_new ? max_new : 1u) * a.group;
    const cudaStream_t s = (cudaStream_t)stream;
    if (rows <= (dim == 128 ? DECODE_ROWS_128 : DECODE_ROWS_64)) return dim == 128 ? launch_decode<128>(a, (uint32_t)rows, s) : launch_decode<64>(a, (uint32_t)rows, s);
    const bool may_split = (uint64_t)width * page > KEYS;
    return dim == 128 ? launch_prompt<128, true>(a, may_split, s) : launch_prompt<64, true>(a, may_split, s);
}

MIORI_API int miori_attention_prompt(const void* q, const void* k, const void* v, void* out, const int64_t* strides, const int32_t* cu,
                                     const int32_t* cu_k, uint32_t requests, uint32_t tokens, uint32_t keys, uint32_t heads, uint32_t kv_heads,
                                     uint32_t dim, float scale, uint32_t flags, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace attention;
    if (const int rc = check_common("attention_prompt", q, k, v, out, strides, 8, requests, tokens, heads, kv_heads, dim, scale, workspace, workspace_bytes)) return rc;
    if (!cu) return fail(MIORI_E_INVALID, "attention_prompt: null pointer");
    if (keys == 0 || keys > 0x3FFFFFFFu) return fail(MIORI_E_INVALID, "attention_prompt: 1..2^30 keys, got %u", keys);
    Args a = {};
    a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v, a.out = (uint16_t*)out;
    a.cu = cu, a.lens = cu_k ? cu_k : cu;
    a.q_token = strides[0], a.q_head = strides[1], a.o_token = strides[2], a.o_head = strides[3];
    a.k_slot = strides[4], a.k_head = strides[5], a.v_slot = strides[6], a.v_head = strides[7];
    a.requests = requests, a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.tokens = tokens, a.keys = keys;
    a.causal = (flags & MIORI_ATTENTION_FULL) == 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    use_workspace(a, workspace);
    if (takes_short(tokens, keys, requests) && kv_heads <= 65535u)
        return dim == 128 ? launch_short<128>(a, (cudaStream_t)stream) : launch_short<64>(a, (cudaStream_t)stream);
    const bool may_split = keys > (uint32_t)KEYS;
    return dim == 128 ? launch_prompt<128, false>(a, may_split, (cudaStream_t)stream) : launch_prompt<64, false>(a, may_split, (cudaStream_t)stream);
}
