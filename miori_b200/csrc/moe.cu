// Entries of the layers of experts: argument checks, the kernel's shape, the launch.  (The reference's models have dense feed-forwards:
// gate + up, silu_mul and down as separate dispatches, src/engine.cpp:484-502.)
#include "moe.cuh"

#include <cmath>

namespace miori_b200 {
namespace moe {

// fp32 values of the workspace in front of the activations
static size_t logits_room(uint32_t tokens, uint32_t experts) { return ((size_t)tokens * experts + 31) / 32 * 32; }

// Warps over K in gate + up: as many as leave few of them without a unit, or with one less than others.
static uint32_t slices_for(uint32_t units) {
    uint32_t best = 1, best_waste = ~0u;
    for (uint32_t s = WARPS; s; s /= 2u) {
        const uint32_t waste = ((units + s - 1u) / s * s - units) * 1000u / units;
        if (waste < best_waste) best = s, best_waste = waste;
    }
    return best;
}

template <Format FMT, int NT>
static int launch_moe(const char* op, Args a, cudaStream_t stream) {
    // all of an SM's shared memory: the ring, and partial sums in the rest
    constexpr size_t smem = 227 * 1024 - (sizeof(Tables) + 127) / 128 * 128;
    a.area = (uint32_t)(smem - Stage<FMT>::RING);
    static_assert(smem - Stage<FMT>::RING >= WARPS * NT * 512u * 5u + MAX_TOKENS * 64u, "cells of a row tile for five entries a warp (288 of one unit each), and its sums");
    a.slices = slices_for(a.up.units);
    const uint32_t sms = (uint32_t)sm_count(), row_tiles = a.H / 16u;
    // clusters of four whole SMs: an SM in nine has no place in one
    const uint32_t most = sms * 8u / 9u / CLUSTER;
    a.per = (row_tiles + most - 1u) / most;
    cudaError_t e = launch(moe_router_kernel, dim3((a.experts + 15u) / 16u), dim3(THREADS), 0, stream, true, a);
    if (e == cudaSuccess) e = launch(moe_up_kernel<FMT, NT>, dim3(sms), dim3(THREADS), smem, stream, true, a);
    if (e == cudaSuccess) e = launch_cluster(moe_down_kernel<FMT, NT>, (row_tiles + a.per - 1u) / a.per * CLUSTER, THREADS, smem, CLUSTER, stream, a);
    return e == cudaSuccess ? MIORI_OK : cuda_fail(e, op);
}

static int check_common(const char* op, const void* x, const void* router, const void* out, uint32_t tokens, uint32_t experts, uint32_t top, uint32_t hidden, uint32_t ff,
                        uint32_t step, float factor, const float* bias, const void* workspace, size_t workspace_bytes) {
    if (!x || !router || !out || !workspace) return fail(MIORI_E_INVALID, "%s: null pointer", op);
    if (tokens == 0 || tokens > MAX_TOKENS) return fail(MIORI_E_INVALID, "%s: 1..%u tokens, got %u", op, MAX_TOKENS, tokens);
    if (experts == 0 || experts > MAX_EXPERTS) return fail(MIORI_E_INVALID, "%s: 1..%u experts, got %u", op, MAX_EXPERTS, experts);
    if (top == 0 || top > MAX_TOP || top > experts) return fail(MIORI_E_INVALID, "%s: 1..%u of %u experts for a token, got %u", op, MAX_TOP, experts, top);
    if (hidden == 0 || ff == 0 || hidden % step || ff % step)
        return fail(MIORI_E_INVALID, "%s: hidden and ff are multiples of %u, got %u and %u", op, step, hidden, ff);
    if (hidden > 65536u || ff > 65536u) return fail(MIORI_E_INVALID, "%s: hidden and ff are at most 65536, got %u and %u", op, hidden, ff);
    if (!std::isfinite(factor)) return fail(MIORI_E_INVALID, "%s: the factor must be finite", op);
    if (!aligned16(x) || !aligned16(router) || !aligned16(out) || !aligned16(workspace) || (reinterpret_cast<uintptr_t>(bias) & 3u))
        return fail(MIORI_E_INVALID, "%s: x, router, out and workspace must be 16-byte aligned, bias by its elements", op);
    if (workspace_bytes < miori_moe_workspace_bytes(tokens, experts, top, ff))
        return fail(MIORI_E_INVALID, "%s: a workspace of %zu bytes is needed, got %zu", op, miori_moe_workspace_bytes(tokens, experts, top, ff), workspace_bytes);
    return MIORI_OK;
}

static Args common_args(const void* x, const void* router, const float* bias, void* out, uint32_t tokens, uint32_t experts, uint32_t top, uint32_t hidden, uint32_t ff,
                        float factor, uint32_t flags, void* workspace) {
    Args a = {};
    a.x = static_cast<const uint16_t*>(x), a.router = static_cast<const uint16_t*>(router), a.bias = bias, a.out = out;
    a.logits = static_cast<float*>(workspace);
    a.h = a.logits + logits_room(tokens, experts);
    a.ahead = flags & MIORI_LAUNCH_PDL ? 1u : 0u;
    a.factor = factor, a.tokens = tokens, a.experts = experts, a.top = top, a.H = hidden, a.F = ff;
    a.sigmoid = flags & MIORI_MOE_SIGMOID ? 1u : 0u, a.norm = flags & MIORI_MOE_NORM ? 1u : 0u, a.bf16 = flags & MIORI_OUT_BF16 ? 1u : 0u;
    auto matrix = [](Matrix& m, uint32_t rows, uint32_t K) { m.rows = rows, m.K = K, m.units = (K + UNIT - 1u) / UNIT; };
    matrix(a.up, 2u * ff, hidden);
    matrix(a.down, hidden, ff);
    return a;
}

}  // namespace moe
}  // namespace miori_b200

using namespace miori_b200;

MIORI_API size_t miori_moe_workspace_bytes(uint32_t tokens, uint32_t experts, uint32_t top, uint32_t ff) {
    return (moe::logits_room(tokens, experts) + (size_t)tokens * top * ff) * sizeof(float);
}

MIORI_API int miori_moe4(const void* x, const void* router, const float* bias, const void* q_up, const void* s_up, const void* b_up, const void* q_down,
                         const void* s_down, const void* b_down, void* out, uint32_t tokens, uint32_t experts, uint32_t top, uint32_t hidden, uint32_t ff,
                         uint32_t group, float factor, uint32_t flags, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace moe;
    const char* op = "miori_moe4";
    if (!q_up || !s_up || !b_up || !q_down || !s_down || !b_down) return fail(MIORI_E_INVALID, "%s: null weight pointer", op);
    if (group != 32 && group != 64) return fail(MIORI_E_INVALID, "%s: group must be 32 or 64 (got %u)", op, group);
    if (const int rc = check_common(op, x, router, out, tokens, experts, top, hidden, ff, UNIT, factor, bias, workspace, workspace_bytes)) return rc;
    for (const void* p : {q_up, s_up, b_up, q_down, s_down, b_down})
        if (!aligned16(p)) return fail(MIORI_E_INVALID, "%s: weights must be 16-byte aligned", op);
    Args a = common_args(x, router, bias, out, tokens, experts, top, hidden, ff, factor, flags, workspace);
    auto u8 = [](const void* p) { return static_cast<const uint8_t*>(p); };
    a.up.q = u8(q_up), a.up.s = u8(s_up), a.up.b = u8(b_up), a.down.q = u8(q_down), a.down.s = u8(s_down), a.down.b = u8(b_down);
    const cudaStream_t s = (cudaStream_t)stream;
    if (group == 64) return tokens <= 8 ? launch_moe<GROUP64, 1>(op, a, s) : launch_moe<GROUP64, 2>(op, a, s);
    return tokens <= 8 ? launch_moe<GROUP32, 1>(op, a, s) : launch_moe<GROUP32, 2>(op, a, s);
}

MIORI_API int miori_moe_fp8(const void* x, const void* router, const float* bias, const void* w_up, const float* s_up, const void* w_down, const float* s_down,
                            void* out, uint32_t tokens, uint32_t experts, uint32_t top, uint32_t hidden, uint32_t ff, float factor, uint32_t flags,
                            void* workspace, size_t workspace_bytes, void* stream) {
    using namespace moe;
    const char* op = "miori_moe_fp8";
    if (!w_up || !s_up || !w_down || !s_down) return fail(MIORI_E_INVALID, "%s: null weight pointer", op);
    if (const int rc = check_common(op, x, router, out, tokens, experts, top, hidden, ff, 16u, factor, bias, workspace, workspace_bytes)) return rc;
    for (const void* p : {w_up, w_down, static_cast<const void*>(s_up), static_cast<const void*>(s_down)})
        if (!aligned16(p)) return fail(MIORI_E_INVALID, "%s: weights must be 16-byte aligned", op);
    Args a = common_args(x, router, bias, out, tokens, experts, top, hidden, ff, factor, flags, workspace);
    a.up.q = static_cast<const uint8_t*>(w_up), a.up.s = reinterpret_cast<const uint8_t*>(s_up);
    a.down.q = static_cast<const uint8_t*>(w_down), a.down.s = reinterpret_cast<const uint8_t*>(s_down);
    const cudaStream_t s = (cudaStream_t)stream;
    return tokens <= 8 ? launch_moe<E4M3, 1>(op, a, s) : launch_moe<E4M3, 2>(op, a, s);
}
