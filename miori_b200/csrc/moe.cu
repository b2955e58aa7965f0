// Entries of the layers of experts: argument checks, the kernel's shape, the launch.  (The reference's models have dense feed-forwards:
// gate + up, silu_mul and down as separate dispatches, src/engine.cpp:484-502.)
#include "moe.cuh"

#include <cmath>

namespace miori_b200 {
namespace moe {

constexpr size_t TOPS_BYTES = MAX_ROWS * sizeof(uint32_t), HEAD_BYTES = (sizeof(Tables) + TOPS_BYTES + 255) / 256 * 256;

// Dynamic shared memory of both products: all of an SM's that the tables leave, a ring and B fragments or partial sums in the rest.
static_assert(sizeof(UpTables) <= sizeof(DownTables), "");
constexpr size_t SMEM = 227 * 1024 - (sizeof(DownTables) + 32 + 127) / 128 * 128;
template <Format FMT>
constexpr size_t frag_room(int depth) { return SMEM - Stage<FMT>::ring(depth) - 2 * WARPS * 512; }

// Of moe_down, were there as many entries as there can be: cells of one row tile for every warp, and the cluster's sums of one.
constexpr uint32_t most_segments(uint32_t most_units) {
    uint32_t most = 0;
    for (uint32_t units = 1; units <= most_units; ++units)
        if (segments_of(MAX_DOWN_ENTRIES * units, units) > most) most = segments_of(MAX_DOWN_ENTRIES * units, units);
    return most;
}
template <Format FMT>
constexpr uint32_t ONE_TILE = WARPS * 512u * most_segments(MAX_FF / Stage<FMT>::UNIT) + CLUSTER * MAX_TOKENS * 64u;

template <Format FMT, int DEPTH>
static int launch_moe(const char* op, Args a, cudaStream_t stream) {
    a.slots = (uint32_t)(frag_room<FMT>(DEPTH) / ((size_t)a.up.units * Stage<FMT>::FRAG));
    a.area = (uint32_t)(SMEM - Stage<FMT>::ring(Stage<FMT>::DOWN));
    static_assert(SMEM - Stage<FMT>::ring(Stage<FMT>::DOWN) >= ONE_TILE<FMT>, "moe_down works on one row tile at a time at least");
    const uint32_t sms = (uint32_t)sm_count(), row_tiles = a.H / 16u;
    // clusters of four whole SMs: an SM in nine has no place in one
    const uint32_t most = sms * 8u / 9u / CLUSTER;
    a.per = (row_tiles + most - 1u) / most;
    a.by_tokens = Div::by(a.tokens), a.by_tiles = Div::by(a.F / 8u), a.by_ctas = Div::by(sms);
    auto router = a.experts <= 32u ? moe_router_kernel<1> : a.experts <= 128u ? moe_router_kernel<4> : moe_router_kernel<8>;
    cudaError_t e = launch_cluster(router, ROUTER_CLUSTER, THREADS, (size_t)a.tokens * 1024u, ROUTER_CLUSTER, stream, a);
    if (e == cudaSuccess) e = launch(moe_up_kernel<FMT, DEPTH>, dim3(sms), dim3(THREADS), SMEM, stream, true, a);
    if (e == cudaSuccess) e = launch_cluster(moe_down_kernel<FMT>, (row_tiles + a.per - 1u) / a.per * CLUSTER, THREADS, SMEM, CLUSTER, stream, a);
    return e == cudaSuccess ? MIORI_OK : cuda_fail(e, op);
}
// Rows whose B fragments do not fit beside it take a ring of two stages.
template <Format FMT>
static int launch_moe(const char* op, Args a, cudaStream_t stream) {
    constexpr int DEPTH = Stage<FMT>::UP;
    constexpr uint32_t UNIT = Stage<FMT>::UNIT;
    auto matrix = [](Matrix& m, uint32_t rows, uint32_t K) {
        m.rows = rows, m.K = K, m.units = (K + UNIT - 1u) / UNIT, m.by_units = Div::by(m.units), m.whole = K % UNIT == 0u;
        m.pitch = FMT == E4M3 ? K : K / 2u, m.scale_pitch = FMT == E4M3 ? 0u : K / (FMT == GROUP64 ? 64u : 32u) * 2u;
    };
    matrix(a.up, 2u * a.F, a.H);
    matrix(a.down, a.H, a.F);
    static_assert((MAX_HIDDEN + UNIT - 1) / UNIT * Stage<FMT>::FRAG <= frag_room<FMT>(2), "the longest rows fit");
    if ((size_t)a.up.units * Stage<FMT>::FRAG > frag_room<FMT>(DEPTH)) return launch_moe<FMT, 2>(op, a, stream);
    return launch_moe<FMT, DEPTH>(op, a, stream);
}

static int check_common(const char* op, const void* x, const void* router, const void* out, uint32_t tokens, uint32_t experts, uint32_t top, uint32_t hidden, uint32_t ff,
                        uint32_t step, float factor, const float* bias, const void* workspace, size_t workspace_bytes) {
    if (!x || !router || !out || !workspace) return fail(MIORI_E_INVALID, "%s: null pointer", op);
    if (tokens == 0 || tokens > MAX_TOKENS) return fail(MIORI_E_INVALID, "%s: 1..%u tokens, got %u", op, MAX_TOKENS, tokens);
    if (experts == 0 || experts > MAX_EXPERTS) return fail(MIORI_E_INVALID, "%s: 1..%u experts, got %u", op, MAX_EXPERTS, experts);
    if (top == 0 || top > MAX_TOP || top > experts) return fail(MIORI_E_INVALID, "%s: 1..%u of %u experts for a token, got %u", op, MAX_TOP, experts, top);
    if (hidden == 0 || ff == 0 || hidden % step || ff % step)
        return fail(MIORI_E_INVALID, "%s: hidden and ff are multiples of %u, got %u and %u", op, step, hidden, ff);
    if (hidden > MAX_HIDDEN || ff > MAX_FF) return fail(MIORI_E_INVALID, "%s: hidden is at most %u and ff %u, got %u and %u", op, MAX_HIDDEN, MAX_FF, hidden, ff);
    if (!std::isfinite(factor)) return fail(MIORI_E_INVALID, "%s: the factor must be finite", op);
    if (!aligned16(x) || !aligned16(router) || !aligned16(out) || !aligned16(workspace) || (reinterpret_cast<uintptr_t>(bias) & 3u))
        return fail(MIORI_E_INVALID, "%s: x, router, out and workspace must be 16-byte aligned, bias by its elements", op);
    if (workspace_bytes < miori_moe_workspace_bytes(tokens, top, ff))
        return fail(MIORI_E_INVALID, "%s: a workspace of %zu bytes is needed, got %zu", op, miori_moe_workspace_bytes(tokens, top, ff), workspace_bytes);
    return MIORI_OK;
}

static Args common_args(const void* x, const void* router, const float* bias, void* out, uint32_t tokens, uint32_t experts, uint32_t top, uint32_t hidden, uint32_t ff,
                        float factor, uint32_t flags, void* workspace) {
    Args a = {};
    a.x = static_cast<const uint16_t*>(x), a.router = static_cast<const uint16_t*>(router), a.bias = bias, a.out = out;
    char* w = static_cast<char*>(workspace);
    a.tables = reinterpret_cast<Tables*>(w), a.h_top = reinterpret_cast<uint32_t*>(w + sizeof(Tables)), a.h = reinterpret_cast<float*>(w + HEAD_BYTES);
    a.ahead = flags & MIORI_LAUNCH_PDL ? 1u : 0u;
    a.factor = factor, a.tokens = tokens, a.experts = experts, a.top = top, a.H = hidden, a.F = ff;
    a.sigmoid = flags & MIORI_MOE_SIGMOID ? 1u : 0u, a.norm = flags & MIORI_MOE_NORM ? 1u : 0u, a.bf16 = flags & MIORI_OUT_BF16 ? 1u : 0u;
    return a;
}

}  // namespace moe
}  // namespace miori_b200

using namespace miori_b200;

MIORI_API size_t miori_moe_workspace_bytes(uint32_t tokens, uint32_t top, uint32_t ff) { return moe::HEAD_BYTES + (size_t)tokens * top * ff * sizeof(float); }

MIORI_API int miori_moe4(const void* x, const void* router, const float* bias, const void* q_up, const void* s_up, const void* b_up, const void* q_down,
                         const void* s_down, const void* b_down, void* out, uint32_t tokens, uint32_t experts, uint32_t top, uint32_t hidden, uint32_t ff,
                         uint32_t group, float factor, uint32_t flags, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace moe;
    const char* op = "miori_moe4";
    if (!q_up || !s_up || !b_up || !q_down || !s_down || !b_down) return fail(MIORI_E_INVALID, "%s: null weight pointer", op);
    if (group != 32 && group != 64) return fail(MIORI_E_INVALID, "%s: group must be 32 or 64 (got %u)", op, group);
    if (const int rc = check_common(op, x, router, out, tokens, experts, top, hidden, ff, 128u, factor, bias, workspace, workspace_bytes)) return rc;
    for (const void* p : {q_up, s_up, b_up, q_down, s_down, b_down})
        if (!aligned16(p)) return fail(MIORI_E_INVALID, "%s: weights must be 16-byte aligned", op);
    Args a = common_args(x, router, bias, out, tokens, experts, top, hidden, ff, factor, flags, workspace);
    auto u8 = [](const void* p) { return static_cast<const uint8_t*>(p); };
    a.up.q = u8(q_up), a.up.s = u8(s_up), a.up.b = u8(b_up), a.down.q = u8(q_down), a.down.s = u8(s_down), a.down.b = u8(b_down);
    const cudaStream_t s = (cudaStream_t)stream;
    return group == 64 ? launch_moe<GROUP64>(op, a, s) : launch_moe<GROUP32>(op, a, s);
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
    return launch_moe<E4M3>(op, a, s);
}
