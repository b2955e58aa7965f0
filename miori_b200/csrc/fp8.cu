// Entries of the operators in 8-bit floating point: argument checks and which kernel takes a call.  (The reference has no such
// format; they stand where miori_rmsnorm + miori_gemm_bf16_cache do.)
#include "gemm_fp8.cuh"
#include "quant_fp8.cuh"

namespace miori_b200 {
namespace fp8 {

// rows `pitch` elements apart that a kernel steps through: positive, and far from the end of 64 bits
static bool fine_pitch(int64_t pitch) { return pitch > 0 && pitch < (1ll << 40); }
static bool fine_stride(int64_t stride) { return stride > -(1ll << 40) && stride < (1ll << 40); }

}  // namespace fp8
}  // namespace miori_b200

using namespace miori_b200;

MIORI_API int miori_quant_fp8(const void* x, int64_t x_row, void* q, int64_t q_row, float* scales, int64_t scale_row, int64_t scale_col,
                              uint32_t rows, uint32_t K, uint32_t tile, uint32_t flags, void* stream) {
    using namespace fp8;
    const char* op = "miori_quant_fp8";
    if (!x || !q || !scales) return fail(MIORI_E_INVALID, "%s: null pointer", op);
    if (rows == 0 || K == 0) return fail(MIORI_E_INVALID, "%s: empty shape rows=%u K=%u", op, rows, K);
    if (rows > 0x7FFFFF00u || K > 0x7FFFFF00u) return fail(MIORI_E_INVALID, "%s: rows and K are below 2^31 - 256", op);
    if (tile != 1 && tile != BLOCK) return fail(MIORI_E_INVALID, "%s: blocks of 1 or 128 rows, got %u", op, tile);
    const bool f32 = (flags & MIORI_QUANT_F32) != 0;
    if (!fine_pitch(x_row) || x_row < (int64_t)K || !fine_pitch(q_row) || q_row < (int64_t)K)
        return fail(MIORI_E_INVALID, "%s: a row pitch is shorter than its row, or too long (x_row=%lld q_row=%lld K=%u)", op, (long long)x_row, (long long)q_row, K);
    if (!fine_stride(scale_row) || !fine_stride(scale_col)) return fail(MIORI_E_INVALID, "%s: strides of the scales must be below 2^40", op);
    if ((scale_row == 0 && (rows + tile - 1) / tile > 1) || (scale_col == 0 && K > BLOCK)) return fail(MIORI_E_INVALID, "%s: scales of several blocks would lie on one another", op);
    if (!aligned16(q) || q_row % 16) return fail(MIORI_E_INVALID, "%s: rows of q must begin on 16-byte boundaries", op);
    if ((reinterpret_cast<uintptr_t>(x) & (f32 ? 3u : 1u)) || (reinterpret_cast<uintptr_t>(scales) & 3u))
        return fail(MIORI_E_INVALID, "%s: x or scales is not aligned to its elements", op);
    QuantArgs a;
    a.x = x, a.q = static_cast<uint8_t*>(q), a.scales = scales;
    a.x_row = x_row, a.q_row = q_row, a.s_row = scale_row, a.s_col = scale_col;
    a.rows = rows, a.K = K, a.k_blocks = (K + BLOCK - 1u) / BLOCK;
    a.by_blocks = Div::by(a.k_blocks);
    if ((uint64_t)(tile == 1 ? rows : (rows + BLOCK - 1u) / BLOCK) * a.k_blocks > 0x7FFFFF00ull) return fail(MIORI_E_INVALID, "%s: too many blocks (rows=%u K=%u)", op, rows, K);
    const bool vec = aligned16(x) && x_row % (f32 ? 4 : 8) == 0;
    const cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = f32 ? (vec ? launch_quant<true, true>(a, tile != 1, s) : launch_quant<true, false>(a, tile != 1, s))
                              : (vec ? launch_quant<false, true>(a, tile != 1, s) : launch_quant<false, false>(a, tile != 1, s));
    return e == cudaSuccess ? MIORI_OK : cuda_fail(e, "quant_fp8 launch");
}

MIORI_API int miori_gemm_fp8(const void* a, int64_t lda, const float* sa, int64_t sa_row, int64_t sa_col, const void* w, int64_t ldw, const float* sw,
                             int64_t sw_row, int64_t sw_col, void* C, int64_t ldc, uint32_t M, uint32_t N, uint32_t K, uint32_t flags, void* stream) {
    using namespace fp8;
    const char* op = "miori_gemm_fp8";
    if (!a || !sa || !w || !sw || !C) return fail(MIORI_E_INVALID, "%s: null pointer", op);
    if (M == 0 || N == 0 || K == 0) return fail(MIORI_E_INVALID, "%s: empty shape M=%u N=%u K=%u", op, M, N, K);
    if (M > 0x7FFFFF00u || N > 0x7FFFFF00u || K > 0x7FFFFF00u) return fail(MIORI_E_INVALID, "%s: M, N and K are below 2^31 - 256", op);
    if (!aligned16(a) || !aligned16(w) || lda % 16 || ldw % 16) return fail(MIORI_E_INVALID, "%s: rows of a and w must begin on 16-byte boundaries", op);
    if (!fine_pitch(lda) || lda < (int64_t)K || !fine_pitch(ldw) || ldw < (int64_t)K || !fine_pitch(ldc) || ldc < (int64_t)N)
        return fail(MIORI_E_INVALID, "%s: a row pitch is shorter than its row, or too long (lda=%lld ldw=%lld K=%u ldc=%lld N=%u)", op, (long long)lda, (long long)ldw, K,
                    (long long)ldc, N);
    if (!fine_stride(sa_row) || !fine_stride(sa_col) || !fine_stride(sw_row) || !fine_stride(sw_col))
        return fail(MIORI_E_INVALID, "%s: strides of the scales must be below 2^40", op);
    GemmArgs g;
    g.c = C, g.sa = sa, g.sw = sw;
    g.ldc = ldc, g.sa_row = sa_row, g.sa_col = sa_col, g.sw_row = sw_row, g.sw_col = sw_col;
    g.M = M, g.N = N, g.K = K;
    g.bf16 = flags & MIORI_OUT_BF16 ? 1u : 0u;
    const uint32_t size = g.bf16 ? 2 : 4;
    if ((reinterpret_cast<uintptr_t>(C) & (size - 1u)) || (reinterpret_cast<uintptr_t>(sa) & 3u) || (reinterpret_cast<uintptr_t>(sw) & 3u))
        return fail(MIORI_E_INVALID, "%s: C or a scale is not aligned to its elements", op);
    // what a TMA store can describe: rows that begin, and end, on 16-byte boundaries
    g.by_tma = aligned16(C) && ldc * size % 16 == 0 && (uint64_t)N * size % 16 == 0 ? 1u : 0u;
    const GemmOperands o = {a, w, lda, ldw};
    const GemmPlan p = plan_gemm_fp8(M, N, K, flags);
    if (!p.pair_n && K > 128u * KB_BYTES) return fail(MIORI_E_INVALID, "%s: the kernel of few rows takes K up to 16384, got %u", op, K);  // by a tuning flag
    const cudaStream_t s = (cudaStream_t)stream;
    if (p.pair_n) return p.pair_n == 256u ? launch_pair<256>(o, g, s) : launch_pair<128>(o, g, s);
    switch (p.mp) {
        case 16: return launch_swap<16>(o, g, p.cs, s);
        case 32: return launch_swap<32>(o, g, p.cs, s);
        case 64: return launch_swap<64>(o, g, p.cs, s);
        default: return launch_swap<128>(o, g, p.cs, s);
    }
}
