// Rows, or tiles of 128 rows, as 8-bit floating point (e4m3) with a scale for each block of TILE x 128 elements:
//   a = max(max |x|, 2^-100);  scale = a / 448;  q = e4m3(x * (448 / a)),
// every operation in fp32 and rounded once, so that the result is the same whoever computes it.  (Floored, because 448 / a
// would overflow below 2^-120; a block of zeros comes out as zeros.)  448 is the type's largest value; nothing is cut off but by
// half a unit of fp32.  A NaN stays one where it is and is not looked at by the maximum; a block with an infinity comes
// out as NaNs once it is multiplied out, zeros by an infinite scale.
#pragma once
#include "common.cuh"

namespace miori_b200 {
namespace fp8 {

constexpr uint32_t BLOCK = 128;  // elements of a block along K
constexpr float TOP = 448.0f;
constexpr float LEAST = 7.888609052210118e-31f;  // 2^-100

// Two fp32 as a pair of e4m3, the first in the lower byte; rounded to nearest even, beyond 448 cut off, NaN kept.
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Eight neighbouring elements of a row, as they lie in memory.
template <bool F32>
struct Eight;
template <>
struct Eight<false> {
    uint4 w;
    __device__ __forceinline__ void value(float (&v)[8]) const {
        v[0] = bf16lo(w.x), v[1] = bf16hi(w.x), v[2] = bf16lo(w.y), v[3] = bf16hi(w.y), v[4] = bf16lo(w.z), v[5] = bf16hi(w.z), v[6] = bf16lo(w.w), v[7] = bf16hi(w.w);
    }
};
template <>
struct Eight<true> {
    float4 a, b;
    __device__ __forceinline__ void value(float (&v)[8]) const { v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w; }
};
// From column k on; those behind K are zeros.  VEC: rows begin on 16-byte boundaries.
template <bool F32, bool VEC>
__device__ __forceinline__ Eight<F32> load8(const void* x, size_t row_at, uint32_t k, uint32_t K) {
    Eight<F32> e;
    if (VEC && k + 8u <= K) {
        if constexpr (F32) {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + row_at + k);
            e.a = ld_fresh<float4, true>(p), e.b = ld_fresh<float4, true>(p + 1);
        } else {
            e.w = ld_fresh<uint4, true>(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + row_at + k));
        }
        return e;
    }
    uint32_t v[8];
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        v[i] = 0u;
        if (k + i < K) {
            if constexpr (F32) v[i] = ld_fresh(static_cast<const uint32_t*>(x) + row_at + k + i);
            else v[i] = ld_fresh(static_cast<const uint16_t*>(x) + row_at + k + i);
        }
    }
    if constexpr (F32) {
        e.a = make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
        e.b = make_float4(__uint_as_float(v[4]), __uint_as_float(v[5]), __uint_as_float(v[6]), __uint_as_float(v[7]));
    } else {
        e.w = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    }
    return e;
}
// The largest magnitude of N such pieces, NaN left out.  Magnitudes of bf16 are ordered as their bits are, two at a time; a NaN's lie above all
// others', and where there is one they are looked at one by one.
template <bool F32, int N>
__device__ __forceinline__ float largest(const Eight<F32> (&e)[N]) {
    if constexpr (!F32) {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < N; ++i)
            m = __vmaxu2(__vmaxu2(m, __vmaxu2(e[i].w.x & 0x7FFF7FFFu, e[i].w.y & 0x7FFF7FFFu)), __vmaxu2(e[i].w.z & 0x7FFF7FFFu, e[i].w.w & 0x7FFF7FFFu));
        m = max(m & 0xFFFFu, m >> 16);
        if (m <= 0x7F80u) return bf16_bits_to_float(m);
    }
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float v[8];
        e[i].value(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
    }
    return m;
}
// Rows of q begin on 16-byte boundaries and k is a multiple of eight; what lies behind K is left as it was.
template <bool F32>
__device__ __forceinline__ void store8(uint8_t* q, size_t row_at, uint32_t k, uint32_t K, const Eight<F32>& e, float inv) {
    if (k >= K) return;
    float v[8];
    e.value(v);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        w[i] = pack_e4m3(__fmul_rn(v[4 * i], inv), __fmul_rn(v[4 * i + 1], inv)) |
               (pack_e4m3(__fmul_rn(v[4 * i + 2], inv), __fmul_rn(v[4 * i + 3], inv)) << 16);
    uint8_t* to = q + row_at + k;
    if (k + 8u <= K) {
        *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    } else {
        for (uint32_t i = 0; i < K - k; ++i) to[i] = (uint8_t)((i < 4u ? w[0] : w[1]) >> (8u * (i & 3u)));
    }
}

struct QuantArgs {
    const void* x;
    uint8_t* q;
    float* scales;
    int64_t x_row, q_row, s_row, s_col;  // elements
    uint32_t rows, K, k_blocks;
    Div by_blocks;
};

// A block of 1 x 128: LANES lanes, 128 / LANES elements each in pieces of eight, the lanes' pieces side by side.  Four lanes, so that what a block costs (two
// divisions, a maximum's shuffles) is shared by 32 elements a thread; sixteen where that leaves the SMs without a warp.  Bound by HBM: 16384 x 8192 bf16 in 64 us,
// 6.3 TB/s, fp32 in 99.5, 6.8.
constexpr uint32_t ROW_THREADS = 128;
template <bool F32, bool VEC, int LANES>
__global__ void __launch_bounds__(ROW_THREADS)
quant_rows_kernel(const QuantArgs a) {
    constexpr int PIECES = 16 / LANES;
    pdl_launch_dependents();
    pdl_wait_prior();
    const uint32_t lane = threadIdx.x % LANES, i = blockIdx.x * (ROW_THREADS / LANES) + threadIdx.x / LANES;
    const bool there = i < a.rows * a.k_blocks;
    const uint32_t row = there ? a.by_blocks(i) : 0u, block = there ? i - row * a.k_blocks : 0u, k = block * BLOCK + lane * 8u;
    const size_t from = (size_t)row * (size_t)a.x_row, to = (size_t)row * (size_t)a.q_row;
    Eight<F32> e[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) e[p] = load8<F32, VEC>(a.x, from, k + p * (LANES * 8u), there ? a.K : 0u);
    float m = largest<F32, PIECES>(e);
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    m = fmaxf(m, LEAST);
    if (!there) return;
    const float inv = __fdiv_rn(TOP, m);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) store8<F32>(a.q, to, k + p * (LANES * 8u), a.K, e[p], inv);
    if (lane == 0) a.scales[(int64_t)row * a.s_row + (int64_t)block * a.s_col] = __fdiv_rn(m, TOP);
}

// A block of 128 x 128: one CTA, everything in registers between the maximum and the store.  Bound by HBM: 16384 x 2048 bf16 in 19.1 us, 5.3 TB/s, a third of
// it writes (512 threads, whose waves are shorter, 19.4; 1024 24.9); fp32, whose 92 registers leave an SM two CTAs, 33.4, 5.0.
constexpr uint32_t TILE_THREADS = 256;
template <bool F32, bool VEC>
__global__ void __launch_bounds__(TILE_THREADS)
quant_tiles_kernel(const QuantArgs a) {
    __shared__ float part[TILE_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait_prior();
    constexpr uint32_t STEPS = BLOCK * BLOCK / 8 / TILE_THREADS, STEP_ROWS = TILE_THREADS / 16;
    const uint32_t tile_row = a.by_blocks(blockIdx.x), block = blockIdx.x - tile_row * a.k_blocks;
    const uint32_t k = block * BLOCK + (threadIdx.x & 15u) * 8u, row0 = tile_row * BLOCK + (threadIdx.x >> 4);
    Eight<F32> e[STEPS];
#pragma unroll
    for (uint32_t s = 0; s < STEPS; ++s) {
        const uint32_t row = row0 + s * STEP_ROWS;
        e[s] = load8<F32, VEC>(a.x, (size_t)min(row, a.rows - 1u) * (size_t)a.x_row, k, row < a.rows ? a.K : 0u);
    }
    float m = fmaxf(largest<F32, STEPS>(e), LEAST);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    if ((threadIdx.x & 31u) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < TILE_THREADS / 32; ++w) m = fmaxf(m, part[w]);
    const float inv = __fdiv_rn(TOP, m);
#pragma unroll
    for (uint32_t s = 0; s < STEPS; ++s) {
        const uint32_t row = row0 + s * STEP_ROWS;
        if (row < a.rows) store8<F32>(a.q, (size_t)row * (size_t)a.q_row, k, a.K, e[s], inv);
    }
    if (threadIdx.x == 0) a.scales[(int64_t)tile_row * a.s_row + (int64_t)block * a.s_col] = __fdiv_rn(m, TOP);
}

template <bool F32, bool VEC>
inline cudaError_t launch_quant(const QuantArgs& a, bool tiles, cudaStream_t stream) {
    if (tiles) return launch(quant_tiles_kernel<F32, VEC>, dim3((a.rows + BLOCK - 1) / BLOCK * a.k_blocks), dim3(TILE_THREADS), 0, stream, true, a);
    const uint32_t total = a.rows * a.k_blocks;
    // four lanes a block once every SM has 16 warps with that (in a chain, four and sixteen lanes: 32 x 2048 1.5 and 1.2 us, 1024 x 2048 3.1 and 2.9, 1536 x 2048 3.5
    // and 3.8, 4096 x 4096 7.7 and 17.3, 16384 x 8192 60 and 136)
    if (total >= (uint32_t)sm_count() * 128u)
        return launch(quant_rows_kernel<F32, VEC, 4>, dim3((total + ROW_THREADS / 4u - 1u) / (ROW_THREADS / 4u)), dim3(ROW_THREADS), 0, stream, true, a);
    return launch(quant_rows_kernel<F32, VEC, 16>, dim3((total + ROW_THREADS / 16u - 1u) / (ROW_THREADS / 16u)), dim3(ROW_THREADS), 0, stream, true, a);
}

}  // namespace fp8
}  // namespace miori_b200
