// Rows, or tiles of 128 rows, as 8-bit floating point (e4m3) with a scale for each block of TILE x 128 elements:
//   a = max(max |x|, 2^-100);  scale = a / 448;  q = e4m3(x * (448 / a)),
// every operation in fp32 and rounded once, so that the result is the same whoever computes it.  (Floored, because 448 / a
// would overflow below 2^-120; a block of zeros comes out as zeros.)  448 is the type's largest value; nothing is cut off but by
// half a unit of fp32.  A NaN stays one where it is and is not looked at by the maximum; a block with an infinity comes
// out as NaNs once it is multiplied out, zeros by an infinite scale.
#pragma once
#include "common.cuh"

#include <cuda_fp8.h>

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

// Eight neighbouring elements from column k on; those behind K are zeros.  VEC: rows begin on 16-byte boundaries.
template <bool F32, bool VEC>
__device__ __forceinline__ void load8(const void* x, size_t row_at, uint32_t k, uint32_t K, float (&v)[8]) {
    if (VEC && k + 8u <= K) {
        if constexpr (F32) {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + row_at + k);
            const float4 a = ld_fresh<float4, true>(p), b = ld_fresh<float4, true>(p + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 a = ld_fresh<uint4, true>(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + row_at + k));
            v[0] = bf16lo(a.x), v[1] = bf16hi(a.x), v[2] = bf16lo(a.y), v[3] = bf16hi(a.y);
            v[4] = bf16lo(a.z), v[5] = bf16hi(a.z), v[6] = bf16lo(a.w), v[7] = bf16hi(a.w);
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        v[i] = 0.0f;
        if (k + i < K)
            v[i] = F32 ? ld_fresh(static_cast<const float*>(x) + row_at + k + i)
                       : bf16_bits_to_float(ld_fresh(static_cast<const uint16_t*>(x) + row_at + k + i));
    }
}
__device__ __forceinline__ float max8(const float (&v)[8]) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
    return m;
}
// Rows of q begin on 16-byte boundaries and k is a multiple of eight; what lies behind K is left as it was.
__device__ __forceinline__ void store8(uint8_t* q, size_t row_at, uint32_t k, uint32_t K, const float (&v)[8], float inv) {
    if (k >= K) return;
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
};

// A block of 1 x 128: 16 lanes, eight elements each.  UNITS blocks a lane group, their loads all under way before the first
// maximum.
constexpr uint32_t ROW_THREADS = 256, ROW_GROUPS = ROW_THREADS / 16;
template <bool F32, bool VEC, int UNITS>
__global__ void __launch_bounds__(ROW_THREADS)
quant_rows_kernel(const QuantArgs a) {
    pdl_launch_dependents();
    pdl_wait_prior();
    const uint32_t group = threadIdx.x >> 4, lane = threadIdx.x & 15u;
    const uint64_t total = (uint64_t)a.rows * a.k_blocks, first = (uint64_t)blockIdx.x * (ROW_GROUPS * UNITS) + group;
    float v[UNITS][8];
    uint32_t row[UNITS], block[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const uint64_t i = first + (uint64_t)u * ROW_GROUPS;
        // 64-bit division only where 32 do not do
        row[u] = total <= 0xFFFFFFFFull ? (uint32_t)i / a.k_blocks : (uint32_t)(i / a.k_blocks);
        block[u] = (uint32_t)(i - (uint64_t)row[u] * a.k_blocks);
        if (i < total) {
            load8<F32, VEC>(a.x, (size_t)row[u] * (size_t)a.x_row, block[u] * BLOCK + lane * 8u, a.K, v[u]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[u][e] = 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        float m = max8(v[u]);
#pragma unroll
        for (int d = 8; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
        m = fmaxf(m, LEAST);
        if (first + (uint64_t)u * ROW_GROUPS >= total) continue;
        store8(a.q, (size_t)row[u] * (size_t)a.q_row, block[u] * BLOCK + lane * 8u, a.K, v[u], __fdiv_rn(TOP, m));
        if (lane == 0) a.scales[(int64_t)row[u] * a.s_row + (int64_t)block[u] * a.s_col] = __fdiv_rn(m, TOP);
    }
}

// A block of 128 x 128: one CTA, everything in registers between the maximum and the store.
constexpr uint32_t TILE_THREADS = 256;
template <bool F32, bool VEC>
__global__ void __launch_bounds__(TILE_THREADS)
quant_tiles_kernel(const QuantArgs a) {
    __shared__ float part[TILE_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait_prior();
    constexpr uint32_t STEPS = BLOCK * BLOCK / 8 / TILE_THREADS, STEP_ROWS = TILE_THREADS / 16;
    const uint32_t tile_row = blockIdx.x / a.k_blocks, block = blockIdx.x - tile_row * a.k_blocks;
    const uint32_t k = block * BLOCK + (threadIdx.x & 15u) * 8u, row0 = tile_row * BLOCK + (threadIdx.x >> 4);
    float v[STEPS][8], m = LEAST;
#pragma unroll
    for (uint32_t s = 0; s < STEPS; ++s) {
        const uint32_t row = row0 + s * STEP_ROWS;
        if (row < a.rows) {
            load8<F32, VEC>(a.x, (size_t)row * (size_t)a.x_row, k, a.K, v[s]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[s][e] = 0.0f;
        }
    }
#pragma unroll
    for (uint32_t s = 0; s < STEPS; ++s) m = fmaxf(m, max8(v[s]));
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
        if (row < a.rows) store8(a.q, (size_t)row * (size_t)a.q_row, k, a.K, v[s], inv);
    }
    if (threadIdx.x == 0) a.scales[(int64_t)tile_row * a.s_row + (int64_t)block * a.s_col] = __fdiv_rn(m, TOP);
}

template <bool F32, bool VEC>
inline cudaError_t launch_quant(const QuantArgs& a, bool tiles, cudaStream_t stream) {
    if (tiles) return launch(quant_tiles_kernel<F32, VEC>, dim3((a.rows + BLOCK - 1) / BLOCK * a.k_blocks), dim3(TILE_THREADS), 0, stream, true, a);
    const uint64_t total = (uint64_t)a.rows * a.k_blocks;
    // four blocks a lane group once the SMs have enough groups with that
    if (total >= (uint64_t)sm_count() * ROW_GROUPS * 16u)
        return launch(quant_rows_kernel<F32, VEC, 4>, dim3((unsigned)((total + ROW_GROUPS * 4 - 1) / (ROW_GROUPS * 4))), dim3(ROW_THREADS), 0, stream, true, a);
    return launch(quant_rows_kernel<F32, VEC, 1>, dim3((unsigned)((total + ROW_GROUPS - 1) / ROW_GROUPS)), dim3(ROW_THREADS), 0, stream, true, a);
}

}  // namespace fp8
}  // namespace miori_b200
