// What lies between an output's gradient and the products that use it:
//
//   dZ[t][n] = dC[t][n] * act'(Z[t][n])          rounded to the products' 16-bit type
//   dbias_g[n] = sum over the rows t of group g of the unrounded dZ[t][n]
//
// Bound by HBM: dC and Z are read once, dZ is written once, and the column sums ride along in registers. A
// block takes 256 columns (a warp reads 512 consecutive bytes of a row) of one slice of a group's rows; its eight
// warps take every eighth row, eight columns per lane, four rows in flight. The slices' sums are added in order by
// bias_sum_kernel, so the result does not depend on timing.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "activation.cuh"
#include "ptx_sm100.cuh"

namespace b200 {

constexpr int kSlopeThreads = 256;
constexpr uint32_t kSlopeColumns = 256;
constexpr uint32_t kRowsInFlight = 4;

struct SlopeParams {
    const void *dc;
    const void *pre;
    void *dz;              // or null: only the sums are wanted
    float *sums;           // slices x groups x n, the bias gradient itself where slices == 1, or null
    const int32_t *offsets;  // or null: one group of all rows
    uint32_t rows, n, groups, slices;
    uint32_t c_type;       // 0 FP16, 1 BF16, 2 FP32: type of dc and pre
    uint32_t dz_bf16;
    uint32_t accumulate;   // slices == 1: add to what `sums` holds
};

// Eight consecutive values of a row.
__device__ __forceinline__ void load8(const void *base, size_t at, uint32_t type, float (&v)[8]) {
    if (type == 2u) {
        const float4 *src = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
        const float4 a = src[0], b = src[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        return;
    }
    const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const __half *>(base) + at);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 f;
        if (type == 1u) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&words[i]));
        else f = __half22float2(*reinterpret_cast<const __half2 *>(&words[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

template <uint32_t KIND>
__global__ void __launch_bounds__(kSlopeThreads) slope_kernel(const SlopeParams p) {
    __shared__ float block_sums[kSlopeThreads / 32][kSlopeColumns];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t col = blockIdx.x * kSlopeColumns + lane * 8u;
    const uint32_t slice = blockIdx.y, g = blockIdx.z;
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    uint32_t start = 0, end = p.rows;
    if (p.offsets) {
        const int32_t a = __ldg(p.offsets + g), b = __ldg(p.offsets + g + 1);
        start = a < 0 ? 0u : min(static_cast<uint32_t>(a), p.rows);
        end = max(b < 0 ? 0u : min(static_cast<uint32_t>(b), p.rows), start);
    }
    const uint64_t r = end - start;
    const uint32_t lo = start + static_cast<uint32_t>(r * slice / p.slices);
    const uint32_t hi = start + static_cast<uint32_t>(r * (slice + 1u) / p.slices);
    const bool live = col < p.n;  // n is a multiple of 8
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
        constexpr uint32_t kWarps = kSlopeThreads / 32;
        for (uint32_t t0 = lo + warp; t0 < hi; t0 += kRowsInFlight * kWarps) {
            // all loads before the first store: dz may be dc, so the compiler could not move them there itself
            float d[kRowsInFlight][8], z[kRowsInFlight][8];
#pragma unroll
            for (uint32_t u = 0; u < kRowsInFlight; ++u) {
                const uint32_t t = t0 + u * kWarps;
                if (t < hi) {
                    const size_t at = static_cast<size_t>(t) * p.n + col;
                    load8(p.dc, at, p.c_type, d[u]);
                    if (KIND != kActNone) load8(p.pre, at, p.c_type, z[u]);
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < kRowsInFlight; ++u) {
                const uint32_t t = t0 + u * kWarps;
                if (t >= hi) break;
                if (KIND != kActNone) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[u][i] *= act_slope<KIND>(z[u][i]);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += d[u][i];
                if (p.dz) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (p.dz_bf16) {
                            __nv_bfloat162 b = __floats2bfloat162_rn(d[u][2 * i], d[u][2 * i + 1]);
                            w[i] = *reinterpret_cast<uint32_t *>(&b);
                        } else {
                            __half2 h = __floats2half2_rn(d[u][2 * i], d[u][2 * i + 1]);
                            w[i] = *reinterpret_cast<uint32_t *>(&h);
                        }
                    }
                    *reinterpret_cast<uint4 *>(static_cast<__half *>(p.dz) + static_cast<size_t>(t) * p.n + col) =
                        make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    }
    if (!p.sums) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) block_sums[warp][lane * 8 + i] = sum[i];
    __syncthreads();
    const uint32_t c = blockIdx.x * kSlopeColumns + threadIdx.x;
    if (c < p.n) {
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < kSlopeThreads / 32; ++w) total += block_sums[w][threadIdx.x];
        float *dst = p.sums + (static_cast<size_t>(slice) * p.groups + g) * p.n + c;
        *dst = p.accumulate ? *dst + total : total;
    }
}

// dbias[i] = sum of the slices' sums, in order (added to what is there with `accumulate`).
__global__ void __launch_bounds__(256) bias_sum_kernel(const float *sums, float *dbias, size_t count, uint32_t slices, uint32_t accumulate) {
    pdl_launch_dependents();
    pdl_wait_prior_grids();
    const size_t i = static_cast<size_t>(blockIdx.x) * 256u + threadIdx.x;
    if (i >= count) return;
    float total = accumulate ? dbias[i] : 0.f;
#pragma unroll 8
    for (uint32_t s = 0; s < slices; ++s) total += sums[static_cast<size_t>(s) * count + i];
    dbias[i] = total;
}

}  // namespace b200
