// What lies between an output's gradient and the products that use it:
//
//   dZ[t][n] = dC[t][n] * act'(Z[t][n])          rounded to the products' 16-bit type
//   dbias_g[n] = sum over the rows t of group g of the unrounded dZ[t][n]
//
// The rounding is what the tensor cores ask for: their operands are 16-bit. It is the only one between dC and the products'
// FP32 sums; each term of dA's and dB's sums is off by half a step of the inputs' type at most, so an FP32 dB behind an activation
// (or of an FP32 dC) is as good as 16-bit terms make it, however it is accumulated. Terms of twice the width, as two 16-bit numbers each,
// would double the time of both products.
//
// Bound by HBM: dC and Z are read once, dZ is written once, and the column sums ride along in registers. A
// block takes 256 columns (a warp reads 512 consecutive bytes of a row) of one slice of a group's rows; its eight
// warps take every eighth row, eight columns per lane, four rows in flight, which leaves registers for four blocks
// on an SM. What is in flight is kept as it lies in memory: with the values already converted the same kernel
// reached 2.3 TB/s. 8192 x 14336 in BF16: 142 us with gelu_tanh (705 MB, 4.9 TB/s), 119 with silu, 208 with gelu; eight rows
// in flight 173 us, slices of 32 rows 173, of 512 rows 212. The slices' sums are added in order by bias_sum_kernel,
// so the result does not depend on timing.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "activation.cuh"
#include "ptx_sm100.cuh"

namespace b200 {

constexpr int kSlopeThreads = 256;
constexpr uint32_t kSlopeColumns = 256;
constexpr uint32_t kRowsInFlight = 4;  // 16-bit rows a warp has asked for before it uses the first (half as many of FP32)

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

// Eight consecutive values of a row as they lie in memory (16 bytes, or 32 of FP32), and as FP32.
template <bool F32>
struct Eight {
    uint4 w[F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void *base, size_t at) {
        const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(base) + at * (F32 ? 4u : 2u));
        w[0] = __ldcs(src);
        if (F32) w[F32 ? 1 : 0] = __ldcs(src + 1);
    }
    __device__ __forceinline__ float2 pair(int i, uint32_t bf16) const {  // values 2i and 2i + 1
        const uint4 &v = w[F32 ? i / 2 : 0];
        if (F32) return i & 1 ? make_float2(__uint_as_float(v.z), __uint_as_float(v.w)) : make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        const uint32_t word = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
        if (bf16) return make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
        return __half22float2(*reinterpret_cast<const __half2 *>(&word));
    }
};

template <uint32_t KIND, bool F32>
__global__ void __launch_bounds__(kSlopeThreads, 4) slope_kernel(const SlopeParams p) {
    __shared__ float block_sums[kSlopeThreads / 32][kSlopeColumns];
    constexpr uint32_t kRows = F32 ? kRowsInFlight / 2 : kRowsInFlight;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t col = blockIdx.x * kSlopeColumns + lane * 8u;
    const uint32_t slice = blockIdx.y, g = blockIdx.z;
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
    const uint32_t c_bf16 = p.c_type == 1u;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
        constexpr uint32_t kWarps = kSlopeThreads / 32;
        for (uint32_t t0 = lo + warp; t0 < hi; t0 += kRows * kWarps) {
            // all loads before the first store: dz may be dc, so the compiler could not move them there itself
            Eight<F32> d[kRows], z[kRows];
#pragma unroll
            for (uint32_t u = 0; u < kRows; ++u) {
                const uint32_t t = t0 + u * kWarps;
                if (t < hi) {
                    const size_t at = static_cast<size_t>(t) * p.n + col;
                    d[u].load(p.dc, at);
                    if (KIND != kActNone) z[u].load(p.pre, at);
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < kRows; ++u) {
                const uint32_t t = t0 + u * kWarps;
                if (t >= hi) break;
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float2 v = d[u].pair(i, c_bf16);
                    if (KIND != kActNone) {
                        const float2 x = z[u].pair(i, c_bf16);
                        v.x *= act_slope<KIND>(x.x);
                        v.y *= act_slope<KIND>(x.y);
                    }
                    sum[2 * i] += v.x;
                    sum[2 * i + 1] += v.y;
                    if (p.dz_bf16) {
                        __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
                        w[i] = *reinterpret_cast<uint32_t *>(&b);
                    } else {
                        __half2 h = __floats2half2_rn(v.x, v.y);
                        w[i] = *reinterpret_cast<uint32_t *>(&h);
                    }
                }
                if (p.dz) {
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
    const size_t i = static_cast<size_t>(blockIdx.x) * 256u + threadIdx.x;
    if (i >= count) return;
    float total = accumulate ? dbias[i] : 0.f;
#pragma unroll 8
    for (uint32_t s = 0; s < slices; ++s) total += sums[static_cast<size_t>(s) * count + i];
    dbias[i] = total;
}

// out[i] = sum of the slices' FP32 results, in order, rounded to out's type (0 FP16, 1 BF16, 2 FP32; added to what is
// there with `accumulate`, FP32 only). Four values per thread; count is a multiple of 4.
__global__ void __launch_bounds__(256) slice_sum_kernel(const float4 *slices, void *out, size_t count4, uint32_t n, uint32_t type,
                                                        uint32_t accumulate) {
    const size_t i = static_cast<size_t>(blockIdx.x) * 256u + threadIdx.x;
    if (i >= count4) return;
    float4 total = accumulate ? static_cast<const float4 *>(out)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (uint32_t s = 0; s < n; ++s) {
        const float4 v = slices[static_cast<size_t>(s) * count4 + i];
        total.x += v.x;
        total.y += v.y;
        total.z += v.z;
        total.w += v.w;
    }
    if (type == 2u) {
        static_cast<float4 *>(out)[i] = total;
    } else if (type == 1u) {
        __nv_bfloat162 a = __floats2bfloat162_rn(total.x, total.y), b = __floats2bfloat162_rn(total.z, total.w);
        static_cast<uint2 *>(out)[i] = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
    } else {
        __half2 a = __floats2half2_rn(total.x, total.y), b = __floats2half2_rn(total.z, total.w);
        static_cast<uint2 *>(out)[i] = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
    }
}

}  // namespace b200
