// Products over ragged groups of rows: the feed-forward products of a layer whose rows were sorted by expert,
// and, with a single group, those of a dense layer. Three forms of one kernel, with A [T x K], B_g [N x K],
// C [T x N] and the rows [offsets[g], offsets[g+1]) belonging to group g:
//
//   kFormForward  C[t][n]    = act(sum_k A[t][k] B_g[n][k] + bias_g[n])   rows of group g
//   kFormInput    dA[t][k]   = sum_n dC[t][n] B_g[n][k]                   rows of group g
//   kFormWeight   dB_g[n][k] = sum_t dC[t][n] A[t][k]                     t over the rows of group g
//
// The MMA's row operand is called P here and its column operand Q. Forward and input gradient put the weights
// on P (n, or k) and the rows of the group on Q, so the accumulator holds the result transposed: tensor-memory
// lane = output column, tensor-memory column = row of the group. An MMA's column count is chosen at run
// time in steps of 16 (32 for a pair), so a group of 300 rows is two blocks of 160 and 140, where the other
// way round it would be three blocks of 128 (or two of 256 on a pair) filled to 78 (59) percent; a group of three
// rows costs an MMA of 16 columns and stages 16 rows. The rows' operand has a tensor map for every height of a
// block (16 to 128 rows), so that one copy stages it: putting a block together from boxes of 128, 64, 32 and 16
// rows kept the thread that issues the copies busy for longer than the MMAs last (8192 x 8192 x 8192 in one group:
// 904 us against 797). The weight gradient sums over the group's rows: both operands are then row-contiguous in the
// other index and read by the MMA as MN-major; the accumulator is not transposed.
//
// Long sums (LONG): the tensor cores cut off what an accumulator cannot hold instead of rounding it, so that a result
// shrinks with the number of MMAs: by 1.3e-5 of itself per 2048 positive terms, 2e-6 per 2048 of mixed signs (measured from 2048
// to 131072, in proportion to the length). That is 200 and 30 times FP32's own rounding after 2048; an FP16 result's half step, 4.9e-4, is
// reached after 77 000 positive terms, BF16's after 610 000. Sums too long for the result's type (longest_sum in lib_state.h)
// are cut into pieces that alternate between the two accumulators, and the epilogue warps add the pieces in registers, rounding
// to nearest. FP32: pieces of 512, an error of 0.5e-6 for mixed signs whatever the length (of 1024: 0.8 to 1.0e-6). 16-bit
// results: pieces of 4096 and 32768 (512 x 1024 x 32768 in FP16: 94 us in one sum, 96 in such
// pieces, 118 in pieces of 512).
//
// Group sizes are known on the device only (a router wrote them): every CTA reads the offsets, cuts the groups
// into tiles and walks its share of them. Offsets past T are held within [0, T]; where they are out of order, the first two
// forms let a group begin no earlier than the highest offset before it.
//
// A block of rows that reaches past its group's end reads rows of the next group. For P and Q of the first two
// forms this only adds accumulator columns that are never stored. In the weight gradient those rows are
// summed over: the lines of the last block behind the group's end (a row of a box is one 128-byte line) are
// overwritten with zeros in both operands before the MMA reads them, so that whatever the next group holds, NaN
// included, stays out of the sum.
//
// Warp roles, ring, accumulators and bounded waits are those of hgemm_tcgen05_kernel (gemm_kernel.cuh); unlike there
// neither this kernel nor its successor starts early (grouped_lib.cu says why). The
// reference has no counterpart (one product per launch, src/main.cu:11).
#pragma once

#include <cuda_bf16.h>

#include "activation.cuh"
#include "lib_state.h"
#include "ptx_sm100.cuh"
#include "sched.h"

namespace b200 {

enum GroupedForm : int {
    kFormForward = 0,
    kFormInput = 1,
    kFormWeight = 2,
};

constexpr int kGroupedEpiWarps = 8;
constexpr int kGroupedThreads = 64 + 32 * kGroupedEpiWarps;
constexpr uint32_t kGroupedMaxGroups = 1024;
constexpr uint32_t kGroupedBand = 8;  // blocks of rows a band of tiles is high

struct alignas(64) GroupedParams {
    CUtensorMap tm_narrow[4];  // forward, kernels of 32 columns: as tm_p with boxes {64, 64}, {64, 80}, {64, 96}, {64, 112}
    CUtensorMap tm_p;     // forward {K, N, groups} box {64, 128}; input {K, N, groups} box {64, 64}; weight {N, T} box {64, 64} or
                          // {64, T, N / 64} box {64, 64, 2}
    CUtensorMap tm_q[8];  // forward {K, T}, input {N, T}: boxes {64, 16 (i + 1)}; weight: [0] = {K, T} as P
    CUtensorMap tm_out;   // weight: {K, N, groups}, box of 128 bytes x 32 rows
    void *out;
    void *pre;             // forward: Z = sum + bias before the activation, or null
    const void *bias;      // forward: groups x N of the inputs' type, or null
    const void *residual;  // forward: T x N of C's type, added behind the activation, or null
    const int32_t *offsets;  // groups + 1, or null: one group of all rows
    uint32_t *error_word;
    uint32_t rows;         // T
    uint32_t groups;
    uint32_t p_dim;        // extent on P: N, K, N
    uint32_t q_dim;        // weight: K
    uint32_t k_blocks;     // forward, input: stages of the summed index
    uint32_t q_max;        // forward, input: most rows of a block
    uint32_t p_blocks;
    uint32_t q_blocks;     // weight
    uint32_t in_bf16;
    uint32_t out_type;     // 0 FP16, 1 BF16, 2 FP32
    uint32_t act;
    uint32_t accumulate;   // weight, FP32: add to the output
    uint32_t slice_rows;   // weight, dense: "group" g is rows [g, g + 1) * slice_rows of one long sum (0: groups as `offsets` says)
    uint32_t piece_shift;  // LONG: a piece is 1 << piece_shift k-blocks
    uint32_t p_wide, q_wide;  // weight: the operand's map takes two boxes with one copy (load_columns)
};

template <int FORM, int CG, int QT, int STAGES, int KPS, bool LONG>
struct GroupedTraits {
    static constexpr bool kWeight = FORM == kFormWeight;
    static_assert(CG == 1 || CG == 2, "single CTAs or CTA pairs");
    static_assert(QT == 32 || QT == 64 || QT == 128 || QT == 256, "columns of an accumulator");
    static_assert(!kWeight || (QT / CG == 128 && KPS == 1), "weight form: two 64-column boxes of Q per CTA");
    static_assert((kLongSumF32 / 64u) % KPS == 0, "whole stages per piece of a long sum");
    static constexpr uint32_t kChunk = QT >= 64 ? 32 : 16;  // accumulator columns an epilogue warp takes at a time
    static constexpr uint32_t kStep = 16u * CG;  // an MMA's columns come in these steps
    static constexpr uint32_t kPBytes = 128u * 128u;
    static constexpr uint32_t kQBytes = (QT / CG) * 128u;
    static constexpr uint32_t kBlockBytes = kPBytes + kQBytes;
    static constexpr uint32_t kStageBytes = KPS * kBlockBytes;
    static constexpr uint32_t kTmemCols = 2u * QT;
    static constexpr uint32_t kStagingBytes = kWeight ? kGroupedEpiWarps * 4096u : 0u;
    static constexpr uint32_t kTableBytes = kWeight ? 0u : 2u * 4u * (kGroupedMaxGroups + 4u);
    static constexpr uint32_t kBarrierBytes = 256;
    static constexpr uint32_t kSmemBytes = 1024 + STAGES * kStageBytes + kStagingBytes + kTableBytes + kBarrierBytes;
    static_assert(kBlockBytes % 1024 == 0, "operand slabs must keep 1024-byte alignment");
    static_assert(kSmemBytes <= 232448, "exceeds 227 KB of shared memory");
    static_assert((kWeight ? 32u : 16u) * STAGES + 40u <= kBarrierBytes, "barrier area too small");
    static_assert(QT / CG <= 128, "rows of Q a CTA stages: the highest box has 128");
    static_assert(STAGES <= 16, "one lane of a warp per barrier to set up");
};

// One piece of work: an output tile and, in the weight form, the rows it sums over.
struct GroupedTile {
    uint32_t group;
    uint32_t p0;     // first index on P of the whole tile (of the pair)
    uint32_t q0;     // forward, input: first row; weight: first index on Q
    uint32_t valid;  // forward, input: rows stored; weight: rows summed over
    uint32_t n_mma;  // columns of the MMA
    uint32_t row0;   // weight: first row of the group
};

__device__ __forceinline__ uint32_t round_up_u32(uint32_t v, uint32_t step) {
    return (v + step - 1u) / step * step;
}

// Rows of a group as the offsets say, held within [0, T].
__device__ __forceinline__ uint32_t held_offset(int32_t v, uint32_t rows) {
    return v < 0 ? 0u : min(static_cast<uint32_t>(v), rows);
}

// Block index inside a group -> (block on Q, block on P): bands of kGroupedBand blocks of rows, the row block
// moving fastest, so that the tiles that run at one time share the weights of a few P blocks and the rows
// of at most eight Q blocks; odd bands walk P backwards.
__device__ __forceinline__ void band_coord(uint32_t local, uint32_t nq, uint32_t np, uint32_t *q, uint32_t *p) {
    if (nq == 1) {
        *q = 0;
        *p = local;
        return;
    }
    const uint32_t per_band = kGroupedBand * np;
    const uint32_t band = local / per_band;
    const uint32_t rem = local - band * per_band;
    const uint32_t high = min(kGroupedBand, nq - band * kGroupedBand);
    const uint32_t pi = rem / high;
    *q = band * kGroupedBand + (rem - pi * high);
    *p = (band & 1u) ? np - 1u - pi : pi;
}

// Forward and input form: tile id -> tile. off / cum: the table of offsets and of row blocks before each group.
template <int CG>
__device__ __forceinline__ void rows_tile(const GroupedParams &p, const uint32_t *off, const uint32_t *cum, uint32_t p_blocks,
                                          uint32_t width, uint32_t t, GroupedTile &out) {
    const uint32_t block = t / p_blocks;
    uint32_t lo = 0, hi = p.groups;  // the largest g with cum[g] <= block; cum[groups] > block
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) >> 1;
        if (cum[mid] <= block) lo = mid; else hi = mid;
    }
    const uint32_t first = cum[lo], nq = cum[lo + 1u] - first;
    const uint32_t start = off[lo], r = off[lo + 1u] - start;
    uint32_t qb, pb;
    band_coord(t - first * p_blocks, nq, p_blocks, &qb, &pb);
    const uint32_t size = round_up_u32((r + nq - 1u) / nq, 16u * CG);  // even blocks
    out.group = lo;
    out.p0 = pb * width;
    out.q0 = start + qb * size;
    out.valid = min(size, r - qb * size);
    out.n_mma = round_up_u32(out.valid, 16u * CG);
    out.row0 = 0;
}

// Weight form: tile id -> tile (the same number of tiles for every group).
template <int CG, int QT>
__device__ __forceinline__ void weight_tile(const GroupedParams &p, uint32_t t, GroupedTile &out) {
    const uint32_t per_group = p.p_blocks * p.q_blocks;
    const uint32_t g = t / per_group;
    uint32_t qb, pb;
    band_coord(t - g * per_group, p.q_blocks, p.p_blocks, &qb, &pb);
    uint32_t start = 0, end = p.rows;
    if (p.offsets) {
        start = held_offset(__ldg(p.offsets + g), p.rows);
        end = max(held_offset(__ldg(p.offsets + g + 1), p.rows), start);
    } else if (p.slice_rows) {
        start = g * p.slice_rows;  // (every slice holds rows: start < rows)
        end = min(start + p.slice_rows, p.rows);
    }
    out.group = g;
    out.p0 = pb * 128u * CG;
    out.q0 = qb * QT;
    out.valid = end - start;
    out.n_mma = min(static_cast<uint32_t>(QT), round_up_u32(p.q_dim - out.q0, 64u * CG));  // whole 64-column boxes per CTA
    out.row0 = start;
}

// Weight form: 64 rows of 128 columns from column x (a multiple of 64) on, as two boxes of 64 columns one behind the other. A matrix
// whose width is a multiple of 64 is mapped as {64, rows, width / 64}, where one copy takes both (`wide`): issuing
// the copies is what the producer's one thread spends its time on.
template <bool PAIR>
__device__ __forceinline__ void load_columns(uint32_t dst, const CUtensorMap &map, uint32_t wide, int32_t x, int32_t row, uint32_t bar) {
    if (wide) {
        if (PAIR) tma_load_3d_pair(dst, &map, 0, row, x >> 6, bar); else tma_load_3d(dst, &map, 0, row, x >> 6, bar);
    } else if (PAIR) {
        tma_load_2d_pair(dst, &map, x, row, bar);
        tma_load_2d_pair(dst + 8192u, &map, x + 64, row, bar);
    } else {
        tma_load_2d(dst, &map, x, row, bar);
        tma_load_2d(dst + 8192u, &map, x + 64, row, bar);
    }
}

// An mbarrier wait that also acquires what other CTAs of the cluster wrote before they arrived.
__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t"
        "}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}

__device__ __forceinline__ uint32_t pack2_typed(uint32_t lo_f32_bits, uint32_t hi_f32_bits, uint32_t bf16) {
    if (bf16) {
        __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(lo_f32_bits), __uint_as_float(hi_f32_bits));
        return *reinterpret_cast<uint32_t *>(&b);
    }
    return pack_half2_rn(lo_f32_bits, hi_f32_bits);
}

// COUNT columns of a transposed accumulator (this lane: output column `col`, register j: row q0 + j) to
// row-major memory. 16-bit outputs whose rows are a whole number of 4-byte words leave two columns at a
// time: neighbouring lanes exchange halves, the even lane takes the even rows and the odd lane the odd rows,
// so that a warp stores two rows of 64 bytes with one instruction instead of one.
template <int COUNT>
__device__ __forceinline__ void store_transposed(void *out, uint32_t out_type, uint32_t q0, uint32_t valid, uint32_t col,
                                                 uint32_t dim, const uint32_t *r, uint32_t lane) {
    if (out_type == 2u) {
        float *dst = static_cast<float *>(out) + static_cast<size_t>(q0) * dim + col;
#pragma unroll
        for (uint32_t j = 0; j < COUNT; ++j) {
            if (j < valid) dst[static_cast<size_t>(j) * dim] = __uint_as_float(r[j]);
        }
        return;
    }
    if ((dim & 1u) == 0) {
        const uint32_t odd = lane & 1u;
        uint32_t *dst = static_cast<uint32_t *>(out) + ((static_cast<size_t>(q0) + odd) * dim + (col & ~1u)) / 2u;
#pragma unroll
        for (uint32_t j = 0; j < COUNT; j += 2) {
            const uint32_t mine = pack2_typed(r[j], r[j + 1], out_type);  // rows j and j + 1 of this column
            const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
            // even lane: row j of (this, next) column; odd lane: row j + 1 of (previous, this)
            const uint32_t word = odd ? __byte_perm(other, mine, 0x7632) : __byte_perm(mine, other, 0x5410);
            if (j + odd < valid) dst[static_cast<size_t>(j) * (dim / 2u)] = word;
        }
        return;
    }
    unsigned short *dst = static_cast<unsigned short *>(out) + static_cast<size_t>(q0) * dim + col;
#pragma unroll
    for (uint32_t j = 0; j < COUNT; ++j) {
        if (j < valid) dst[static_cast<size_t>(j) * dim] = static_cast<unsigned short>(pack2_typed(r[j], r[j], out_type));
    }
}

// Adds the residual's values at the same places. All of them are read before any is stored over (it may be C itself).
template <int COUNT>
__device__ __forceinline__ void add_residual(const void *residual, uint32_t type, uint32_t q0, uint32_t valid, uint32_t col,
                                             uint32_t dim, uint32_t *r) {
    const size_t at = static_cast<size_t>(q0) * dim + col;
    float v[COUNT];
    // (one loop per type: a choice between them inside would be a branch between every two loads, and the loads
    // would come back one at a time -- 28 us at 777 x 4099)
    if (type == 2u) {
#pragma unroll
        for (uint32_t j = 0; j < COUNT; ++j) v[j] = j < valid ? static_cast<const float *>(residual)[at + static_cast<size_t>(j) * dim] : 0.f;
    } else {
        unsigned short bits[COUNT];
#pragma unroll
        for (uint32_t j = 0; j < COUNT; ++j) {
            bits[j] = j < valid ? static_cast<const unsigned short *>(residual)[at + static_cast<size_t>(j) * dim] : static_cast<unsigned short>(0);
        }
#pragma unroll
        for (uint32_t j = 0; j < COUNT; ++j) v[j] = type == 1u ? __uint_as_float(static_cast<uint32_t>(bits[j]) << 16) : __half2float(__ushort_as_half(bits[j]));
    }
#pragma unroll
    for (uint32_t j = 0; j < COUNT; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + v[j]);
}

// What becomes of COUNT columns of an accumulator of the forward or input form.
template <int FORM, int COUNT>
__device__ __forceinline__ void finish_rows(const GroupedParams &p, uint32_t *r, float bias, uint32_t q0, uint32_t valid, uint32_t col,
                                            uint32_t col_end, uint32_t lane) {
    valid = col < col_end ? valid : 0u;  // (lanes without a column still take part in the exchanges)
    if (FORM == kFormForward) {
        if (p.bias) {
#pragma unroll
            for (uint32_t j = 0; j < COUNT; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + bias);
        }
        if (p.pre) store_transposed<COUNT>(p.pre, p.out_type, q0, valid, col, p.p_dim, r, lane);
        act_apply<COUNT>(r, p.act);
        if (p.residual) add_residual<COUNT>(p.residual, p.out_type, q0, valid, col, p.p_dim, r);
    }
    store_transposed<COUNT>(p.out, p.out_type, q0, valid, col, p.p_dim, r, lane);
}

// COUNT (16 or 32) accumulator columns of this lane's row.
template <int COUNT>
__device__ __forceinline__ void tmem_ld_columns(uint32_t taddr, uint32_t *r) {
    if (COUNT == 32) tmem_ld_32x32b_x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(r));
    else tmem_ld_32x32b_x16(taddr, *reinterpret_cast<uint32_t(*)[16]>(r));
}

template <int FORM, int CG, int QT, int STAGES, int KPS, bool LONG>
__global__ void __launch_bounds__(kGroupedThreads, 1) hgemm_grouped_kernel(const __grid_constant__ GroupedParams p) {
    using T = GroupedTraits<FORM, CG, QT, STAGES, KPS, LONG>;
    constexpr bool WEIGHT = FORM == kFormWeight;
    constexpr bool P_MN = FORM != kFormForward;  // P is read MN-major
    constexpr uint32_t kStepK = 64u;             // summed index per k-block

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t *base_ptr = smem_raw + (base - raw_addr);
    const uint32_t staging = base + STAGES * T::kStageBytes;
    uint8_t *staging_ptr = base_ptr + STAGES * T::kStageBytes;
    uint32_t *off = reinterpret_cast<uint32_t *>(staging_ptr + T::kStagingBytes);
    uint32_t *cum = off + kGroupedMaxGroups + 4u;
    const uint32_t bars = staging + T::kStagingBytes + T::kTableBytes;
    uint8_t *bars_ptr = staging_ptr + T::kStagingBytes + T::kTableBytes;
    // full[STAGES] | empty[STAGES] | tmem_full[2] | tmem_empty[2] | tmem base | abort | tail_full[STAGES] | tail_ready[STAGES]
    const uint32_t full_bar = bars;
    const uint32_t empty_bar = bars + 8u * STAGES;
    const uint32_t tfull_bar = bars + 16u * STAGES;
    const uint32_t tempty_bar = tfull_bar + 16u;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(bars_ptr + 16u * STAGES + 32u);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    // pairs in the weight form: a stage that holds a tail has landed in this CTA / has been cleared in both CTAs. One of
    // each per stage: several tails may be in the ring at once, and a stage is armed again only after its MMAs.
    const uint32_t tail_bar = tfull_bar + 40u;
    const uint32_t ready_bar = tail_bar + 8u * STAGES;

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t cta_rank = (CG == 2) ? cluster_cta_rank() : 0u;
    const uint32_t worker = blockIdx.x / CG;
    const uint32_t workers = gridDim.x / CG;

    if (warp == 0) {
        if (lane < static_cast<uint32_t>(STAGES)) {
            mbar_init(full_bar + 8u * lane, 1);
            mbar_init(empty_bar + 8u * lane, 1);
        } else if (lane < static_cast<uint32_t>(STAGES) + 2u) {
            const uint32_t a = lane - STAGES;
            mbar_init(tfull_bar + 8u * a, 1);
            mbar_init(tempty_bar + 8u * a, kGroupedEpiWarps * CG);
        } else if (lane == static_cast<uint32_t>(STAGES) + 2u) {
            *abort_flag = 0;
        }
        if (WEIGHT && CG == 2 && lane < static_cast<uint32_t>(STAGES)) {
            mbar_init(tail_bar + 8u * lane, 1);
            mbar_init(ready_bar + 8u * lane, 2);  // the MMA warps of both CTAs
        }
        fence_mbar_init();
        __syncwarp();
    }
    if (warp == 2 && lane == 0) {
        tma_prefetch_desc(&p.tm_p);
        tma_prefetch_desc(&p.tm_q[0]);
        if (WEIGHT) tma_prefetch_desc(&p.tm_out);
    }
    if (warp == 1) {
        tmem_alloc<CG>(smem_u32(const_cast<uint32_t *>(tmem_slot)), T::kTmemCols);
        tmem_relinquish<CG>();
    }

    uint32_t tiles;
    if (WEIGHT) {
        tiles = p.groups * p.p_blocks * p.q_blocks;
    } else {
        for (uint32_t g = threadIdx.x; g <= p.groups; g += kGroupedThreads) {
            off[g] = p.offsets ? held_offset(__ldg(p.offsets + g), p.rows) : (g == 0 ? 0u : p.rows);
        }
        __syncthreads();
        if (warp == 0) {
            // Blocks of at most q_max rows before each group: a running sum over 32 groups at a time. The offsets are put in order by
            // a running maximum first: the groups then hold no more rows than there are, and the sum fits 32 bits.
            uint32_t total = 0, high = off[0];
            for (uint32_t g0 = 0; g0 < p.groups; g0 += 32u) {
                const uint32_t g = g0 + lane;
                uint32_t end = g < p.groups ? off[g + 1u] : 0u;
#pragma unroll
                for (uint32_t d = 1; d < 32; d <<= 1) {
                    const uint32_t up = __shfl_up_sync(0xffffffffu, end, d);
                    if (lane >= d) end = max(end, up);
                }
                end = max(end, high);
                const uint32_t before = __shfl_up_sync(0xffffffffu, end, 1);
                const uint32_t start = lane == 0 ? high : before;
                high = __shfl_sync(0xffffffffu, end, 31);
                const uint32_t blocks = (end - start + p.q_max - 1u) / p.q_max;  // (none past the last group: end is start)
                uint32_t sum = blocks;
#pragma unroll
                for (uint32_t d = 1; d < 32; d <<= 1) {
                    const uint32_t up = __shfl_up_sync(0xffffffffu, sum, d);
                    if (lane >= d) sum += up;
                }
                if (g < p.groups) {
                    cum[g] = total + sum - blocks;
                    off[g + 1u] = end;
                }
                total += __shfl_sync(0xffffffffu, sum, 31);
            }
            if (lane == 0) cum[p.groups] = total;
        }
    }
    tcgen05_fence_before_sync();
    __syncthreads();
    if (CG == 2) cluster_sync_all();  // the peer's copies and arrivals target this CTA's barriers
    tcgen05_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    // Columns of the result per tile. Where a tile takes few rows its time is that of reading its weights, and the
    // kernel's that of the SM with the most of them: 26 groups of 1024 columns are 208 tiles of 128, two for an SM, or 286 of
    // 96, two for an SM as well. The width with the least waves x (width + the rows' share of a stage and a tile's fixed
    // cost, about 40 columns' worth) is taken; the MMA's other rows multiply what lies in the slab and are not stored.
    uint32_t width = 128u * CG, p_blocks = p.p_blocks;
    if (!WEIGHT) {
        const uint32_t row_blocks = cum[p.groups];
        if (QT == 32) {
            uint32_t least = 0xffffffffu;
            for (uint32_t w = 128u; w >= 64u; w -= FORM == kFormForward ? 16u : 64u) {
                const uint32_t n = (p.p_dim + w - 1u) / w;
                const uint32_t cost = (row_blocks * n + workers - 1u) / workers * (w + 40u);
                if (cost < least) {
                    least = cost;
                    width = w;
                    p_blocks = n;
                }
            }
        }
        tiles = row_blocks * p_blocks;
    }
    const CUtensorMap *p_map = QT == 32 && FORM == kFormForward && width < 128u ? &p.tm_narrow[width / 16u - 4u] : &p.tm_p;
    const uint32_t p_bytes = QT == 32 ? width * 128u : T::kPBytes;  // of a slab of P, as staged

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        bool chosen;
        elect_lane(&chosen);
        if (chosen) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t t = worker; ok && t < tiles; t += workers) {
                GroupedTile tile;
                if (WEIGHT) weight_tile<CG, QT>(p, t, tile); else rows_tile<CG>(p, off, cum, p_blocks, width, t, tile);
                const uint32_t blocks = WEIGHT ? (tile.valid + kStepK - 1u) / kStepK : p.k_blocks;
                const uint32_t q_rows = tile.n_mma / CG;  // forward, input: rows this CTA stages
                const int32_t p_at = static_cast<int32_t>(tile.p0 + cta_rank * 128u);
                const int32_t q_at = static_cast<int32_t>(tile.q0 + cta_rank * q_rows);
                const CUtensorMap *q_map = &p.tm_q[WEIGHT ? 0u : q_rows / 16u - 1u];
                const uint32_t bytes = KPS * (p_bytes + (WEIGHT ? T::kQBytes : q_rows * 128u));
                const uint32_t rest = WEIGHT ? (tile.valid & (kStepK - 1u)) : 0u;  // rows of a tail, 0: whole blocks
                const uint32_t whole = blocks - (rest != 0 ? 1u : 0u);
                for (uint32_t kb = 0; kb < whole; ++kb) {
                    if (!mbar_wait(empty_bar + 8u * stage, phase ^ 1u, abort_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t slot = base + stage * T::kStageBytes;
                    uint32_t bar = full_bar + 8u * stage;
                    if (CG == 2) {
                        // both CTAs' copies complete on the leader's barrier, which expects the bytes of both
                        if (cta_rank == 0) mbar_arrive_expect_tx(bar, 2u * bytes);
                        bar = map_to_cta(bar, 0);
                    } else {
                        mbar_arrive_expect_tx(bar, bytes);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < KPS; ++j) {
                        const uint32_t sp = slot + j * T::kBlockBytes;
                        const uint32_t sq = sp + T::kPBytes;
                        const int32_t kx = static_cast<int32_t>((kb * KPS + j) * kStepK);  // past the end: zeros in both operands
                        if (WEIGHT) {
                            const int32_t row = static_cast<int32_t>(tile.row0) + kx;
                            load_columns<CG == 2>(sp, p.tm_p, p.p_wide, p_at, row, bar);
                            load_columns<CG == 2>(sq, p.tm_q[0], p.q_wide, q_at, row, bar);
                        } else {
                            const int32_t g = static_cast<int32_t>(tile.group);
                            if (FORM == kFormForward) {
                                if (CG == 2) tma_load_3d_pair(sp, p_map, kx, p_at, g, bar); else tma_load_3d(sp, p_map, kx, p_at, g, bar);
                            } else {
#pragma unroll
                                for (int32_t h = 0; h < 2; ++h) {
                                    if (QT == 32 && h == 1 && width < 128u) break;
                                    if (CG == 2) tma_load_3d_pair(sp + h * 8192u, &p.tm_p, p_at + h * 64, kx, g, bar);
                                    else tma_load_3d(sp + h * 8192u, &p.tm_p, p_at + h * 64, kx, g, bar);
                                }
                            }
                            if (CG == 2) tma_load_2d_pair(sq, q_map, kx, q_at, bar); else tma_load_2d(sq, q_map, kx, q_at, bar);
                        }
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (WEIGHT && ok && rest != 0) {
                    // the last block of a group that does not fill it: the MMA warp of each CTA clears its lines behind the
                    // group's end, so in a pair each CTA's copies complete on a barrier of its own
                    if (!mbar_wait(empty_bar + 8u * stage, phase ^ 1u, abort_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sp = base + stage * T::kStageBytes;
                    uint32_t bar = full_bar + 8u * stage;
                    if (CG == 2) {
                        if (cta_rank == 0) mbar_arrive(bar);  // keeps the stage's phase; nothing lands there
                        bar = tail_bar + 8u * stage;
                    }
                    mbar_arrive_expect_tx(bar, bytes);
                    const int32_t row = static_cast<int32_t>(tile.row0 + whole * kStepK);
                    load_columns<false>(sp, p.tm_p, p.p_wide, p_at, row, bar);
                    load_columns<false>(sp + T::kPBytes, p.tm_q[0], p.q_wide, q_at, row, bar);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        // The whole warp walks the tiles; one lane of the leader issues. In the weight form all lanes clear the lines
        // of a tail (in both CTAs of a pair).
        bool chosen;
        const uint32_t issuer = elect_lane(&chosen);
        if (cta_rank == 0 || WEIGHT) {
            const uint32_t idesc_base = umma_idesc_f16_f32(128 * CG, 0) | (P_MN ? kUmmaIdescAMn : 0u) | (WEIGHT ? (1u << 16) : 0u) |
                                        (p.in_bf16 ? kUmmaIdescBf16 : 0u);
            uint32_t stage = 0, phase = 0, it = 0;
            uint32_t tail_phase = 0;  // bit s: parity of stage s's next tail
            bool ok = true;
            for (uint32_t t = worker; ok && t < tiles; t += workers) {
                GroupedTile tile;
                if (WEIGHT) weight_tile<CG, QT>(p, t, tile); else rows_tile<CG>(p, off, cum, p_blocks, width, t, tile);
                const uint32_t blocks = WEIGHT ? (tile.valid + kStepK - 1u) / kStepK : p.k_blocks;
                if (blocks == 0) continue;
                const uint32_t rest = WEIGHT ? (tile.valid & (kStepK - 1u)) : 0u;  // rows of a tail, 0: whole blocks
                const uint32_t idesc = idesc_base | ((tile.n_mma >> 3) << 17);
                const uint32_t whole = blocks - (rest != 0 ? 1u : 0u);
                uint32_t d_tmem = tmem_base + (it & 1u) * QT;
                if (cta_rank == 0 && chosen) {
                    if (!mbar_wait(tempty_bar + 8u * (it & 1u), ((it >> 1) & 1u) ^ 1u, abort_flag)) ok = false;
                    tcgen05_fence_after_sync();
                    uint32_t begun = 0;  // 1: the accumulator holds a part of this piece
                    for (uint32_t kb = 0; ok && kb < whole; ++kb) {
                        if (LONG && kb != 0 && ((kb * KPS) & ((1u << p.piece_shift) - 1u)) == 0) {
                            // the next piece, in the other accumulator
                            if (CG == 1) umma_commit(tfull_bar + 8u * (it & 1u)); else umma_commit_pair(tfull_bar + 8u * (it & 1u), 0x3);
                            ++it;
                            d_tmem = tmem_base + (it & 1u) * QT;
                            begun = 0;
                            if (!mbar_wait(tempty_bar + 8u * (it & 1u), ((it >> 1) & 1u) ^ 1u, abort_flag)) {
                                ok = false;
                                break;
                            }
                            tcgen05_fence_after_sync();
                        }
                        if (!mbar_wait(full_bar + 8u * stage, phase, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tcgen05_fence_after_sync();
                        const uint32_t slot = base + stage * T::kStageBytes;
#pragma unroll
                        for (uint32_t j = 0; j < KPS; ++j) {
                            const uint32_t sp = slot + j * T::kBlockBytes, sq = sp + T::kPBytes;
                            const uint64_t dp = P_MN ? umma_smem_desc_sw128_mn(sp, 8192u) : umma_smem_desc_sw128(sp);
                            const uint64_t dq = WEIGHT ? umma_smem_desc_sw128_mn(sq, 8192u) : umma_smem_desc_sw128(sq);
#pragma unroll
                            for (uint32_t k = 0; k < 4; ++k) {
                                umma_f16<CG>(d_tmem, dp + (P_MN ? 128u : 2u) * k, dq + (WEIGHT ? 128u : 2u) * k, idesc,
                                             (j > 0 || k > 0) ? 1u : begun);
                            }
                        }
                        begun = 1;
                        if (CG == 1) umma_commit(empty_bar + 8u * stage); else umma_commit_pair(empty_bar + 8u * stage, 0x3);
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
                if constexpr (WEIGHT) {
                    // every lane follows: where the ring stands, and whether to go on
                    ok = __shfl_sync(0xffffffffu, ok ? 1u : 0u, issuer) != 0;
                    it = __shfl_sync(0xffffffffu, it, issuer);
                    if (CG == 2 && cta_rank != 0) {
                        const uint32_t at = stage + blocks - (rest != 0 ? 1u : 0u);
                        stage = at % STAGES;
                        phase ^= (at / STAGES) & 1u;
                    } else {
                        stage = __shfl_sync(0xffffffffu, stage, issuer);
                        phase = __shfl_sync(0xffffffffu, phase, issuer);
                    }
                    if (ok && rest != 0) {
                        const uint32_t slot = base + stage * T::kStageBytes;
                        const uint32_t landed_bar = (CG == 2 ? tail_bar : full_bar) + 8u * stage;
                        const uint32_t parity = CG == 2 ? (tail_phase >> stage) & 1u : phase;
                        uint32_t landed = 1;
                        if (chosen) landed = mbar_wait(landed_bar, parity, abort_flag) ? 1u : 0u;
                        landed = __shfl_sync(0xffffffffu, landed, issuer);
                        if (landed) {
                            // each lane passes the completed barrier itself: the copies' bytes are then ordered before its stores
                            mbar_try_wait(landed_bar, parity);
                            const uint32_t steps = (rest + 15u) / 16u;  // MMAs of 16 rows that hold any
                            const uint32_t words = (steps * 16u - rest) * 8u;  // 16-byte words behind the end, per box
                            for (uint32_t i = lane; i < words * 4u; i += 32u) {
                                const uint32_t box = i / words, w = i - box * words;
                                // four boxes of 8 KB, one behind the other: two of P, two of Q
                                *reinterpret_cast<uint4 *>(base_ptr + stage * T::kStageBytes + box * 8192u + rest * 128u + w * 16u) =
                                    make_uint4(0u, 0u, 0u, 0u);
                            }
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (chosen) {
                                if (CG == 2) mbar_arrive_cluster(map_to_cta(ready_bar + 8u * stage, 0));
                                if (cta_rank == 0) {
                                    if (CG == 2) {
                                        // both CTAs have cleared their parts, and the stage's own barrier has passed its phase
                                        if (!mbar_wait(ready_bar + 8u * stage, parity, abort_flag) ||
                                            !mbar_wait(full_bar + 8u * stage, phase, abort_flag)) {
                                            ok = false;
                                        } else {
                                            mbar_try_wait_cluster(ready_bar + 8u * stage, parity);
                                        }
                                    }
                                    if (ok) {
                                        tcgen05_fence_after_sync();
                                        const uint64_t dp = umma_smem_desc_sw128_mn(slot, 8192u);
                                        const uint64_t dq = umma_smem_desc_sw128_mn(slot + T::kPBytes, 8192u);
                                        for (uint32_t k = 0; k < steps; ++k) {
                                            umma_f16<CG>(d_tmem, dp + 128u * k, dq + 128u * k, idesc, (blocks > 1u || k > 0) ? 1u : 0u);  // (joins the last piece)
                                        }
                                        if (CG == 1) umma_commit(empty_bar + 8u * stage); else umma_commit_pair(empty_bar + 8u * stage, 0x3);
                                    }
                                }
                            }
                        } else {
                            ok = false;
                        }
                        ok = __shfl_sync(0xffffffffu, ok ? 1u : 0u, issuer) != 0;
                        tail_phase ^= 1u << stage;
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
                if (cta_rank == 0 && chosen && ok) {
                    if (CG == 1) umma_commit(tfull_bar + 8u * (it & 1u)); else umma_commit_pair(tfull_bar + 8u * (it & 1u), 0x3);
                }
                if (!WEIGHT) {
                    ok = __shfl_sync(0xffffffffu, ok ? 1u : 0u, issuer) != 0;
                    it = __shfl_sync(0xffffffffu, it, issuer);
                }
                ++it;
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ epilogue
        // Warp w may read tensor-memory lanes 32 (w % 4) .. + 31; the two warps of a quadrant take alternate chunks of
        // columns. LONG: the pieces of a tile are added up in `run` as they come; else there is one piece.
        const uint32_t q = warp & 3u, half = (warp - 2u) >> 2;
        constexpr uint32_t W = T::kChunk;
        constexpr uint32_t kChunks = QT / W / 2u;  // of this warp
        uint8_t *my_ptr = staging_ptr + (warp - 2u) * 4096u;
        const uint32_t my_staging = staging + (warp - 2u) * 4096u;
        uint32_t it = 0;
        bool alive = true;
        // waits for the accumulator of piece `it`; false: given up
        auto wait_piece = [&]() -> bool {
            uint32_t ready = 1;
            if (lane == 0) ready = mbar_wait(tfull_bar + 8u * (it & 1u), (it >> 1) & 1u, abort_flag) ? 1u : 0u;
            ready = __shfl_sync(0xffffffffu, ready, 0);
            tcgen05_fence_after_sync();
            return ready != 0;
        };
        auto release_piece = [&]() {
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (CG == 1) mbar_arrive(tempty_bar + 8u * (it & 1u)); else mbar_arrive_cluster(map_to_cta(tempty_bar + 8u * (it & 1u), 0));
            }
            ++it;
        };
        for (uint32_t t = worker; alive && t < tiles; t += workers) {
            GroupedTile tile;
            if (WEIGHT) weight_tile<CG, QT>(p, t, tile); else rows_tile<CG>(p, off, cum, p_blocks, width, t, tile);
            const bool summed = !WEIGHT || tile.valid != 0;  // a group without rows: a gradient of zeros, no accumulator
            const uint32_t p_warp = tile.p0 + cta_rank * 128u + q * 32u;  // first index on P of this warp's lanes
            const uint32_t lanes = tmem_base + ((q * 32u) << 16);
            const uint32_t cols = WEIGHT ? min(static_cast<uint32_t>(QT), p.q_dim - tile.q0) : tile.valid;  // columns stored
            // forward, input: this lane's output column, and where the columns of this tile end
            const uint32_t col = p_warp + lane, col_end = QT == 32 ? min(p.p_dim, tile.p0 + width) : p.p_dim;
            const bool live = p_warp < col_end && (summed || !p.accumulate);
            float bias = 0.f;
            if (FORM == kFormForward && p.bias && col < col_end) {
                const size_t at = static_cast<size_t>(tile.group) * p.p_dim + col;
                bias = p.in_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p.bias)[at])
                                 : __half2float(static_cast<const __half *>(p.bias)[at]);
            }
            if (FORM == kFormForward && p.residual && live) {
                // the residual's rows of this warp, into L2 while the sums run: one row of a chunk per lane.
                const size_t size = p.out_type == 2u ? 4u : 2u;
                for (uint32_t at = half * W + lane; at < cols && lane < W; at += 2u * W) {
                    const uint8_t *row = static_cast<const uint8_t *>(p.residual) + (static_cast<size_t>(tile.q0 + at) * p.p_dim + p_warp) * size;
                    prefetch_l2(row);
                    if (size == 4u) prefetch_l2(row + min(124u, (p.p_dim - p_warp - 1u) * 4u));  // 128 bytes may lie in two lines
                }
            }
            uint32_t run[LONG ? kChunks * W : 1];
            // LONG: first column of group i of 16 running sums. The two warps of a quadrant alternate every `span` columns:
            // a chunk, or, in the weight form, what 128 bytes of a row of the result take.
            const uint32_t span = WEIGHT && p.out_type != 2u ? 64u : W;
            auto run_column = [&](uint32_t i) -> uint32_t { return (2u * (i * 16u / span) + half) * span + i * 16u % span; };
            if constexpr (LONG) {
                const uint32_t k_blocks = WEIGHT ? (tile.valid + kStepK - 1u) / kStepK : p.k_blocks * KPS;
                // (a tail joins the last piece, so pieces are counted over the whole blocks)
                const uint32_t whole = WEIGHT ? tile.valid / kStepK : k_blocks;
                const uint32_t pieces = max((whole + (1u << p.piece_shift) - 1u) >> p.piece_shift, k_blocks != 0 ? 1u : 0u);
#pragma unroll
                for (uint32_t j = 0; j < kChunks * W; ++j) run[j] = 0u;
                for (uint32_t piece = 0; alive && piece < pieces; ++piece) {
                    alive = wait_piece();
                    if (!alive) break;
#pragma unroll
                    for (uint32_t c = 0; c < kChunks * W / 16u; ++c) {
                        const uint32_t at = run_column(c);
                        if (at < cols) {
                            uint32_t r[16];
                            tmem_ld_32x32b_x16(lanes + (it & 1u) * QT + at, r);
                            tmem_ld_wait();
#pragma unroll
                            for (uint32_t j = 0; j < 16; ++j) {
                                run[c * 16u + j] = __float_as_uint(__uint_as_float(run[c * 16u + j]) + __uint_as_float(r[j]));
                            }
                        }
                    }
                    release_piece();
                }
            } else if (summed) {
                alive = wait_piece();
            }
            if (!alive) break;
            const uint32_t taddr = lanes + (it & 1u) * QT;
            if (!WEIGHT) {
                if (live) {
                    if constexpr (LONG) {
#pragma unroll
                        for (uint32_t i = 0; i < kChunks * W / 16u; ++i) {  // (16 at a time: the running sums leave few registers)
                            const uint32_t at = run_column(i);
                            if (at < cols) finish_rows<FORM, 16>(p, run + i * 16u, bias, tile.q0 + at, cols - at, col, col_end, lane);
                        }
                    } else {
#pragma unroll 1
                        for (uint32_t at = half * W; at < cols; at += 2u * W) {
                            uint32_t r[W];
                            tmem_ld_columns<W>(taddr + at, r);
                            tmem_ld_wait();
                            finish_rows<FORM, W>(p, r, bias, tile.q0 + at, cols - at, col, col_end, lane);
                        }
                    }
                }
            } else if (live) {
                // rows of the result: through swizzled staging (32 rows of 128 bytes) and TMA, which clips what lies
                // past N and K; with `accumulate` the copy adds to what is there
                uint8_t *row_ptr = my_ptr + lane * 128u;
                auto staging_free = [&]() {
                    if (lane == 0) tma_store_wait_read<0>();  // the last copy out of it has read it
                    __syncwarp();
                };
                auto send = [&](uint32_t at) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        const int32_t x = static_cast<int32_t>(tile.q0 + at), y = static_cast<int32_t>(p_warp);
                        const int32_t z = static_cast<int32_t>(tile.group);
                        if (p.accumulate) tma_reduce_add_3d(&p.tm_out, my_staging, x, y, z); else tma_store_3d(&p.tm_out, my_staging, x, y, z);
                        tma_store_commit();
                    }
                };
                auto put_f32 = [&](const uint32_t *r) {
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        *reinterpret_cast<uint4 *>(row_ptr + ((j ^ (lane & 7u)) << 4)) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
                    }
                };
                // 32 values of this lane's row, as part 0 or 1 of its 128 bytes
                auto put_16 = [&](const uint32_t *r, uint32_t part) {
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        uint4 v;
                        v.x = pack2_typed(r[8 * j + 0], r[8 * j + 1], p.out_type);
                        v.y = pack2_typed(r[8 * j + 2], r[8 * j + 3], p.out_type);
                        v.z = pack2_typed(r[8 * j + 4], r[8 * j + 5], p.out_type);
                        v.w = pack2_typed(r[8 * j + 6], r[8 * j + 7], p.out_type);
                        *reinterpret_cast<uint4 *>(row_ptr + (((part * 4u + j) ^ (lane & 7u)) << 4)) = v;
                    }
                };
                if constexpr (LONG) {
                    if (p.out_type == 2u) {
#pragma unroll
                        for (uint32_t i = 0; i < kChunks; ++i) {
                            const uint32_t at = (2u * i + half) * 32u;
                            if (at < cols) {
                                staging_free();
                                put_f32(run + i * 32u);
                                send(at);
                            }
                        }
                    } else {
#pragma unroll
                        for (uint32_t i = 0; i < kChunks / 2u; ++i) {
                            const uint32_t at = (2u * i + half) * 64u;
                            if (at < cols) {
                                staging_free();
                                put_16(run + i * 64u, 0);
                                put_16(run + i * 64u + 32u, 1);
                                send(at);
                            }
                        }
                    }
                } else {
                    const bool f32 = p.out_type == 2u;
                    const uint32_t width = f32 ? 32u : 64u;  // columns of 128 bytes
#pragma unroll 1
                    for (uint32_t at = half * width; at < cols; at += 2u * width) {
                        staging_free();
#pragma unroll 1
                        for (uint32_t part = 0; part * 32u < width; ++part) {
                            uint32_t r[32];
                            if (summed) {
                                tmem_ld_32x32b_x32(taddr + at + part * 32u, r);
                                tmem_ld_wait();
                            } else {
#pragma unroll
                                for (uint32_t j = 0; j < 32; ++j) r[j] = 0u;
                            }
                            if (f32) {
                                put_f32(r);
                            } else {
                                put_16(r, part);
                            }
                        }
                        send(at);
                    }
                }
            }
            if (!LONG && summed) release_piece();
        }
        if (WEIGHT && lane == 0) tma_store_wait_read<0>();
        __syncwarp();
    }

    // ---------------------------------------------------------------------- teardown
    tcgen05_fence_before_sync();
    __syncthreads();
    if (*abort_flag != 0) {
        // give copies still in flight time to land before shared memory is released
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) {
        }
        if (threadIdx.x == 0) atomicExch(p.error_word, 1u);
        __syncthreads();
    }
    if (CG == 2) cluster_sync_all();
    if (warp == 1) {
        tcgen05_fence_after_sync();
        tmem_dealloc<CG>(tmem_base, T::kTmemCols);
    }
}

}  // namespace b200
