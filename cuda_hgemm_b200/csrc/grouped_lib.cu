// Host side of the feed-forward products (include/b200_hgemm.h): argument checks, the choice of tile and the
// launches of the grouped kernel in its three forms and of the pass over an output's gradient.
#include <math.h>
#include <string.h>

#include "../../include/b200_hgemm.h"
#include "gemm_kernel_grouped.cuh"
#include "lib_state.h"
#include "slope_kernel.cuh"

#include <initializer_list>

namespace b200 {

static bool known_act(int32_t act) {
    return act >= B200_ACT_NONE && act <= B200_ACT_SILU;
}

// Types a caller may name: 16-bit inputs, and outputs of that type or FP32.
static bool known_types(int32_t in_type, int32_t out_type) {
    return (in_type == B200_C_F16 || in_type == B200_C_BF16) && (out_type == in_type || out_type == B200_C_F32);
}

static bool misaligned(std::initializer_list<const void *> ptrs) {
    uintptr_t bits = 0;
    for (const void *p : ptrs) bits |= reinterpret_cast<uintptr_t>(p);
    return (bits & 15u) != 0;
}

// All kernels here are launched plainly, each when the one before it in the stream has ended, and so are the short-A
// kernels of a linear layer (skinny_start in hgemm_lib.cu). Started early (programmatic dependent launch, 1 to 2 us less between
// two of them) and waiting beside one another, the small CTAs of the pass over dC and the whole-SM CTAs and pairs of
// the products have been seen to stand still for good; the cause is not known.
static void pair_attribute(cudaLaunchConfig_t *cfg, cudaLaunchAttribute *attr) {
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = 2;
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cfg->attrs = attr;
    cfg->numAttrs = 1;
}

// Whether a result's sum of `length` products is added up from pieces, and, if so, how long those are.
static bool sum_in_pieces(GroupedParams &p, size_t length) {
    const int32_t type = static_cast<int32_t>(p.out_type);
    const uint32_t blocks = sum_piece(type) / 64u;  // a power of two
    while ((1u << p.piece_shift) < blocks) ++p.piece_shift;
    return length > longest_sum(type);
}

// `most_tiles`: an upper bound of the tiles there can be; the grid is persistent and never larger than what
// is resident at once.
template <int FORM, int CG, int QT, int STAGES, int KPS, bool LONG = false>
static int launch_grouped(DeviceState &st, int slot, const GroupedParams &p, uint64_t most_tiles, cudaStream_t stream) {
    using T = GroupedTraits<FORM, CG, QT, STAGES, KPS, LONG>;
    auto kern = hgemm_grouped_kernel<FORM, CG, QT, STAGES, KPS, LONG>;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr;
    cfg.blockDim = dim3(kGroupedThreads, 1, 1);
    cfg.dynamicSmemBytes = T::kSmemBytes;
    cfg.stream = stream;
    if (CG == 2) pair_attribute(&cfg, &attr);
    uint32_t resident = static_cast<uint32_t>(st.sm_count);
    {
        std::lock_guard<std::mutex> lock(st.mu);
        if (!st.attr_set[slot]) {
            if (!cuda_ok(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmemBytes), "cudaFuncSetAttribute")) {
                return B200_HGEMM_ERR_CUDA;
            }
            st.attr_set[slot] = true;
        }
        if (CG == 2) {
            if (st.max_clusters[slot] == 0) {
                int n = 0;
                cfg.gridDim = dim3(2u * (st.sm_count / 2), 1, 1);
                if (!cuda_ok(cudaOccupancyMaxActiveClusters(&n, kern, &cfg), "cudaOccupancyMaxActiveClusters") || n < 1) {
                    return B200_HGEMM_ERR_CUDA;
                }
                st.max_clusters[slot] = n;
            }
            resident = static_cast<uint32_t>(st.max_clusters[slot]);
        }
    }
    const uint32_t workers = most_tiles < resident ? static_cast<uint32_t>(most_tiles) : resident;
    cfg.gridDim = dim3(workers * CG, 1, 1);
    if (!cuda_ok(cudaLaunchKernelEx(&cfg, kern, p), "cudaLaunchKernelEx")) return B200_HGEMM_ERR_CUDA;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return B200_HGEMM_OK;
}

// The kernels of the forward and input form: CTAs per tile, most rows of a tile, k-blocks per stage.
enum RowsKernel : uint32_t { kRowsPair256, kRowsPair128, kRowsSingle128, kRowsSingle32 };
struct RowsKernelShape {
    int cg;
    uint32_t q_cap;
    int kps;
};
constexpr RowsKernelShape rows_kernels[4] = {{2, 256, 1}, {2, 128, 2}, {1, 128, 2}, {1, 32, 2}};

struct RowsPlan {
    uint32_t kernel;
    uint32_t q_max;
};

// The kernel and the most rows per block that should take the least time: waves of tiles times the time of one.
// Measured with one to 144 CTAs at work (K = 2048 against 8192), a k-block of a tile takes the longest of
//   * what the issuing threads need: 0.14 us for single CTAs, 0.10 for pairs and for blocks of 32 rows,
//   * its MMAs: 1.1 ns per row of the block (1.3 with the whole GPU at work), 128 columns of the result per CTA,
//   * its operands' way out of L2: 20.5 TB/s for all SMs together;
// a kernel costs 4 us besides (5.5 where two CTAs have to meet), and 10 ns per row of a block for the last
// epilogue. Group sizes are not known here: the estimate spreads the rows evenly over the groups, and with 32 rows or fewer
// on average takes the blocks of 32. One hot expert then reads its weights once per 32 rows: 64 experts of 1024 x 2048, 2048 rows in
// BF16, take 47 us at 32 rows each and 57 with 1500 rows in one.
static RowsPlan choose_rows_plan(const DeviceState &st, size_t rows, size_t p_dim, size_t k_dim, size_t groups) {
    const uint64_t live = groups < rows ? groups : rows;  // groups that can hold any rows
    const uint64_t average = (rows + live - 1) / live;
    RowsPlan best{kRowsSingle32, 32};
    if (average <= 32) return best;
    double best_us = 1e30;
    for (uint32_t kernel = kRowsPair256; kernel <= kRowsSingle32; ++kernel) {
        const RowsKernelShape &shape = rows_kernels[kernel];
        const double slots = st.sm_count / shape.cg;
        for (uint32_t q_max = shape.q_cap; q_max >= 32u; q_max -= 32u) {
            if (kernel == kRowsPair256 && q_max < 160u) break;  // the other pair kernel's
            const uint64_t blocks = (average + q_max - 1) / q_max;
            const double q = static_cast<double>((average + blocks - 1) / blocks);
            const double tiles = static_cast<double>(blocks * live) * ceil_div_u32(p_dim, 128u * shape.cg);
            const double active = tiles < slots ? tiles : slots;
            double per_block = active * shape.cg * (16384.0 + q / shape.cg * 128.0) / 20.5e6;
            // (lower blocks read the weights more often: 6 percent more at none, measured 2 at 205 rows instead of 256)
            const double mma = (active * shape.cg > 100.0 ? 0.0013 : 0.0011) * q * (1.06 - 0.06 * q / 256.0);
            const double issue = kernel == kRowsSingle128 ? 0.14 : 0.10;
            if (per_block < mma) per_block = mma;
            if (per_block < issue) per_block = issue;
            const double us = ceil(tiles / slots) * per_block * ceil_div_u32(k_dim, 64) + (shape.cg == 2 ? 5.5 : 4.0) + 0.010 * q;
            if (us < best_us * 0.999) {
                best_us = us;
                best = RowsPlan{kernel, q_max};
            }
        }
    }
    return best;
}

// Forward and input form. X: the rows' operand [rows x k_dim]; W: groups matrices [w_rows x w_cols], stride_w apart.
template <int FORM>
static int run_rows(DeviceState &st, const void *X, const void *W, size_t rows, size_t p_dim, size_t k_dim, size_t w_rows,
                    size_t w_cols, size_t groups, size_t stride_w, GroupedParams &p, cudaStream_t stream) {
    constexpr int kSlots = FORM == kFormForward ? 96 : 104;
    p.error_word = st.error_word;
    p.rows = static_cast<uint32_t>(rows);
    p.groups = static_cast<uint32_t>(groups);
    p.p_dim = static_cast<uint32_t>(p_dim);
    const RowsPlan plan = choose_rows_plan(st, rows, p_dim, k_dim, groups);
    const int cg = rows_kernels[plan.kernel].cg, kps = rows_kernels[plan.kernel].kps;
    p.q_max = plan.q_max;
    p.p_blocks = ceil_div_u32(p_dim, 128u * cg);
    p.k_blocks = ceil_div_u32(k_dim, 64u * kps);
    // an upper bound: every group may end in a block that is not full, and tiles may be as narrow as 64
    const uint64_t tiles = (rows / p.q_max + (groups < rows ? groups : rows)) *
                           (plan.kernel == kRowsSingle32 ? ceil_div_u32(p_dim, 64) : p.p_blocks);
    if (tiles > 0x7fffffffull) return B200_HGEMM_ERR_TOO_LARGE;
    int rc;
    const uint32_t box_rows = FORM == kFormForward ? 128u : 64u;
    if ((rc = get_tensor_map(st, W, w_rows, w_cols, box_rows, 64, &p.tm_p, true, groups, stride_w)) != B200_HGEMM_OK) return rc;
    if (FORM == kFormForward && plan.kernel == kRowsSingle32) {
        for (uint32_t i = 0; i < 4; ++i) {
            if ((rc = get_tensor_map(st, W, w_rows, w_cols, 64u + 16u * i, 64, &p.tm_narrow[i], true, groups, stride_w)) != B200_HGEMM_OK) return rc;
        }
    }
    for (uint32_t i = 0; i < p.q_max / (16u * cg); ++i) {
        if ((rc = get_tensor_map(st, X, rows, k_dim, 16u * (i + 1u), 64, &p.tm_q[i])) != B200_HGEMM_OK) return rc;
    }
    const int slot = kSlots + static_cast<int>(plan.kernel);
    if (sum_in_pieces(p, k_dim)) {
        switch (plan.kernel) {
            case kRowsPair256: return launch_grouped<FORM, 2, 256, 6, 1, true>(st, slot + 4, p, tiles, stream);
            case kRowsPair128: return launch_grouped<FORM, 2, 128, 4, 2, true>(st, slot + 4, p, tiles, stream);
            case kRowsSingle128: return launch_grouped<FORM, 1, 128, 3, 2, true>(st, slot + 4, p, tiles, stream);
            default: return launch_grouped<FORM, 1, 32, 5, 2, true>(st, slot + 4, p, tiles, stream);
        }
    }
    switch (plan.kernel) {
        case kRowsPair256: return launch_grouped<FORM, 2, 256, 6, 1>(st, slot, p, tiles, stream);
        case kRowsPair128: return launch_grouped<FORM, 2, 128, 4, 2>(st, slot, p, tiles, stream);
        case kRowsSingle128: return launch_grouped<FORM, 1, 128, 3, 2>(st, slot, p, tiles, stream);
        default: return launch_grouped<FORM, 1, 32, 5, 2>(st, slot, p, tiles, stream);
    }
}

// An operand of the weight form, 64 rows of 64 columns to a box. Where the width is a multiple of 64 the columns are
// mapped in blocks of 64 and a copy takes two of them; elsewhere such a block would reach into the next row, and
// past the end of the last one.
static int columns_map(DeviceState &st, const void *ptr, size_t rows, size_t width, CUtensorMap *map, uint32_t *wide) {
    *wide = width % 64 == 0 ? 1u : 0u;
    if (*wide) return get_tensor_map(st, ptr, rows, 64, 64, 64, map, true, width / 64, 64, 2, width, 2);
    return get_tensor_map(st, ptr, rows, width, 64, 64, map);
}

// Weight form: pairs on 256 x 256 or single CTAs on 128 x 128, by the estimate of choose_rows_plan (single CTAs need 0.16 us
// per block of 64 rows, pairs 0.28; a tile costs 1.0 and 2.8 us besides, which decides for groups of few rows: 32 groups
// of 128 rows, 1024 x 2048 in FP16, 38 us on single CTAs and 48 on pairs).
static int weight_cg(const DeviceState &st, size_t M, size_t N, size_t K, size_t G) {
    const double blocks = ceil_div_u32((M + G - 1) / G, 64);
    double us[2];
    for (int cg = 1; cg <= 2; ++cg) {
        const double slots = st.sm_count / cg;
        const double tiles = static_cast<double>(G) * ceil_div_u32(N, 128u * cg) * ceil_div_u32(K, 128u * cg);
        const double active = tiles < slots ? tiles : slots;
        double per_block = active * cg * 32768.0 / 20.5e6;
        const double least = cg == 1 ? 0.16 : active > 50.0 ? 0.33 : 0.28;
        if (per_block < least) per_block = least;
        us[cg - 1] = ceil(tiles / slots) * (per_block * blocks + (cg == 1 ? 1.0 : 2.8)) + (cg == 1 ? 4.0 : 5.5);
    }
    return us[1] < us[0] ? 2 : 1;
}

// Slices a dense layer's long sum over the rows is cut into where its gradient has too few tiles for the GPU: as many as
// give every SM a tile, of at least 512 rows each. They lie in FP32 in the workspace (at most 148 tiles of 128 x 128: 9.7 MB) and slice_sum_kernel
// adds them in order. 8192 rows of 256 x 256: 31 us in one piece, 11 in sixteen; of 1024 x
// 1024: 33 us, 26 in two.
static uint32_t weight_slices(size_t M, size_t N, size_t K, size_t G, bool ragged) {
    constexpr uint64_t kSms = 148;  // (of a B200; the workspace size must not depend on the current device)
    if (ragged || G != 1 || M < 1024) return 1;
    const uint64_t tiles = static_cast<uint64_t>(ceil_div_u32(N, 128)) * ceil_div_u32(K, 128);
    const uint64_t slices = kSms / tiles < M / 512 ? kSms / tiles : M / 512;
    // the sum of the slices is a kernel of its own, about 4 us: 1600 rows' worth of one tile's sum
    return slices < 2 || M - M / slices < 1600 ? 1u : static_cast<uint32_t>(slices);
}

static size_t align256(size_t v) {
    return (v + 255) / 256 * 256;
}

static size_t slices_bytes(size_t M, size_t N, size_t K, size_t G, bool ragged, const b200_linear_grads &g) {
    const uint32_t slices = g.dB ? weight_slices(M, N, K, G, ragged) : 1u;
    return slices > 1 ? align256(slices * N * K * sizeof(float)) : 0;
}

// Weight form: dB_g = dZ_g^T A_g.
static int run_weight(DeviceState &st, const void *dZ, const void *A, void *dB, const int32_t *offsets, size_t M, size_t N, size_t K,
                      size_t G, const b200_linear_grads &g, void *parts, cudaStream_t stream) {
    GroupedParams p;
    memset(&p, 0, sizeof(p));
    p.out = dB;
    p.offsets = offsets;
    p.error_word = st.error_word;
    p.rows = static_cast<uint32_t>(M);
    p.p_dim = static_cast<uint32_t>(N);
    p.q_dim = static_cast<uint32_t>(K);
    p.in_bf16 = g.in_type == B200_C_BF16 ? 1u : 0u;
    p.out_type = static_cast<uint32_t>(g.db_type);
    p.accumulate = g.accumulate ? 1u : 0u;
    size_t longest = M;  // rows of the longest sum there can be
    const uint32_t slices = weight_slices(M, N, K, G, offsets != nullptr);
    if (slices > 1) {
        p.out = parts;
        p.out_type = B200_C_F32;
        p.accumulate = 0;
        p.slice_rows = static_cast<uint32_t>((M + slices - 1) / slices);
        G = ceil_div_u32(M, p.slice_rows);  // (rounding up may leave the last ones without rows)
        longest = p.slice_rows;
    }
    p.groups = static_cast<uint32_t>(G);
    const int cg = slices > 1 ? 1 : weight_cg(st, M, N, K, G);
    p.p_blocks = ceil_div_u32(N, 128u * cg);
    p.q_blocks = ceil_div_u32(K, 128u * cg);
    const uint64_t tiles = static_cast<uint64_t>(G) * p.p_blocks * p.q_blocks;
    if (tiles > 0x7fffffffull) return B200_HGEMM_ERR_TOO_LARGE;
    int rc;
    if ((rc = columns_map(st, dZ, M, N, &p.tm_p, &p.p_wide)) != B200_HGEMM_OK) return rc;
    if ((rc = columns_map(st, A, M, K, &p.tm_q[0], &p.q_wide)) != B200_HGEMM_OK) return rc;
    const bool f32 = p.out_type == B200_C_F32;
    const bool in_pieces = sum_in_pieces(p, longest);
    if ((rc = get_tensor_map(st, p.out, N, K, 32, f32 ? 32 : 64, &p.tm_out, true, G, N * K, f32 ? 4 : 2)) != B200_HGEMM_OK) return rc;
    if (slices > 1) {
        rc = in_pieces ? launch_grouped<kFormWeight, 1, 128, 5, 1, true>(st, 113, p, tiles, stream)
                       : launch_grouped<kFormWeight, 1, 128, 5, 1>(st, 115, p, tiles, stream);
        if (rc != B200_HGEMM_OK) return rc;
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof(cfg));
        const size_t count4 = N * K / 4;
        cfg.gridDim = dim3(ceil_div_u32(count4, 256), 1, 1);
        cfg.blockDim = dim3(256, 1, 1);
        cfg.stream = stream;
        if (!cuda_ok(cudaLaunchKernelEx(&cfg, slice_sum_kernel, static_cast<const float4 *>(parts), dB, count4, p.groups,
                                        static_cast<uint32_t>(g.db_type), g.accumulate ? 1u : 0u),
                     "cudaLaunchKernelEx")) {
            return B200_HGEMM_ERR_CUDA;
        }
        g_launches.fetch_add(1, std::memory_order_relaxed);
        return B200_HGEMM_OK;
    }
    if (in_pieces) {
        if (cg == 2) return launch_grouped<kFormWeight, 2, 256, 6, 1, true>(st, 112, p, tiles, stream);
        return launch_grouped<kFormWeight, 1, 128, 5, 1, true>(st, 113, p, tiles, stream);
    }
    if (cg == 2) return launch_grouped<kFormWeight, 2, 256, 6, 1>(st, 114, p, tiles, stream);
    return launch_grouped<kFormWeight, 1, 128, 5, 1>(st, 115, p, tiles, stream);
}

// ---- the pass over dC -----------------------------------------------------------------------
// Slices a group's rows are cut into: about 128 rows each where the groups are even, four times as many where there
// are several (one may hold much more than its share), and enough blocks to fill the GPU when there are few rows.
// One slice, and no second kernel, for up to 64 rows: eight per warp.
static uint32_t slope_slices(size_t M, size_t N, size_t G) {
    if (M <= 64) return 1u;
    const uint64_t spread = G < 4 ? G : 4;
    uint64_t slices = (M * spread + 128 * G - 1) / (128 * G);
    const uint64_t strips = ceil_div_u32(N, kSlopeColumns);
    const uint64_t fill = 296 / (strips * G) + 1, most = (M + 15) / 16;
    if (slices < fill) slices = fill;
    if (slices > most) slices = most;
    if (slices > 4096) slices = 4096;
    return slices < 1 ? 1u : static_cast<uint32_t>(slices);
}

// Whether the products read a dZ other than the caller's dC.
static bool needs_dz(const b200_linear_grads &g) {
    return g.act != B200_ACT_NONE || g.c_type != g.in_type;
}

static size_t dz_bytes(size_t M, size_t N, const b200_linear_grads &g) {
    return (!g.dZ && needs_dz(g) && (g.dA || g.dB)) ? align256(M * N * 2) : 0;
}

static size_t sums_bytes(size_t M, size_t N, size_t G, const b200_linear_grads &g) {
    const uint32_t slices = slope_slices(M, N, G);
    return g.dbias && slices > 1 ? align256(static_cast<size_t>(slices) * G * N * sizeof(float)) : 0;
}

template <bool F32>
static cudaError_t launch_slope_kernel(const cudaLaunchConfig_t *cfg, const SlopeParams &p, uint32_t act) {
    switch (act) {
        case kActRelu: return cudaLaunchKernelEx(cfg, slope_kernel<kActRelu, F32>, p);
        case kActGelu: return cudaLaunchKernelEx(cfg, slope_kernel<kActGelu, F32>, p);
        case kActGeluTanh: return cudaLaunchKernelEx(cfg, slope_kernel<kActGeluTanh, F32>, p);
        case kActSilu: return cudaLaunchKernelEx(cfg, slope_kernel<kActSilu, F32>, p);
        default: return cudaLaunchKernelEx(cfg, slope_kernel<kActNone, F32>, p);
    }
}

static int launch_slope(const SlopeParams &p, uint32_t act, dim3 grid, cudaStream_t stream) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kSlopeThreads, 1, 1);
    cfg.stream = stream;
    const cudaError_t e = p.c_type == B200_C_F32 ? launch_slope_kernel<true>(&cfg, p, act) : launch_slope_kernel<false>(&cfg, p, act);
    if (!cuda_ok(e, "cudaLaunchKernelEx")) return B200_HGEMM_ERR_CUDA;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return B200_HGEMM_OK;
}

static int run_slope(const b200_linear_grads &g, void *dz, float *sums, const int32_t *offsets, size_t M, size_t N, size_t G,
                     cudaStream_t stream) {
    SlopeParams p;
    memset(&p, 0, sizeof(p));
    p.dc = g.dC;
    p.pre = g.pre;
    p.dz = dz;
    p.offsets = offsets;
    p.rows = static_cast<uint32_t>(M);
    p.n = static_cast<uint32_t>(N);
    p.groups = static_cast<uint32_t>(G);
    p.slices = slope_slices(M, N, G);
    p.c_type = static_cast<uint32_t>(g.c_type);
    p.dz_bf16 = g.in_type == B200_C_BF16 ? 1u : 0u;
    const bool one = p.slices == 1;
    p.sums = g.dbias ? (one ? g.dbias : sums) : nullptr;
    p.accumulate = one && g.accumulate ? 1u : 0u;
    const dim3 grid(ceil_div_u32(N, kSlopeColumns), p.slices, static_cast<unsigned>(G));
    int rc = launch_slope(p, static_cast<uint32_t>(g.act), grid, stream);
    if (rc != B200_HGEMM_OK || !g.dbias || one) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    const size_t count = G * N;
    cfg.gridDim = dim3(ceil_div_u32(count, 256), 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = stream;
    if (!cuda_ok(cudaLaunchKernelEx(&cfg, bias_sum_kernel, static_cast<const float *>(sums), g.dbias, count, p.slices,
                                    g.accumulate ? 1u : 0u),
                 "cudaLaunchKernelEx")) {
        return B200_HGEMM_ERR_CUDA;
    }
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return B200_HGEMM_OK;
}

static int check_sizes(size_t M, size_t N, size_t K) {
    if (N == 0 || K == 0) return B200_HGEMM_ERR_INVALID_ARG;
    if (M > 0x7fffff00ull || N > 0x7fffff00ull || K > 0x7fffff00ull) return B200_HGEMM_ERR_UNSUPPORTED;
    return B200_HGEMM_OK;
}

static int check_groups(const int32_t *offsets, size_t N, size_t K, size_t G, size_t stride_b) {
    if (!offsets || G == 0) return B200_HGEMM_ERR_INVALID_ARG;
    if (G > kGroupedMaxGroups) return B200_HGEMM_ERR_TOO_LARGE;
    if ((reinterpret_cast<uintptr_t>(offsets) & 3u) != 0 || stride_b % 8 != 0) return B200_HGEMM_ERR_MISALIGNED;
    if (G > 1 && stride_b < N * K) return B200_HGEMM_ERR_INVALID_ARG;
    return B200_HGEMM_OK;
}

static GroupedParams forward_params(void *C, const int32_t *offsets, const b200_linear_args &args) {
    GroupedParams p;
    memset(&p, 0, sizeof(p));
    p.out = C;
    p.pre = args.pre;
    p.bias = args.bias;
    p.residual = args.residual;
    p.offsets = offsets;
    p.in_bf16 = args.in_type == B200_C_BF16 ? 1u : 0u;
    p.out_type = static_cast<uint32_t>(args.c_type);
    p.act = static_cast<uint32_t>(args.act);
    return p;
}

int run_linear_rows(DeviceState &st, const void *A, const void *B, void *C, size_t M, size_t N, size_t K, const b200_linear_args &args,
                    cudaStream_t stream) {
    GroupedParams p = forward_params(C, nullptr, args);
    return run_rows<kFormForward>(st, A, B, M, N, K, N, K, 1, N * K, p, stream);
}

static int grouped_forward(const void *A, const void *B, void *C, const int32_t *offsets, size_t M, size_t N, size_t K, size_t G,
                           size_t stride_b, const b200_linear_args *args, cudaStream_t stream) {
    if (!args || !B || (M > 0 && (!A || !C))) return B200_HGEMM_ERR_INVALID_ARG;
    int rc = check_sizes(M, N, K);
    if (rc != B200_HGEMM_OK) return rc;
    if ((rc = check_groups(offsets, N, K, G, stride_b)) != B200_HGEMM_OK) return rc;
    if (!known_act(args->act) || !known_types(args->in_type, args->c_type)) return B200_HGEMM_ERR_INVALID_ARG;
    if (args->residual || K % 8 != 0) return B200_HGEMM_ERR_UNSUPPORTED;
    if (misaligned({A, B, C, args->bias, args->pre})) return B200_HGEMM_ERR_MISALIGNED;
    if (M == 0) return B200_HGEMM_OK;
    DeviceState *st = nullptr;
    if ((rc = current_state(&st)) != B200_HGEMM_OK) return rc;
    if (!st->sm100) return B200_HGEMM_ERR_NO_SM100;
    GroupedParams p = forward_params(C, offsets, *args);
    return run_rows<kFormForward>(*st, A, B, M, N, K, N, K, G, G > 1 ? stride_b : N * K, p, stream);
}

// Both backward entry points; `offsets` is null for the dense one.
static int backward(const void *A, const void *B, const int32_t *offsets, size_t M, size_t N, size_t K, size_t G, size_t stride_b,
                    const b200_linear_grads *grads, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    if (!grads) return B200_HGEMM_ERR_INVALID_ARG;
    const b200_linear_grads &g = *grads;
    int rc = check_sizes(M, N, K);
    if (rc != B200_HGEMM_OK) return rc;
    if (!known_act(g.act) || !known_types(g.in_type, g.c_type)) return B200_HGEMM_ERR_INVALID_ARG;
    if (g.db_type != g.in_type && g.db_type != B200_C_F32) return B200_HGEMM_ERR_INVALID_ARG;
    if (M > 0 && (!g.dC || (g.act != B200_ACT_NONE && !g.pre))) return B200_HGEMM_ERR_INVALID_ARG;
    if (M > 0 && ((g.dA && !B) || (g.dB && !A))) return B200_HGEMM_ERR_INVALID_ARG;
    if (M > 0 && !g.dA && !g.dB && !g.dbias && !g.dZ) return B200_HGEMM_ERR_INVALID_ARG;
    if (N % 8 != 0 || K % 8 != 0) return B200_HGEMM_ERR_UNSUPPORTED;
    if (g.accumulate && g.dB && g.db_type != B200_C_F32) return B200_HGEMM_ERR_UNSUPPORTED;
    if (misaligned({A, B, g.dC, g.pre, g.dZ, g.dA, g.dB, g.dbias})) return B200_HGEMM_ERR_MISALIGNED;
    const size_t need_dz = dz_bytes(M, N, g), need_sums = sums_bytes(M, N, G, g);
    const size_t need_parts = slices_bytes(M, N, K, G, offsets != nullptr, g);
    if (need_dz + need_sums + need_parts > 0) {
        if (!workspace || workspace_bytes < need_dz + need_sums + need_parts) return B200_HGEMM_ERR_WORKSPACE;
        if (reinterpret_cast<uintptr_t>(workspace) & 255u) return B200_HGEMM_ERR_MISALIGNED;
    }
    DeviceState *st = nullptr;
    if ((rc = current_state(&st)) != B200_HGEMM_OK) return rc;
    if (!st->sm100) return B200_HGEMM_ERR_NO_SM100;
    if (M == 0) {
        // nothing was multiplied: the gradients of the weights are zeros
        if (g.accumulate) return B200_HGEMM_OK;
        const size_t db_bytes = G * N * K * (g.db_type == B200_C_F32 ? 4 : 2);
        if (g.dB && !cuda_ok(cudaMemsetAsync(g.dB, 0, db_bytes, stream), "cudaMemsetAsync")) return B200_HGEMM_ERR_CUDA;
        if (g.dbias && !cuda_ok(cudaMemsetAsync(g.dbias, 0, G * N * sizeof(float), stream), "cudaMemsetAsync")) return B200_HGEMM_ERR_CUDA;
        return B200_HGEMM_OK;
    }
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    void *dz = g.dZ ? g.dZ : (need_dz ? ws : nullptr);
    float *sums = reinterpret_cast<float *>(ws + need_dz);
    if (dz || g.dbias) {
        if ((rc = run_slope(g, dz, sums, offsets, M, N, G, stream)) != B200_HGEMM_OK) return rc;
    }
    const void *dz_read = needs_dz(g) ? dz : g.dC;
    if (g.dA) {
        GroupedParams p;
        memset(&p, 0, sizeof(p));
        p.out = g.dA;
        p.offsets = offsets;
        p.in_bf16 = g.in_type == B200_C_BF16 ? 1u : 0u;
        p.out_type = static_cast<uint32_t>(g.in_type);
        rc = run_rows<kFormInput>(*st, dz_read, B, M, K, N, N, K, G, G > 1 ? stride_b : N * K, p, stream);
        if (rc != B200_HGEMM_OK) return rc;
    }
    if (g.dB) return run_weight(*st, dz_read, A, g.dB, offsets, M, N, K, G, g, ws + need_dz + need_sums, stream);
    return B200_HGEMM_OK;
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_hgemm_grouped(const void *A, const void *B, void *C, const int32_t *offsets, size_t M, size_t N, size_t K, size_t G,
                       size_t stride_b, const b200_linear_args *args, b200_stream_t stream) {
    return grouped_forward(A, B, C, offsets, M, N, K, G, stride_b, args, reinterpret_cast<cudaStream_t>(stream));
}

int b200_hgemm_grouped_backward(const void *A, const void *B, const int32_t *offsets, size_t M, size_t N, size_t K, size_t G,
                                size_t stride_b, const b200_linear_grads *grads, void *workspace, size_t workspace_bytes,
                                b200_stream_t stream) {
    const int rc = N == 0 || K == 0 ? B200_HGEMM_ERR_INVALID_ARG : check_groups(offsets, N, K, G, stride_b);
    if (rc != B200_HGEMM_OK) return rc;
    return backward(A, B, offsets, M, N, K, G, stride_b, grads, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

int b200_hgemm_linear_backward(const void *A, const void *B, size_t M, size_t N, size_t K, const b200_linear_grads *grads,
                               void *workspace, size_t workspace_bytes, b200_stream_t stream) {
    return backward(A, B, nullptr, M, N, K, 1, N * K, grads, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

size_t b200_hgemm_backward_workspace_bytes(size_t M, size_t N, size_t K, size_t G, const b200_linear_grads *grads) {
    if (!grads || N == 0 || K == 0 || G == 0) return 0;
    // (G = 1 may be either form: the dense one's share is counted)
    return dz_bytes(M, N, *grads) + sums_bytes(M, N, G, *grads) + slices_bytes(M, N, K, G, false, *grads);
}

}  // extern "C"
