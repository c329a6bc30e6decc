// What the library's translation units share: per-device state, the tensor-map cache, launch accounting.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/b200_hgemm.h"

#include <atomic>
#include <mutex>
#include <vector>

namespace b200 {

constexpr int kMaxDevices = 64;

struct TensorMapKey {
    const void *ptr;
    uint64_t rows, cols;
    uint32_t box_rows, box_cols;
    bool swizzle;
    uint64_t batch, batch_stride;  // stacks of matrices: how many, and elements from one to the next (1, 0: a single matrix)
    uint32_t elem_bytes;           // 2: 16-bit elements of either kind (a copy does not tell them apart), 4: FP32
    uint64_t pitch;                // elements from row to row
    uint32_t box_batch;            // matrices a box spans
    bool operator==(const TensorMapKey &o) const {
        return ptr == o.ptr && rows == o.rows && cols == o.cols && box_rows == o.box_rows && box_cols == o.box_cols &&
               swizzle == o.swizzle && batch == o.batch && batch_stride == o.batch_stride && elem_bytes == o.elem_bytes &&
               pitch == o.pitch && box_batch == o.box_batch;
    }
};

struct TensorMapSlot {
    bool used = false;
    uint64_t last_use = 0;
    TensorMapKey key{};
    CUtensorMap map{};
};
constexpr size_t kTensorMapWays = 4, kTensorMapSets = 256;

struct DeviceState {
    std::mutex mu;
    bool probed = false;       // attributes known and the error word allocated
    bool attrs_known = false;  // sm100 / sm_count filled in (no allocation needed for that)
    bool sm100 = false;
    int sm_count = 0;
    uint32_t *error_word = nullptr;
    // stream-k workspace [64 KiB header | FP32 partial slots]: either one the caller handed over
    // (ws), or one per stream that the library allocates and grows itself, so that GEMMs running
    // on different streams at the same time never share partial-tile slots
    void *ws = nullptr;
    size_t ws_bytes = 0;
    struct StreamWorkspace {
        cudaStream_t stream;
        void *ptr;
        size_t bytes;
        uint64_t last_use;
    };
    std::vector<StreamWorkspace> owned_ws;
    uint64_t ws_clock = 0;
    // staging buffers of the host-pointer entry point
    void *host_a = nullptr, *host_b = nullptr, *host_c = nullptr;
    size_t host_a_bytes = 0, host_b_bytes = 0, host_c_bytes = 0;
    cudaStream_t host_stream[3] = {nullptr, nullptr, nullptr};  // upload, GEMMs, download
    cudaEvent_t host_event[2] = {nullptr, nullptr};
    bool attr_set[128] = {};    // slots from 96 on: the grouped kernels
    int max_clusters[128] = {};
    int ck_clusters[16][9] = {};  // short-A kernels that sum inside clusters: clusters of each size the device holds at once (-1: none)  // CTA pairs the device can keep resident at once, per pair kernel
    TensorMapSlot tm_cache[kTensorMapSets * kTensorMapWays];
    uint64_t tm_clock = 0;
};

extern std::atomic<uint64_t> g_launches;

// Logs a failing CUDA call when B200_HGEMM_DEBUG is set; true on success.
bool cuda_ok(cudaError_t e, const char *what);
// State of the current device, probed on first use (a status on failure).
int current_state(DeviceState **out);
// The tensor map of a row-major matrix (or stack of matrices) viewed through boxes, from the cache or encoded.
int get_tensor_map(DeviceState &st, const void *ptr, uint64_t rows, uint64_t cols, uint32_t box_rows, uint32_t box_cols,
                   CUtensorMap *out, bool swizzle = true, uint64_t batch = 1, uint64_t batch_stride = 0, uint32_t elem_bytes = 2,
                   uint64_t pitch = 0, uint32_t box_batch = 1);

// Longest sum a result may take from one accumulator of the tensor cores, and the pieces that longer ones are added up
// from (gemm_kernel_grouped.cuh says why). FP32: 512 and 512. A 16-bit result loses a fifth of the half step that its
// rounding costs anyway at the longest single sum, and a twentieth in pieces.
constexpr uint32_t kLongSumF32 = 512, kLongSumF16 = 16384, kLongSumBf16 = 131072;
inline uint32_t longest_sum(int32_t out_type) {
    return out_type == B200_C_F32 ? kLongSumF32 : out_type == B200_C_F16 ? kLongSumF16 : kLongSumBf16;
}
inline uint32_t sum_piece(int32_t out_type) {
    return out_type == B200_C_F32 ? kLongSumF32 : longest_sum(out_type) / 4;
}
// A linear layer on the grouped kernel, all rows one group (arguments checked by the caller).
int run_linear_rows(DeviceState &st, const void *A, const void *B, void *C, size_t M, size_t N, size_t K, const b200_linear_args &args,
                    cudaStream_t stream);

inline uint32_t ceil_div_u32(uint64_t a, uint64_t b) {
    return static_cast<uint32_t>((a + b - 1) / b);
}

}  // namespace b200
