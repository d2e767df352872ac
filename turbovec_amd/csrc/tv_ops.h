// The operators beside the search: 8-bit rows, their products, re-scoring of candidates, drawing from scores.
// What the entry points (tv_ops.hip) hand to the kernels; every size has been checked there.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <tuple>

#include "tv_device.h"

namespace tv {

constexpr int kScaleBlock = 128;      // coordinates that share a scale
enum { kF32 = 0, kF16 = 1, kBF16 = 2 };
enum { kScaleE8M0 = 0, kScaleF32 = 1 };

// Rows in 8 bits: e4m3 codes and a scale for each block of 128 coordinates of `1 << group_shift` rows.  Strides in elements.
struct Rows8 {
    const uint8_t *codes;
    const void *scales;
    size_t stride, scale_stride;
    uint32_t rows;
    int group_shift;                  // 0 or 7
};

struct QuantizeArgs {
    const void *x;
    uint8_t *codes;
    void *scales;
    size_t x_stride, code_stride, scale_stride;
    uint32_t rows, dim;
};
hipError_t launch_fp8_quantize(const QuantizeArgs &a, int x_type, int scale_type, int group_shift, hipStream_t s);

struct MatmulArgs {
    Rows8 a, b;                       // a: group_shift 0
    uint32_t dim;
    void *out;
    size_t out_stride;
    int out_type;
};
hipError_t launch_fp8_matmul(const MatmulArgs &a, int scale_type, hipStream_t s);

struct RescoreArgs {
    const void *queries;
    const int64_t *slots;
    size_t q_stride, slot_stride;
    Rows8 rows;
    uint32_t dim, nq, m, k;
    float *out_scores;
    int64_t *out_slots;
    uint64_t *keys;                   // workspace: nq * m sort keys, or none (rescore_workspace)
};
constexpr uint32_t kMaxRescore = 16384;      // candidates of a query: their sort keys fit a workgroup's LDS
size_t rescore_workspace(size_t nq, size_t m, size_t dim);
hipError_t launch_fp8_rescore(const RescoreArgs &a, int q_type, int scale_type, hipStream_t s);

struct SampleArgs {
    const void *scores;
    const uint64_t *mask;             // null: every slot is allowed
    const float *u, *temperature, *top_p, *min_p;      // a value a row; the last three may be null
    const int32_t *top_k;             // may be null
    size_t stride, mask_stride;       // of a row; mask words: 0 where the rows share them
    uint32_t rows, n;
    int64_t *out_slots;
    float *out_probs;
    uint8_t *ws;
};
size_t sample_workspace(size_t rows, size_t n);
hipError_t launch_sample(const SampleArgs &a, int score_type, hipStream_t s);

// For tv_last_error (tv_api.hip).
int op_refused(const char *why);      // TV_ERR_BAD_ARGUMENT
int op_failed(hipError_t e, const char *what);

// Dynamic LDS beyond 64 KiB has to be asked for, on every device a kernel runs on.
inline hipError_t allow_lds(const void *kernel, size_t bytes) {
    return bytes <= 65536 ? hipSuccess : hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
}
// A launch that reports its own error, and none that an earlier call of the process left behind.
template <typename... P, typename... A>
hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 threads, size_t lds, hipStream_t s, const A &...a) {
    std::tuple<P...> held{P(a)...};
    return std::apply([&](auto &...x) {
        void *at[] = {static_cast<void *>(&x)...};
        return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, threads, at, lds, s);
    }, held);
}

typedef _Float16 f16;
typedef __bf16 bf16;

typedef int v4i_any __attribute__((ext_vector_type(4), aligned(1)));

// 16 bytes moved down by so many, zeros from above; 16 and more leave nothing.
__device__ __forceinline__ v4i bytes_down(v4i v, uint32_t bytes) {
    uint64_t lo = uint64_t(uint32_t(v[0])) | uint64_t(uint32_t(v[1])) << 32, hi = uint64_t(uint32_t(v[2])) | uint64_t(uint32_t(v[3])) << 32;
    if (bytes & 8u) { lo = hi; hi = 0; }
    const uint32_t bits = (bytes & 7u) * 8u;
    lo = lo >> bits | (hi << 1) << (63u - bits);
    hi >>= bits;
    if (bytes >= 16u) lo = hi = 0;
    return v4i{int(uint32_t(lo)), int(uint32_t(lo >> 32)), int(uint32_t(hi)), int(uint32_t(hi >> 32))};
}
// 16 codes of a row from k on, those past `dim` zero, without touching what lies behind the row: a run that the row ends in is
// the end of the row's last 16 codes.
__device__ __forceinline__ v4i codes16(const uint8_t *row, uint32_t k, uint32_t dim) {
    if (dim >= 16u) {
        const uint32_t at = min(k, dim - 16u);
        return bytes_down(*reinterpret_cast<const v4i_any *>(row + at), k - at);
    }
    v4i v{0, 0, 0, 0};
    for (uint32_t i = 0; k + i < dim; ++i) {
        const v4i x = bytes_down(v4i{0, 0, 0, int(uint32_t(row[k + i]) << 24)}, 15u - i);
        v |= x;
    }
    return v;
}


}  // namespace tv
