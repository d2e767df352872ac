// The root-mean-square norm of rows, a residual added before it, made into rows of 8 or 4 bits in the same pass.
#include "tv_rows.h"

namespace tv {

// h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight; then the scales and codes of y's blocks.  A thread holds runs of eight
// neighbouring coordinates in registers from the first reading to the codes; sixteen lanes hold a block of 8-bit rows, four one of 4-bit rows.
__device__ __forceinline__ float row16_max(float v) {
    v = max_moved<0xb1>(v);
    v = max_moved<0x4e>(v);
    v = max_moved<0x141>(v);
    return max_moved<0x140>(v);
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) v += __shfl_xor(v, i);
    return v;
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8], int left) {
    typedef T T8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (left >= 8) {
        T8 x;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = T(v[i]);
        *reinterpret_cast<T8 *>(p) = x;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = T(v[i]);
}
__device__ __forceinline__ void load_weight(float (&w)[8], const void *p, int type, uint32_t at, int left) {
    if (type == kF32) load8<float>(w, static_cast<const float *>(p) + at, left);
    else if (type == kF16) load8<f16>(w, static_cast<const f16 *>(p) + at, left);
    else load8<bf16>(w, static_cast<const bf16 *>(p) + at, left);
}

enum { kToFp8E8 = 0, kToFp8F32 = 1, kToFp4 = 2 };

// A workgroup to a row, a thread to RUNS runs.
constexpr int kNormThreads = 256;
template <typename T, int TO, int RUNS>
__global__ __launch_bounds__(kNormThreads) void k_rms_norm(NormArgs a) {
    __shared__ float part[kNormThreads / 64];
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *const x = static_cast<const T *>(a.x) + size_t(row) * a.x_stride, *const r = static_cast<const T *>(a.residual) + size_t(row) * a.residual_stride;
        T *const sum = static_cast<T *>(a.sum) + size_t(row) * a.sum_stride;
        float h[RUNS][8], squares = 0.0f;
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = (uint32_t(i) * kNormThreads + threadIdx.x) * 8u;
            const int left = int(a.dim) - int(at);
            load8<T>(h[i], x + at, left);
            if (a.residual != nullptr) {
                float more[8];
                load8<T>(more, r + at, left);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] += more[j];
            }
            if (a.sum != nullptr) store8<T>(sum + at, h[i], left);
#pragma unroll
            for (int j = 0; j < 8; ++j) squares = fmaf(h[i][j], h[i][j], squares);
        }
        squares = wave_sum(squares);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = squares;
        __syncthreads();
        squares = part[0] + part[1] + part[2] + part[3];
        __syncthreads();
        const float mean = squares / float(a.dim) + a.eps;
        const float inverse = mean < __int_as_float(0x7f800000) ? 1.0f / sqrtf(mean) : __int_as_float(0x7fc00000);
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = (uint32_t(i) * kNormThreads + threadIdx.x) * 8u;
            const int left = int(a.dim) - int(at);
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = j < left ? h[i][j] * inverse : 0.0f;
            if (a.weight != nullptr) {
                float w[8];
                load_weight(w, a.weight, a.weight_type, at, left);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = j < left ? y[j] * w[j] : 0.0f;
            }
            uint32_t stored;
            if (TO == kToFp4) {
                const uint32_t most = quad_max(magnitude8(y));
                const uint32_t c = codes4_of(y, scale4_of(most, stored), most);
                if (left <= 0) continue;
                store_nibbles(a.codes + size_t(row) * a.code_stride + at / 2u, c, left);
                if ((threadIdx.x & 3) == 0) static_cast<uint8_t *>(a.scales)[size_t(row) * a.scale_stride + at / kScaleBlock4] = uint8_t(stored);
            } else {
                float most = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) most = fmaxf(most, finite_abs(y[j]));
                const float s = scale_of<TO == kToFp8E8>(row16_max(most), stored);
                if (left <= 0) continue;
                const float lo[4] = {y[0], y[1], y[2], y[3]}, hi[4] = {y[4], y[5], y[6], y[7]};
                uint8_t *const to = a.codes + size_t(row) * a.code_stride + at;
                const uint32_t c0 = codes_of<TO == kToFp8E8>(lo, s), c1 = codes_of<TO == kToFp8E8>(hi, s);
                store4(to, c0, left);
                store4(to + 4, c1, left - 4);
                if ((threadIdx.x & 15) == 0) store_scale<TO == kToFp8E8>(a.scales, size_t(row) * a.scale_stride + at / kScaleBlock, stored);
            }
        }
    }
}
template <typename T, int TO>
static hipError_t norm(const NormArgs &a, hipStream_t s) {
    const uint32_t grid = uint32_t(a.rows < kMostGroups ? a.rows : kMostGroups), runs = (a.dim + 8 * kNormThreads - 1) / (8 * kNormThreads);
    if (runs <= 1) return launch(k_rms_norm<T, TO, 1>, grid, kNormThreads, 0, s, a);
    if (runs <= 2) return launch(k_rms_norm<T, TO, 2>, grid, kNormThreads, 0, s, a);
    return runs <= 4 ? launch(k_rms_norm<T, TO, 4>, grid, kNormThreads, 0, s, a) : launch(k_rms_norm<T, TO, 8>, grid, kNormThreads, 0, s, a);
}
template <typename T>
static hipError_t norm_as(const NormArgs &a, int row_kind, int scale_type, hipStream_t s) {
    if (row_kind == kRowsFp4) return norm<T, kToFp4>(a, s);
    return scale_type == kScaleE8M0 ? norm<T, kToFp8E8>(a, s) : norm<T, kToFp8F32>(a, s);
}
hipError_t launch_rms_norm(const NormArgs &a, int x_type, int row_kind, int scale_type, hipStream_t s) {
    if (x_type == kF32) return norm_as<float>(a, row_kind, scale_type, s);
    return x_type == kF16 ? norm_as<f16>(a, row_kind, scale_type, s) : norm_as<bf16>(a, row_kind, scale_type, s);
}

}  // namespace tv
