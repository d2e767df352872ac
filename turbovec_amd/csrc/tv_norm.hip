// The root-mean-square norm of rows, a residual added before it, made into rows of 8 or 4 bits in the same pass.
#include "tv_rows.h"

namespace tv {

// h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight; then the scales and codes of y's blocks.  A lane holds runs of eight
// neighbouring coordinates in registers from the first reading to the codes; sixteen lanes hold a block of 8-bit rows, four one of 4-bit rows.
__device__ __forceinline__ float row16_max(float v) {
    v = max_moved<0xb1>(v);
    v = max_moved<0x4e>(v);
    v = max_moved<0x141>(v);
    return max_moved<0x140>(v);
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int i = LANES / 2; i > 0; i >>= 1) v += __shfl_xor(v, i);
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

// LANES lanes to a row, each with RUNS runs: sixteen to sixty-four, or all of a workgroup, whose sums then go through LDS.  Bound by memory: 16384 rows of 4096 bfloat16 with a
// residual take 88 us, 5.4 TB/s, a third of it written (a copy reaches 4.6 to 4.9).  As many lanes as a row fills, one run or two each: with 256 threads to every
// row 100000 rows of 512 take 155 us where these take 66, 100000 of 130 floats 117 and 21; with eight runs to a lane 4096 rows of 16384 take 156 and 110, 16384 of 4096 153 and 88.
template <typename T, int TO, int LANES, int RUNS, int THREADS>
__global__ __launch_bounds__(THREADS) void k_rms_norm(NormArgs a) {
    constexpr uint32_t kTogether = THREADS / LANES;
    constexpr bool kAll = LANES > 64;
    __shared__ float part[kAll ? THREADS / 64 : 1];
    const uint32_t lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    for (uint64_t first = uint64_t(blockIdx.x) * kTogether; first < a.rows; first += uint64_t(gridDim.x) * kTogether) {
        const bool there = first + sub < a.rows;
        const uint32_t row = there ? uint32_t(first) + sub : a.rows - 1;
        const T *const x = static_cast<const T *>(a.x) + size_t(row) * a.x_stride, *const r = static_cast<const T *>(a.residual) + size_t(row) * a.residual_stride;
        T *const sum = static_cast<T *>(a.sum) + size_t(row) * a.sum_stride;
        float h[RUNS][8], squares = 0.0f;
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = (uint32_t(i) * LANES + lane) * 8u;
            load8<T>(h[i], x + at, there ? int(a.dim) - int(at) : 0);
        }
        if (a.residual != nullptr) {
            float more[RUNS][8];
#pragma unroll
            for (int i = 0; i < RUNS; ++i) {
                const uint32_t at = (uint32_t(i) * LANES + lane) * 8u;
                load8<T>(more[i], r + at, there ? int(a.dim) - int(at) : 0);
            }
#pragma unroll
            for (int i = 0; i < RUNS; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] += more[i][j];
        }
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = (uint32_t(i) * LANES + lane) * 8u;
            if (a.sum != nullptr) store8<T>(sum + at, h[i], there ? int(a.dim) - int(at) : 0);
#pragma unroll
            for (int j = 0; j < 8; ++j) squares = fmaf(h[i][j], h[i][j], squares);
        }
        squares = lanes_sum<kAll ? 64 : LANES>(squares);
        if constexpr (kAll) {
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = squares;
            __syncthreads();
            squares = part[0];
#pragma unroll
            for (int i = 1; i < THREADS / 64; ++i) squares += part[i];
            __syncthreads();
        }
        const float mean = squares / float(a.dim) + a.eps;
        const float inverse = mean < __int_as_float(0x7f800000) ? 1.0f / sqrtf(mean) : __int_as_float(0x7fc00000);
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = (uint32_t(i) * LANES + lane) * 8u;
            const int left = there ? int(a.dim) - int(at) : 0;
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
                if (left >= 8) {
                    typedef uint32_t Two __attribute__((ext_vector_type(2), aligned(1)));
                    *reinterpret_cast<Two *>(to) = Two{c0, c1};
                } else {
                    store4(to, c0, left);
                    store4(to + 4, c1, left - 4);
                }
                if ((threadIdx.x & 15) == 0) store_scale<TO == kToFp8E8>(a.scales, size_t(row) * a.scale_stride + at / kScaleBlock, stored);
            }
        }
    }
}
template <typename T, int TO, int LANES, int RUNS, int THREADS>
static hipError_t norm_form(const NormArgs &a, hipStream_t s) {
    const uint64_t groups = (uint64_t(a.rows) + THREADS / LANES - 1) / (THREADS / LANES);
    return launch(k_rms_norm<T, TO, LANES, RUNS, THREADS>, uint32_t(groups < kMostGroups ? groups : kMostGroups), THREADS, 0, s, a);
}
// (By a row's length alone: the order of its sums is the same whatever rows stand beside it.)
template <typename T, int TO>
static hipError_t norm(const NormArgs &a, hipStream_t s) {
    if (a.dim <= 128) return norm_form<T, TO, 16, 1, 256>(a, s);
    if (a.dim <= 256) return norm_form<T, TO, 32, 1, 256>(a, s);
    if (a.dim <= 512) return norm_form<T, TO, 64, 1, 256>(a, s);
    if (a.dim <= 1024) return norm_form<T, TO, 128, 1, 128>(a, s);
    if (a.dim <= 2048) return norm_form<T, TO, 256, 1, 256>(a, s);
    if (a.dim <= 4096) return norm_form<T, TO, 256, 2, 256>(a, s);
    return a.dim <= 8192 ? norm_form<T, TO, 512, 2, 512>(a, s) : norm_form<T, TO, 1024, 2, 1024>(a, s);
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
