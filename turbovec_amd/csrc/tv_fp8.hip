// 8-bit rows: making them, and the product of two sets of them.
//
// A row's coordinates are e4m3 codes (4 exponent bits, 3 of mantissa, largest value 448); each block of 128 coordinates has
// a scale, of its own row or of the tile of 128 rows it lies in: a float, or the exponent alone of a power of two (e8m0), which
// the matrix unit applies itself.
#include "tv_device.h"
#include "tv_ops.h"

namespace tv {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// Making 8-bit rows.  Scale of a block: amax / 448 over its finite values, or the smallest power of two not below that; codes
// are x / scale rounded to the nearest, ties to even.
// ---------------------------------------------------------------------------

// Four values from p, those of them past `left` zero.
template <typename T, bool VEC>
__device__ __forceinline__ void load4(float (&v)[4], const T *p, int left) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (VEC && left >= 4) {
        const T4 x = *reinterpret_cast<const T4 *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = float(x[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? float(p[i]) : 0.0f;
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < __int_as_float(0x7f800000) ? a : 0.0f;      // (a comparison with NaN is false)
}
// Largest over the half wave.
__device__ __forceinline__ float half_wave_max(float v) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
// The scale of a block whose largest finite magnitude is `most`; `stored` is what goes to memory.
template <bool E8>
__device__ __forceinline__ float scale_of(float most, uint32_t &stored) {
    if (!E8) {
        const float s = fmaxf(most / 448.0f, 0x1p-126f);
        stored = __float_as_uint(s);
        return s;
    }
    // most = f * 2^e with 1 <= f < 2, 448 = 1.75 * 2^8: the power is e - 8, one more where f > 1.75
    const uint32_t b = __float_as_uint(most);
    const int e = int(b >> 23) - 127 - 8 + int((b & 0x7fffffu) > 0x600000u);
    const int power = e < -126 ? -126 : e;                 // (denormal maxima, zero among them, end here)
    stored = uint32_t(power + 127);
    return __uint_as_float(stored << 23);
}
__device__ __forceinline__ uint32_t codes_of(const float (&v)[4], float s) {
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = fabsf(v[i]) < __int_as_float(0x7f800000) ? v[i] / s : __int_as_float(0x7fc00000);
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], r, true));
}
template <bool VEC>
__device__ __forceinline__ void store4(uint8_t *p, uint32_t c, int left) {
    if (VEC && left >= 4) {
        *reinterpret_cast<uint32_t *>(p) = c;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) p[i] = uint8_t(c >> (8 * i));
}
template <bool E8>
__device__ __forceinline__ void store_scale(void *scales, size_t at, uint32_t stored) {
    if (E8) static_cast<uint8_t *>(scales)[at] = uint8_t(stored);
    else static_cast<uint32_t *>(scales)[at] = stored;
}

// A scale for each row: half a wave to a block, four blocks at a time.
constexpr int kQuantThreads = 256, kQuantUnits = 4;
constexpr uint64_t kMostGroups = 1 << 20;    // workgroups of a launch: a grid of 2^32 threads is not allowed
template <typename T, bool E8, bool VEC>
__global__ __launch_bounds__(kQuantThreads) void k_fp8_quantize_rows(QuantizeArgs a) {
    const uint32_t blocks = (a.dim + kScaleBlock - 1) / kScaleBlock;
    const uint64_t units = uint64_t(a.rows) * blocks;
    const int lane = threadIdx.x & 31;
    constexpr uint32_t kPer = kQuantThreads / 32 * kQuantUnits;
    for (uint64_t first = uint64_t(blockIdx.x) * kPer + (threadIdx.x >> 5); first - (threadIdx.x >> 5) < units; first += uint64_t(gridDim.x) * kPer) {
    float v[kQuantUnits][4];
    uint32_t row[kQuantUnits], block[kQuantUnits];
#pragma unroll
    for (int i = 0; i < kQuantUnits; ++i) {
        const uint64_t unit = first + i * (kQuantThreads / 32);
        row[i] = unit < units ? uint32_t(unit / blocks) : ~0u;
        block[i] = uint32_t(unit % blocks);
        const uint32_t at = block[i] * kScaleBlock + lane * 4;
        load4<T, VEC>(v[i], static_cast<const T *>(a.x) + size_t(row[i]) * a.x_stride + at, row[i] == ~0u ? 0 : int(a.dim) - int(at));
    }
#pragma unroll
    for (int i = 0; i < kQuantUnits; ++i) {
        const float most = half_wave_max(fmaxf(fmaxf(finite_abs(v[i][0]), finite_abs(v[i][1])), fmaxf(finite_abs(v[i][2]), finite_abs(v[i][3]))));
        if (row[i] == ~0u) continue;
        uint32_t stored;
        const float s = scale_of<E8>(most, stored);
        const uint32_t at = block[i] * kScaleBlock + lane * 4;
        store4<VEC>(a.codes + size_t(row[i]) * a.code_stride + at, codes_of(v[i], s), int(a.dim) - int(at));
        if (lane == 0) store_scale<E8>(a.scales, size_t(row[i]) * a.scale_stride + block[i], stored);
    }
    }
}

// A scale for each 128 x 128 tile: a workgroup to a tile, sixteen rows to half a wave.
template <typename T, bool E8, bool VEC>
__global__ __launch_bounds__(kQuantThreads) void k_fp8_quantize_tiles(QuantizeArgs a) {
    __shared__ float part[kQuantThreads / 32];
    constexpr int kRows = 128 / (kQuantThreads / 32);
    const uint32_t blocks = (a.dim + kScaleBlock - 1) / kScaleBlock;
    const uint32_t tiles = (a.rows + 127u) / 128u;
    for (uint64_t unit = blockIdx.x; unit < uint64_t(tiles) * blocks; unit += gridDim.x) {
    const uint32_t tile = uint32_t(unit / blocks), block = uint32_t(unit % blocks);
    const int lane = threadIdx.x & 31, half = threadIdx.x >> 5;
    const uint32_t at = block * kScaleBlock + lane * 4;
    float v[kRows][4], most = 0.0f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t row = tile * 128u + uint32_t(i * (kQuantThreads / 32) + half);
        load4<T, VEC>(v[i], static_cast<const T *>(a.x) + size_t(row) * a.x_stride + at, row < a.rows ? int(a.dim) - int(at) : 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) most = fmaxf(most, finite_abs(v[i][j]));
    }
    most = half_wave_max(most);
    if (lane == 0) part[half] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQuantThreads / 32; ++i) most = fmaxf(most, part[i]);
    uint32_t stored;
    const float s = scale_of<E8>(most, stored);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t row = tile * 128u + uint32_t(i * (kQuantThreads / 32) + half);
        if (row < a.rows) store4<VEC>(a.codes + size_t(row) * a.code_stride + at, codes_of(v[i], s), int(a.dim) - int(at));
    }
    if (threadIdx.x == 0) store_scale<E8>(a.scales, size_t(tile) * a.scale_stride + block, stored);
    __syncthreads();
    }
}

template <typename T, bool E8, bool VEC>
static hipError_t quantize(const QuantizeArgs &a, int group_shift, hipStream_t s) {
    const uint64_t blocks = (a.dim + kScaleBlock - 1) / kScaleBlock;
    if (group_shift == 0) {
        constexpr uint64_t per = kQuantThreads / 32 * kQuantUnits;
        const uint64_t groups = (a.rows * blocks + per - 1) / per;
        return launch(k_fp8_quantize_rows<T, E8, VEC>, uint32_t(groups < kMostGroups ? groups : kMostGroups), kQuantThreads, 0, s, a);
    } else {
        const uint64_t groups = (uint64_t(a.rows) + 127) / 128 * blocks;
        return launch(k_fp8_quantize_tiles<T, E8, VEC>, uint32_t(groups < kMostGroups ? groups : kMostGroups), kQuantThreads, 0, s, a);
    }
}
template <typename T>
static hipError_t quantize_as(const QuantizeArgs &a, int scale_type, int group_shift, hipStream_t s) {
    // four values at a time where every row starts at a multiple of four
    const bool vec = (uintptr_t(a.x) % (4 * sizeof(T)) | a.x_stride % 4 | uintptr_t(a.codes) % 4 | a.code_stride % 4) == 0;
    if (scale_type == kScaleE8M0) return vec ? quantize<T, true, true>(a, group_shift, s) : quantize<T, true, false>(a, group_shift, s);
    return vec ? quantize<T, false, true>(a, group_shift, s) : quantize<T, false, false>(a, group_shift, s);
}
hipError_t launch_fp8_quantize(const QuantizeArgs &a, int x_type, int scale_type, int group_shift, hipStream_t s) {
    if (x_type == kF32) return quantize_as<float>(a, scale_type, group_shift, s);
    return x_type == kF16 ? quantize_as<f16>(a, scale_type, group_shift, s) : quantize_as<bf16>(a, scale_type, group_shift, s);
}

// ---------------------------------------------------------------------------
// The product: out[m][n] = sum over blocks of a's scale * b's scale * (sum over the block's codes), in f32.
//
// 16 x 16 x 128 matrix instructions: one covers a block of 128 coordinates of 16 rows of b (its first operand) and 16 rows of
// a (its second).  A lane holds 32 codes of one row of each; which 32 of the 128 does not matter as long as both operands
// agree, so a lane takes two runs of 16 bytes.  Lane l of the result holds row l % 16 of a against rows 4 * (l / 16) .. + 3 of b.
// ---------------------------------------------------------------------------

constexpr int kUnitScale = 0x7f7f7f7f;       // 2^0 in each byte

// 16 codes of a row from k on, those past `dim` zero, without touching what lies behind the row.
__device__ __forceinline__ void codes16(int *to, const uint8_t *row, uint32_t k, uint32_t dim) {
    if (k + 16u <= dim) {
        __builtin_memcpy(to, row + k, 16);
        return;
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t x = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (k + w * 4 + i < dim) x |= uint32_t(row[k + w * 4 + i]) << (8 * i);
        to[w] = int(x);
    }
}
__device__ __forceinline__ v8i operand(const uint8_t *row, uint32_t block, int g, uint32_t dim) {
    int w[8];
    codes16(w, row, block * kScaleBlock + g * 16, dim);
    codes16(w + 4, row, block * kScaleBlock + 64 + g * 16, dim);
    return v8i{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]};
}

__device__ __forceinline__ void store_out(void *out, size_t at, float v, int type) {
    if (type == kF32) static_cast<float *>(out)[at] = v;
    else if (type == kF16) static_cast<f16 *>(out)[at] = f16(v);
    else static_cast<bf16 *>(out)[at] = bf16(v);
}

constexpr int kDirectThreads = 256;
template <bool E8, int MT>
__global__ __launch_bounds__(kDirectThreads) void k_fp8_direct(MatmulArgs p) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const uint32_t n0 = (blockIdx.x * (kDirectThreads / 64) + (threadIdx.x >> 6)) * 16u;
    if (n0 >= p.b.rows) return;
    const uint32_t blocks = (p.dim + kScaleBlock - 1) / kScaleBlock;
    // (rows past the end are the last one: their results are not stored)
    const uint32_t br = min(n0 + uint32_t(col), p.b.rows - 1);
    const uint8_t *b = p.b.codes + size_t(br) * p.b.stride;
    for (uint32_t m0 = blockIdx.y * (16u * MT); m0 < p.a.rows; m0 += gridDim.y * (16u * MT)) {
    const uint8_t *a[MT];
    uint32_t ar[MT];
    v4f acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        ar[t] = min(m0 + uint32_t(t * 16 + col), p.a.rows - 1);
        a[t] = p.a.codes + size_t(ar[t]) * p.a.stride;
        acc[t] = v4f{0, 0, 0, 0};
    }
    for (uint32_t k = 0; k < blocks; ++k) {
        const v8i bv = operand(b, k, g, p.dim);
        if (E8) {
            const int bs = static_cast<const uint8_t *>(p.b.scales)[size_t(br >> p.b.group_shift) * p.b.scale_stride + k];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int as = static_cast<const uint8_t *>(p.a.scales)[size_t(ar[t]) * p.a.scale_stride + k];
                acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bv, operand(a[t], k, g, p.dim), acc[t], 0, 0, 0, bs, 0, as);
            }
        } else {
            float bs[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                bs[r] = static_cast<const float *>(p.b.scales)[size_t(min(n0 + uint32_t(4 * g + r), p.b.rows - 1) >> p.b.group_shift) * p.b.scale_stride + k];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float as = static_cast<const float *>(p.a.scales)[size_t(ar[t]) * p.a.scale_stride + k];
                const v4f part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bv, operand(a[t], k, g, p.dim), v4f{0, 0, 0, 0}, 0, 0, 0, kUnitScale, 0, kUnitScale);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[t][r] = fmaf(part[r], bs[r] * as, acc[t][r]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const uint32_t m = m0 + uint32_t(t * 16 + col);
        if (m >= p.a.rows) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t n = n0 + uint32_t(4 * g + r);
            if (n < p.b.rows) store_out(p.out, size_t(m) * p.out_stride + n, acc[t][r], p.out_type);
        }
    }
    }
}

template <bool E8, int MT>
static hipError_t direct(const MatmulArgs &a, hipStream_t s) {
    const uint32_t tiles = (a.a.rows + 16 * MT - 1) / (16 * MT);
    const dim3 grid((a.b.rows + 63) / 64, tiles < 65535u ? tiles : 65535u);
    return launch(k_fp8_direct<E8, MT>, grid, kDirectThreads, 0, s, a);
}
hipError_t launch_fp8_matmul(const MatmulArgs &a, int scale_type, hipStream_t s) {
    const bool few = a.a.rows <= 16;
    if (scale_type == kScaleE8M0) return few ? direct<true, 1>(a, s) : direct<true, 4>(a, s);
    return few ? direct<false, 1>(a, s) : direct<false, 4>(a, s);
}

}  // namespace tv
