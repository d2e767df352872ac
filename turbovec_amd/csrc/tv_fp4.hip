// 4-bit rows: making them, reading them back, and the product of two sets of them.
//
// A row's coordinates are e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two a byte; each block of 32 coordinates of a row has a power of two
// as its scale (e8m0).
#include "tv_rows.h"

namespace tv {

// ---------------------------------------------------------------------------
// Making 4-bit rows, and reading them.  A block's scale is the smallest power of two 2^e with amax < 7 * 2^e: 7 lies in the middle between
// the largest code, 6, and what would be the next, 8, so that the largest value is rounded as the others are.
// ---------------------------------------------------------------------------

// A thread to eight coordinates, four neighbours to a block.
constexpr int kThreads4 = 256;
template <typename T>
__global__ __launch_bounds__(kThreads4) void k_fp4_quantize(Quantize4Args a) {
    const uint32_t eights = (a.dim + 31u) / 32u * 4u;
    const uint64_t units = uint64_t(a.rows) * eights;
    for (uint64_t first = uint64_t(blockIdx.x) * kThreads4; first < units; first += uint64_t(gridDim.x) * kThreads4) {
        const uint64_t unit = first + threadIdx.x;
        const bool there = unit < units;
        const uint32_t row = there ? uint32_t(unit / eights) : 0u, at = uint32_t(unit % eights) * 8u;
        const int left = there ? int(a.dim) - int(at) : 0;
        float v[8];
        load8<T>(v, static_cast<const T *>(a.x) + size_t(row) * a.x_stride + at, left);
        const uint32_t most = quad_max(magnitude8(v));
        uint32_t stored;
        const uint32_t c = codes4_of(v, scale4_of(most, stored), most);
        if (left > 0) store_nibbles(a.codes + size_t(row) * a.code_stride + at / 2, c, left);
        if ((threadIdx.x & 3u) == 0u && left > 0) a.scales[size_t(row) * a.scale_stride + at / 32u] = uint8_t(stored);
    }
}
hipError_t launch_fp4_quantize(const Quantize4Args &a, int x_type, hipStream_t s) {
    const uint64_t groups = (uint64_t(a.rows) * ((a.dim + 31u) / 32u * 4u) + kThreads4 - 1) / kThreads4;
    const uint32_t grid = uint32_t(groups < kMostGroups ? groups : kMostGroups);
    if (x_type == kF32) return launch(k_fp4_quantize<float>, grid, kThreads4, 0, s, a);
    return x_type == kF16 ? launch(k_fp4_quantize<f16>, grid, kThreads4, 0, s, a) : launch(k_fp4_quantize<bf16>, grid, kThreads4, 0, s, a);
}

template <typename T>
__global__ __launch_bounds__(kThreads4) void k_fp4_values(Values4Args a) {
    typedef T T8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    const uint32_t eights = (a.dim + 7u) / 8u;
    const uint64_t units = uint64_t(a.rows.rows) * eights;
    for (uint64_t unit = uint64_t(blockIdx.x) * kThreads4 + threadIdx.x; unit < units; unit += uint64_t(gridDim.x) * kThreads4) {
        const uint32_t row = uint32_t(unit / eights), at = uint32_t(unit % eights) * 8u;
        const int left = int(a.dim) - int(at);
        const uint8_t *const from = a.rows.codes + size_t(row) * a.rows.stride + at / 2;
        uint32_t c = 0;
        if (left >= 7) __builtin_memcpy(&c, from, 4);
        else
            for (int i = 0; 2 * i < left; ++i) c |= uint32_t(from[i]) << (8 * i);
        const float s = e8_value(a.rows.scales[size_t(row) * a.rows.scale_stride + at / 32u]);
        float v[8];
        values_of4(v, c, s);
        T *const to = static_cast<T *>(a.out) + size_t(row) * a.out_stride + at;
        if (left >= 8) {
            T8 x;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = T(v[i]);
            *reinterpret_cast<T8 *>(to) = x;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) to[i] = T(v[i]);
        }
    }
}
hipError_t launch_fp4_values(const Values4Args &a, int out_type, hipStream_t s) {
    const uint64_t groups = (uint64_t(a.rows.rows) * ((a.dim + 7u) / 8u) + kThreads4 - 1) / kThreads4;
    const uint32_t grid = uint32_t(groups < kMostGroups ? groups : kMostGroups);
    if (out_type == kF32) return launch(k_fp4_values<float>, grid, kThreads4, 0, s, a);
    return out_type == kF16 ? launch(k_fp4_values<f16>, grid, kThreads4, 0, s, a) : launch(k_fp4_values<bf16>, grid, kThreads4, 0, s, a);
}

// ---------------------------------------------------------------------------
// The product: out[m][n] = sum over blocks of both scales times the sum of the block's products, by the matrix instructions, which apply a scale a lane at no cost.
// Products of codes are multiples of 1/4 up to 36, so that a block's sum is exact; blocks are added as 32-bit sums are (2e-8 to 1.2e-7 of the result where
// scales differ by orders, as much as a product in 32 bits loses; nothing where they are alike).  So one form serves results of every type.
// A lane holds 32 codes of one row, one block: lane group g the g-th block of 128 coordinates.
// ---------------------------------------------------------------------------

// The 32 codes from coordinate 2 * k on, those past the row's end zero.
__device__ __forceinline__ v4i codes32(const uint8_t *row, uint32_t k, uint32_t dim) {
    const uint32_t bytes = (dim + 1u) / 2u;
    if (k >= bytes) return v4i{0, 0, 0, 0};
    v4i v = codes16(row, k, bytes);
    if ((dim & 1u) && bytes - k <= 16u) {
        const uint32_t last = bytes - 1u - k;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (last / 4u == uint32_t(i)) v[i] &= int(~(0xf0u << (last % 4u * 8u)));
    }
    return v;
}
__device__ __forceinline__ v8i operand4(v4i v) { return v8i{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

template <typename T>
__global__ __launch_bounds__(64) void k_fp4_small(Matmul4Args p, uint32_t n_tiles) {
    const int lane = threadIdx.x, col = lane & 15, g = lane >> 4;
    const uint32_t blocks = (p.dim + 31u) / 32u;
    const uint32_t m0 = blockIdx.x / n_tiles * 16u, n0 = blockIdx.x % n_tiles * 16u;
    const uint32_t ra = min(m0 + col, p.a.rows - 1), rb = min(n0 + col, p.b.rows - 1);
    const uint8_t *const a = p.a.codes + size_t(ra) * p.a.stride, *const b = p.b.codes + size_t(rb) * p.b.stride;
    const uint8_t *const as = p.a.scales + size_t(ra) * p.a.scale_stride, *const bs = p.b.scales + size_t(rb) * p.b.scale_stride;
    v4f acc{0, 0, 0, 0};
    for (uint32_t k = 0; k < blocks; k += 4) {
        const uint32_t block = k + uint32_t(g);
        const v4i x = codes32(a, block * 16u, p.dim), y = codes32(b, block * 16u, p.dim);
        const int xs = block < blocks ? as[block] : 127, ys = block < blocks ? bs[block] : 127;
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand4(x), operand4(y), acc, 4, 4, 0, xs, 0, ys);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t m = m0 + 4u * g + r, n = n0 + col;
        if (m < p.a.rows && n < p.b.rows) static_cast<T *>(p.out)[size_t(m) * p.out_stride + n] = T(acc[r]);
    }
}
template <typename T>
static hipError_t matmul4(const Matmul4Args &a, hipStream_t s) {
    const uint64_t mt = (a.a.rows + 15u) / 16u, nt = (a.b.rows + 15u) / 16u;
    if (mt * nt * 64u >> 32) return hipErrorInvalidConfiguration;
    return launch(k_fp4_small<T>, uint32_t(mt * nt), 64, 0, s, a, uint32_t(nt));
}
hipError_t launch_fp4_matmul(const Matmul4Args &a, hipStream_t s) {
    if (a.out_type == kF32) return matmul4<float>(a, s);
    return a.out_type == kF16 ? matmul4<f16>(a, s) : matmul4<bf16>(a, s);
}

}  // namespace tv
