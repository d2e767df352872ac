// The root-mean-square norm of rows, a residual added before it, made into rows of 8 or 4 bits in the same pass.
#include <type_traits>

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
__device__ __forceinline__ double lanes_sum(double v) {
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
    if (p == nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 1.0f;
    } else if (type == kF32) load8<float>(w, static_cast<const float *>(p) + at, left);
    else if (type == kF16) load8<f16>(w, static_cast<const f16 *>(p) + at, left);
    else load8<bf16>(w, static_cast<const bf16 *>(p) + at, left);
}

enum { kToFp8E8 = 0, kToFp8F32 = 1, kToFp4 = 2 };

// A block's largest magnitude decides its power of two, and 32 bits (a root, a quotient and two products behind the mean) may put one next to the border, 1.75 times a power, on its wrong side: there it is
// taken again from the mean of the squares in 64 bits.  WHOLE: products too, by the lanes whose largest value it may be; where there are no registers left for that, the products
// stay rounded.  (`mean` is then how far the mean is above one over the inverse's square, as a share of it.)  `block`: the largest magnitude's bits, the same in the block's lanes, `mine` the lane's own; returned on the right side.
template <bool FP4, bool WHOLE>
__device__ __forceinline__ uint32_t settled(uint32_t block, uint32_t mine, const float (&h)[8], const float (&w)[8], const float (&y)[8], std::conditional_t<WHOLE, double, float> mean) {
    const bool near = (block & 0x7fffffu) - 0x5ffff8u <= 16u;
    if (!__any(near)) return block;
    double border = __hiloint2double(int((((block >> 23) + 896u) << 20) | 0xc0000u), 0), at = double(__uint_as_float(block));
    bool over;
    if constexpr (WHOLE) {
        float hm = 0.0f, wm = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool it = (__float_as_uint(y[j]) & 0x7fffffffu) == mine;
            hm = it ? h[j] : hm;
            wm = it ? w[j] : wm;
        }
        border *= border * mean;
        at = double(hm) * double(wm);
        constexpr uint32_t kLanes = FP4 ? 4u : 16u;
        over = mine + 16u >= block && (FP4 ? at * at >= border : at * at > border);
        over = (uint32_t(__ballot(over) >> (threadIdx.x & (64u - kLanes))) & ((1u << kLanes) - 1u)) != 0;
    } else {
        border *= border * (1.0 + double(mean));
        over = FP4 ? at * at >= border : at * at > border;
    }
    return near ? (block & 0xff800000u) + (FP4 ? 0x5fffffu : 0x600000u) + uint32_t(over) : block;
}
// Eight neighbouring values as they are stored; those past `left` are 0.
template <typename T>
struct Run8 {
    typedef T T8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    T8 v;
    __device__ __forceinline__ void load(const T *p, int left) {
        if (left >= 8) {
            v = *reinterpret_cast<const T8 *>(p);
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : T(0.0f);
    }
};

// Whether a workgroup that goes on to a next row asks for it, and keeps the weights, while it has the row before in hand.  Floats have twice the bytes on their way and no registers left, but for
// the longest rows, where few workgroups are held (4096 of 16384 84 us so and 97).
template <typename T> constexpr bool norm_ahead(int runs, int most) { return sizeof(T) == 2 || (runs == 2 && most == 1024); }
// Waves of a SIMD at once, which leave 64, 72, 80 or 128 registers to each.  Two runs a lane spill 2 to 7 of 80, but for floats into float scales, and one run of floats 2 of 64 where a workgroup's row goes
// into 8 bits with power-of-two scales.  More registers hold all, for fewer rows on their way (us so and with those: bfloat16 without a residual, 96 registers, 16384 of 5120 64 and 78, 8192 of 8192 50
// and 54, but 16384 of 4096 48 and 44; floats with a residual, 72, 8192 of 8192 165 and 175, but 40000 of 1536 150 and 139).
template <typename T> constexpr int norm_waves(int lanes, int runs, int most) { return runs == 1 ? (sizeof(T) == 2 || lanes == 0 ? 8 : 7) : runs == 2 && most < 1024 ? 6 : 4; }
// LANES lanes to a row, each with RUNS runs: sixteen to sixty-four, or (0) all of a workgroup, as many waves as the row fills, whose sums then go through LDS.
template <typename T, int TO, int LANES, int RUNS, int MOST>
__global__ __launch_bounds__(MOST, norm_waves<T>(LANES, RUNS, MOST)) void k_rms_norm(NormArgs a) {
    static_assert(RUNS * 8 <= 16, "squares of a thread that are added in 32 bits: 16 of up to 2^124 are below 2^128");
    constexpr bool kAll = LANES == 0;
    constexpr int kLanes = kAll ? 64 : LANES;
    __shared__ double part[kAll ? MOST / 64 : 1];
    const uint32_t lanes = kAll ? blockDim.x : uint32_t(LANES), together = kAll ? 1u : uint32_t(MOST / kLanes);
    const uint32_t lane = kAll ? threadIdx.x : threadIdx.x % kLanes, sub = kAll ? 0u : threadIdx.x / kLanes;
    constexpr bool kAhead = norm_ahead<T>(RUNS, MOST);
    float w[kAhead ? RUNS : 1][8];
    if constexpr (kAhead) {
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = (uint32_t(i) * lanes + lane) * 8u;
            load_weight(w[i], a.weight, a.weight_type, at, int(a.dim) - int(at));
        }
    }
    Run8<T> x[RUNS], r[RUNS];
    auto fetch = [&](uint64_t first) {
        if (first + sub >= a.rows) return;
        const T *const px = static_cast<const T *>(a.x) + size_t(first + sub) * a.x_stride, *const pr = static_cast<const T *>(a.residual) + size_t(first + sub) * a.residual_stride;
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = (uint32_t(i) * lanes + lane) * 8u;
            x[i].load(px + at, int(a.dim) - int(at));
            if (a.residual != nullptr) r[i].load(pr + at, int(a.dim) - int(at));
        }
    };
    if constexpr (kAhead) fetch(uint64_t(blockIdx.x) * together);
    for (uint64_t first = uint64_t(blockIdx.x) * together; first < a.rows; first += uint64_t(gridDim.x) * together) {
        const bool there = first + sub < a.rows;
        const uint32_t row = there ? uint32_t(first) + sub : a.rows - 1;
        T *const sum = static_cast<T *>(a.sum) + size_t(row) * a.sum_stride;
        float h[RUNS][8], squares = 0.0f;
        if constexpr (!kAhead) fetch(first);
#pragma unroll
        for (int i = 0; i < RUNS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = float(x[i].v[j]);
        if (a.residual != nullptr) {
#pragma unroll
            for (int i = 0; i < RUNS; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] += float(r[i].v[j]);
        }
        if constexpr (kAhead) fetch(first + uint64_t(gridDim.x) * together);          // (no row of the sum is one that is still to be read)
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = (uint32_t(i) * lanes + lane) * 8u;
            if (a.sum != nullptr) store8<T>(sum + at, h[i], there ? int(a.dim) - int(at) : 0);
#pragma unroll
            for (int j = 0; j < 8; ++j) squares = fmaf(h[i][j], h[i][j], squares);
        }
        double total = lanes_sum<kLanes>(double(squares));
        if constexpr (kAll) {
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = total;
            __syncthreads();
            total = part[0];
            for (uint32_t i = 1; i < lanes / 64u; ++i) total += part[i];
            __syncthreads();
        }
        const double exact_mean = total * a.share + double(a.eps);
        const float mean = float(exact_mean);
        const float inverse = mean < __int_as_float(0x7f800000) ? 1.0f / sqrtf(mean) : __int_as_float(0x7fc00000);
        constexpr bool kWhole = RUNS == 1 && kAll && TO == kToFp8E8 && sizeof(T) == 2;
        std::conditional_t<kWhole, double, float> settle_by;
        if constexpr (kWhole) settle_by = exact_mean;
        else settle_by = float(exact_mean * (double(inverse) * double(inverse)) - 1.0);
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const uint32_t at = (uint32_t(i) * lanes + lane) * 8u;
            const int left = there ? int(a.dim) - int(at) : 0;
            // (What lies behind a row's end is 0 here, or NaN where all of the row is.)
            float y[8];
            if constexpr (!kAhead) load_weight(w[0], a.weight, a.weight_type, at, left);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = h[i][j] * inverse * w[kAhead ? i : 0][j];
            uint32_t most = magnitude8(y), stored;
            if (TO == kToFp4) {
                const uint32_t block = settled<true, kWhole>(quad_max(most), most, h[i], w[kAhead ? i : 0], y, settle_by), c = codes4_of(y, scale4_of(block, stored), block);
                if (left <= 0) continue;
                store_nibbles(a.codes + size_t(row) * a.code_stride + at / 2u, c, left);
                if ((threadIdx.x & 3) == 0) static_cast<uint8_t *>(a.scales)[size_t(row) * a.scale_stride + at / kScaleBlock4] = uint8_t(stored);
            } else {
                const bool fine = TO == kToFp8E8 && !__any(most >= kInfBits);
                if (!fine) {
                    most = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        y[j] = j < left ? y[j] : 0.0f;
                        most = max(most, __float_as_uint(finite_abs(y[j])));
                    }
                }
                uint32_t block = __float_as_uint(row16_max(__uint_as_float(most)));
                if (TO == kToFp8E8) block = settled<false, kWhole>(block, most, h[i], w[kAhead ? i : 0], y, settle_by);
                const float s = scale_of<TO == kToFp8E8>(__uint_as_float(block), stored);
                uint32_t c[2];
                if (TO == kToFp8E8 && fine) {
                    const float by = __uint_as_float((254u << 23) - __float_as_uint(s));
#pragma unroll
                    for (int l = 0; l < 2; ++l)
                        c[l] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * l + 2] * by, y[4 * l + 3] * by, __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * l] * by, y[4 * l + 1] * by, 0, false), true));
                } else {
                    const float lo[4] = {y[0], y[1], y[2], y[3]}, hi[4] = {y[4], y[5], y[6], y[7]};
                    c[0] = codes_of<TO == kToFp8E8>(lo, s);
                    c[1] = codes_of<TO == kToFp8E8>(hi, s);
                }
                if (left <= 0) continue;
                uint8_t *const to = a.codes + size_t(row) * a.code_stride + at;
                if (left >= 8) {
                    typedef uint32_t Two __attribute__((ext_vector_type(2), aligned(1)));
                    *reinterpret_cast<Two *>(to) = Two{c[0], c[1]};
                } else {
                    store4(to, c[0], left);
                    store4(to + 4, c[1], left - 4);
                }
                if ((threadIdx.x & 15) == 0) store_scale<TO == kToFp8E8>(a.scales, size_t(row) * a.scale_stride + at / kScaleBlock, stored);
            }
        }
    }
}
template <typename T, int TO, int LANES, int RUNS, int MOST>
static hipError_t norm_form(const NormArgs &a, hipStream_t s) {
    const uint32_t threads = LANES == 0 ? (a.dim + 512u * RUNS - 1) / (512u * RUNS) * 64u : uint32_t(MOST);
    const uint64_t together = LANES == 0 ? 1 : MOST / (LANES == 0 ? 1 : LANES), groups = (uint64_t(a.rows) + together - 1) / together;
    const bool stays = norm_ahead<T>(RUNS, MOST) && (RUNS > 1 || a.residual == nullptr);
    const uint64_t held = stays ? 256u * (4u * norm_waves<T>(LANES, RUNS, MOST) * 64u / threads) : kMostGroups;
    return launch(k_rms_norm<T, TO, LANES, RUNS, MOST>, uint32_t(groups < held ? groups : held), threads, 0, s, a);
}
// Bound by memory: 16384 rows of 4096 bfloat16 with a residual take 82 us, 5.7 TB/s, 43 % of it written (a copy reaches 4.6 to 4.9), 8192 of 8192 85, 16384 of 5120 113.  With a residual most is on its
// way at a time with a run to a lane and a workgroup to a row (with two runs and workgroups that stay 90, 90 and 112); without one, with two runs and workgroups that stay and ask for their
// next row in time (16384 of 4096 made 8-bit 43 us so, a workgroup to each row 48 to 59; 16384 of 5120 made 4-bit 54, and 81 with a power of two of lanes).  The longest rows have
// two runs and workgroups that stay either way (4096 of 16384 bfloat16 with a residual 88 us, a workgroup to each row 109).
// (A row's form follows from its length, its type and whether there is a residual: the order of its sums is the same whatever rows stand beside it.)
template <typename T, int TO>
static hipError_t norm(const NormArgs &a, hipStream_t s) {
    if (a.dim <= 128) return norm_form<T, TO, 16, 1, 256>(a, s);
    if (a.dim <= 256) return norm_form<T, TO, 32, 1, 256>(a, s);
    if (a.dim <= 512) return norm_form<T, TO, 64, 1, 256>(a, s);
    if (a.dim <= 2048 || (a.dim <= 8192 && a.residual != nullptr)) return norm_form<T, TO, 0, 1, 1024>(a, s);
    if (a.dim <= 8192) return norm_form<T, TO, 0, 2, 512>(a, s);
    return norm_form<T, TO, 0, 2, 1024>(a, s);
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
