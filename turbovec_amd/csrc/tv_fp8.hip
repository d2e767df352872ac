// 8-bit rows: making them, and the product of two sets of them.
//
// A row's coordinates are e4m3 codes (4 exponent bits, 3 of mantissa, largest value 448); each block of 128 coordinates has
// a scale, of its own row or of the tile of 128 rows it lies in: a float, or the exponent alone of a power of two (e8m0), which
// the matrix unit applies itself.
#include <cmath>

#include "tv_device.h"
#include "tv_rows.h"

namespace tv {

// ---------------------------------------------------------------------------
// Making 8-bit rows.  Scale of a block: amax / 448 over its finite values, or the smallest power of two not below that; codes
// are x / scale rounded to the nearest, ties to even.
// ---------------------------------------------------------------------------

// A scale for each row: half a wave to a block, four blocks at a time, 16 bytes of floats a lane wherever a row starts (100K of 1535: 145 us, 207 an
// element at a time).  Bound by memory: 400K rows of 1536 floats take 549 us, 5.6 TB/s read and
// written (a copy reaches 4.9, half of it writes).
constexpr int kQuantThreads = 256, kQuantUnits = 4;
template <typename T, bool E8>
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
        load4<T>(v[i], static_cast<const T *>(a.x) + size_t(row[i]) * a.x_stride + at, row[i] == ~0u ? 0 : int(a.dim) - int(at));
    }
#pragma unroll
    for (int i = 0; i < kQuantUnits; ++i) {
        const float most = half_wave_max(fmaxf(fmaxf(finite_abs(v[i][0]), finite_abs(v[i][1])), fmaxf(finite_abs(v[i][2]), finite_abs(v[i][3]))));
        if (row[i] == ~0u) continue;
        uint32_t stored;
        const float s = scale_of<E8>(most, stored);
        const uint32_t at = block[i] * kScaleBlock + lane * 4;
        store4(a.codes + size_t(row[i]) * a.code_stride + at, codes_of<E8>(v[i], s), int(a.dim) - int(at));
        if (lane == 0) store_scale<E8>(a.scales, size_t(row[i]) * a.scale_stride + block[i], stored);
    }
    }
}

// A scale for each 128 x 128 tile: a workgroup to a tile, sixteen rows to half a wave, which holds them until the scale is known.
template <typename T, bool E8>
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
        load4<T>(v[i], static_cast<const T *>(a.x) + size_t(row) * a.x_stride + at, row < a.rows ? int(a.dim) - int(at) : 0);
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
        if (row < a.rows) store4(a.codes + size_t(row) * a.code_stride + at, codes_of<E8>(v[i], s), int(a.dim) - int(at));
    }
    if (threadIdx.x == 0) store_scale<E8>(a.scales, size_t(tile) * a.scale_stride + block, stored);
    __syncthreads();
    }
}

template <typename T, bool E8>
static hipError_t quantize(const QuantizeArgs &a, int group_shift, hipStream_t s) {
    const uint64_t blocks = (a.dim + kScaleBlock - 1) / kScaleBlock;
    if (group_shift == 0) {
        constexpr uint64_t per = kQuantThreads / 32 * kQuantUnits;
        const uint64_t groups = (a.rows * blocks + per - 1) / per;
        return launch(k_fp8_quantize_rows<T, E8>, uint32_t(groups < kMostGroups ? groups : kMostGroups), kQuantThreads, 0, s, a);
    } else {
        const uint64_t groups = (uint64_t(a.rows) + 127) / 128 * blocks;
        return launch(k_fp8_quantize_tiles<T, E8>, uint32_t(groups < kMostGroups ? groups : kMostGroups), kQuantThreads, 0, s, a);
    }
}
template <typename T>
static hipError_t quantize_as(const QuantizeArgs &a, int scale_type, int group_shift, hipStream_t s) {
    return scale_type == kScaleE8M0 ? quantize<T, true>(a, group_shift, s) : quantize<T, false>(a, group_shift, s);
}
hipError_t launch_fp8_quantize(const QuantizeArgs &a, int x_type, int scale_type, int group_shift, hipStream_t s) {
    if (x_type == kF32) return quantize_as<float>(a, scale_type, group_shift, s);
    return x_type == kF16 ? quantize_as<f16>(a, scale_type, group_shift, s) : quantize_as<bf16>(a, scale_type, group_shift, s);
}

// ---------------------------------------------------------------------------
// The product: out[m][n] = sum over blocks of a's scale * b's scale * (sum over the block's codes), in f32.
//
// Two ways to a block's sum, by the type of the result:
//  * 16-bit results: the 8-bit matrix instructions, 16 x 16 x 128, one to a block.  They add products in groups of eight
//    neighbours, each product cut off (towards zero) at 2^-13 of the group's largest, whose factors count as the powers of two at or below them: on random
//    rows 1.4e-5 of the usual result (root mean square), 1/280 of half a step of bfloat16 there, 1/35 of float16's, more of a result that is small among
//    large products.  In bfloat16 operands these results would be 24 bits good and take 2.3 times as long.  4.2 PFLOP/s measured on registers alone.
//  * 32-bit results: the same codes as bfloat16, which holds them exactly, and the 16 x 16 x 32 instructions for those, whose sums
//    round as 32-bit ones do (1e-8).  1.8 PFLOP/s.  A power-of-two scale goes in with the conversion (one instruction for two
//    codes, scale included), exactly as long as code * scale is one of bfloat16's: below 2^128, a multiple of 2^-133.
// Power-of-two scales cost no instruction in either form.  Scales that are floats multiply each block's sum: a
// multiply-add a result, and one more multiplication where both sides have a scale of each row.  The product of two scales may lie outside 32 bits
// where the result is a number (rows of 1e-20 on both sides, or of 1e23 whose products are 0), so it is not taken: the sum is multiplied
// by a's scale, then by b's.  Where 128 rows of b share theirs, its power of two goes into their operand and what is left, 1 to 2, into a's scale.
// (As fast as taking that product, except 4096 by 4096 of 4096 with shared scales: 69 us for 67.  Powers of two into the operands for each row
// of both sides: 1024 by 20000 of 1536 into floats 90 us where this takes 82.)
//
// A lane of a matrix operand holds 32 codes of one row in a block.  Which 32 of the 128 does not matter as long as both operands
// agree, so lane group g takes the runs of 16 at 16 g and 64 + 16 g.
// ---------------------------------------------------------------------------

constexpr int kUnitScale = 0x7f;             // 2^0
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));

// An operand of a block: 32 codes of a lane, as they are or as bfloat16 times a power of two.
template <bool EXACT> struct Operand;
template <> struct Operand<false> {
    v8i v;
    __device__ __forceinline__ void set(v4i lo, v4i hi, float) { v = v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}; }
};
template <> struct Operand<true> {
    v8b v[4];
    __device__ __forceinline__ static v8b eight(int x, int y, float s) {
        const v2b a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, true);
        const v2b c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, s, true);
        return v8b{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    __device__ __forceinline__ void set(v4i lo, v4i hi, float s) {
        v[0] = eight(lo[0], lo[1], s); v[1] = eight(lo[2], lo[3], s);
        v[2] = eight(hi[0], hi[1], s); v[3] = eight(hi[2], hi[3], s);
    }
};
// c + x * y over a block; the scales (e8m0 bytes) count where the instruction applies them.
__device__ __forceinline__ v4f block_product(const Operand<false> &x, const Operand<false> &y, v4f c, int xs, int ys) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x.v, y.v, c, 0, 0, 0, xs, 0, ys);
}
__device__ __forceinline__ v4f block_product(const Operand<true> &x, const Operand<true> &y, v4f c, int, int) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v[i], y.v[i], c, 0, 0, 0);
    return c;
}
// The power of two (an e8m0 byte) that the operand takes of a scale that rows of b share, and what is left.  From 2^-100 to 2^103: codes times that
// are normal numbers, and sums of their products less than 2^128.
__device__ __forceinline__ float shared_scale(float s, uint32_t &power) {
    power = min(max((__float_as_uint(s) >> 23) & 255u, 127u - 100u), 127u + 103u);
    return ldexpf(s, 127 - int(power));
}

__device__ __forceinline__ void store_out(void *out, size_t at, float v, int type) {
    if (type == kF32) static_cast<float *>(out)[at] = v;
    else if (type == kF16) static_cast<f16 *>(out)[at] = f16(v);
    else static_cast<bf16 *>(out)[at] = bf16(v);
}

// Up to sixteen rows of a: bound by reading b once.  A wave streams 16 rows of b from memory into registers, four blocks while the four
// before are multiplied, and goes on to its next 16 rows without a pause; a lies in LDS.  Where there are few rows of b (SPLIT), the four
// waves of a workgroup share 16 rows, each taking every fourth step, and their sums are added in the waves' order.
// One row against 1M of 1536 coordinates, into floats: 266 us, 5.8 TB/s where a pure read reaches 6.5.
constexpr int kDirectThreads = 256, kDirectWaves = kDirectThreads / 64, kDirectBlocks = 4;
constexpr uint32_t kDirectGroups = 4;         // workgroups of a compute unit at a time
constexpr size_t kDirectLds = 64 << 10;      // of a's rows, at most, where workgroups stream
constexpr size_t kMostLds = 160 << 10;        // of a compute unit

// Scales of kDirectBlocks blocks from k on, of `blocks` in the row; those past the end are whatever.
struct Scales4 {
    uint32_t v[4];
    template <bool E8>
    __device__ __forceinline__ void load(const void *scales, size_t row, uint32_t k, uint32_t blocks) {
        static_assert(kDirectBlocks == 4, "a word of bytes");
        if (E8) {
            const uint8_t *const s = static_cast<const uint8_t *>(scales) + row;
            if (k + 4u <= blocks) {
                __builtin_memcpy(&v[0], s + k, 4);
            } else {
                v[0] = 0;
                for (uint32_t i = 0; k + i < blocks; ++i) v[0] |= uint32_t(s[k + i]) << (8 * i);
            }
        } else {
            const uint32_t *const s = static_cast<const uint32_t *>(scales) + row;
            if (k + 4u <= blocks) __builtin_memcpy(v, s + k, 16);
            else
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = s[min(k + i, blocks - 1)];
        }
    }
    template <bool E8>
    __device__ __forceinline__ uint32_t at(int i) const { return E8 ? (v[0] >> (8 * i)) & 255u : v[i]; }
};

__host__ __device__ inline uint32_t direct_row(uint32_t dim) { return (dim + 127u) / 128u * 128u + 16u; }     // (rows of a a few banks apart)
inline size_t direct_lds(uint32_t rows, uint32_t dim) { return size_t(rows) * direct_row(dim) + (dim + 127) / 128 * 64 + kDirectWaves * 64 * 16; }

template <bool EXACT, bool E8, bool SPLIT>
__global__ __launch_bounds__(kDirectThreads, kDirectGroups) void k_fp8_direct(MatmulArgs p) {
    extern __shared__ uint8_t smem[];
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const uint32_t blocks = (p.dim + kScaleBlock - 1) / kScaleBlock, whole = p.dim / kScaleBlock, row_bytes = direct_row(p.dim), m = p.a.rows;
    uint32_t *const a_scales = reinterpret_cast<uint32_t *>(smem + m * row_bytes);       // [block][16]
    v4f *const sums = reinterpret_cast<v4f *>(a_scales + blocks * 16);                   // SPLIT: [wave][lane]
    for (uint32_t i = threadIdx.x; i < m * blocks * 8u; i += kDirectThreads) {
        const uint32_t r = i / (blocks * 8u), c = i % (blocks * 8u) * 16u;
        *reinterpret_cast<v4i *>(smem + r * row_bytes + c) = codes16(p.a.codes + size_t(r) * p.a.stride, c, p.dim);
    }
    for (uint32_t i = threadIdx.x; i < blocks * 16u; i += kDirectThreads) {
        const size_t at = size_t(min(i & 15u, m - 1)) * p.a.scale_stride + (i >> 4);
        a_scales[i] = E8 ? static_cast<const uint8_t *>(p.a.scales)[at] : static_cast<const uint32_t *>(p.a.scales)[at];
    }
    __syncthreads();
    // (rows past the end are the last one: their results are not stored)
    const uint8_t *const a = smem + min(uint32_t(col), m - 1) * row_bytes + g * 16;

    const uint32_t tiles = (p.b.rows + 15) / 16, steps = (blocks + kDirectBlocks - 1) / kDirectBlocks;
    const uint32_t tile_stride = SPLIT ? gridDim.x : gridDim.x * kDirectWaves, step_stride = SPLIT ? kDirectWaves : 1, first_step = SPLIT ? wave : 0;
    struct Place {
        uint32_t tile, step;
        const uint8_t *codes;
        size_t scales;
    };
    auto go_to = [&](Place &at, uint32_t tile) {
        const uint32_t row = min(tile * 16u + uint32_t(col), p.b.rows - 1);
        at = Place{tile, first_step, p.b.codes + size_t(row) * p.b.stride, size_t(row >> p.b.group_shift) * p.b.scale_stride};
    };
    struct Step {
        v4i codes[kDirectBlocks][2];
        Scales4 scales;
    };
    auto load = [&](Step &s, const Place &at) {
        if (at.tile >= tiles || at.step >= steps) return;
#pragma unroll
        for (int i = 0; i < kDirectBlocks; ++i) {
            const uint32_t k = (at.step * kDirectBlocks + i) * kScaleBlock + g * 16;
            s.codes[i][0] = *reinterpret_cast<const v4i_any *>(at.codes + min(k, p.dim - 16));
            s.codes[i][1] = *reinterpret_cast<const v4i_any *>(at.codes + min(k + 64, p.dim - 16));
        }
        s.scales.template load<E8>(p.b.scales, at.scales, at.step * kDirectBlocks, blocks);
    };
    v4f acc = v4f{0, 0, 0, 0};
    auto block = [&](uint32_t k, const v4i &b0, const v4i &b1, uint32_t bs) {
        const uint8_t *const from = a + k * kScaleBlock;
        const v4i a0 = *reinterpret_cast<const v4i *>(from), a1 = *reinterpret_cast<const v4i *>(from + 64);
        Operand<EXACT> x, y;
        if (E8) {
            const uint32_t as = a_scales[k * 16 + col];
            x.set(a0, a1, EXACT ? e8_value(as) : 1.0f);
            y.set(b0, b1, EXACT ? e8_value(bs) : 1.0f);
            acc = block_product(x, y, acc, int(as), int(bs));
        } else {
            x.set(a0, a1, 1.0f);
            y.set(b0, b1, 1.0f);
            const v4f part = block_product(x, y, v4f{0, 0, 0, 0}, kUnitScale, kUnitScale);
            const v4f as = *reinterpret_cast<const v4f *>(a_scales + k * 16 + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = fmaf(part[r] * as[r], __uint_as_float(bs), acc[r]);
        }
    };
    auto multiply = [&](const Step &s, const Place &at) {
#pragma unroll
        for (int i = 0; i < kDirectBlocks; ++i) {
            const uint32_t k = at.step * kDirectBlocks + i, from = k * kScaleBlock + g * 16;
            if (k < whole) block(k, s.codes[i][0], s.codes[i][1], s.scales.template at<E8>(i));
            else if (k < blocks)               // (the last block ends early: what was loaded are the row's last 16 codes)
                block(k, bytes_down(s.codes[i][0], from - min(from, p.dim - 16)), bytes_down(s.codes[i][1], from + 64 - min(from + 64, p.dim - 16)), s.scales.template at<E8>(i));
        }
    };
    auto finish = [&](const Place &at) {
        if (SPLIT) {
            sums[threadIdx.x] = acc;
            __syncthreads();
            if (wave != 0) return;
#pragma unroll
            for (int w = 1; w < kDirectWaves; ++w) acc += sums[w * 64 + lane];
        }
        const uint32_t n = at.tile * 16u + uint32_t(col);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (uint32_t(4 * g + r) < m && n < p.b.rows) store_out(p.out, size_t(4 * g + r) * p.out_stride + n, acc[r], p.out_type);
        acc = v4f{0, 0, 0, 0};
    };
    Place here, next;
    Step even, odd;
    go_to(here, SPLIT ? blockIdx.x : blockIdx.x * kDirectWaves + wave);
    load(even, here);
    auto turn = [&](const Step &now, Step &then) {
        next = here;
        next.step += step_stride;
        if (next.step >= steps) go_to(next, SPLIT ? tiles : here.tile + tile_stride);
        load(then, next);
        multiply(now, here);
        if (next.tile != here.tile) finish(here);
        here = next;
    };
    while (here.tile < tiles) {
        turn(even, odd);
        if (here.tile >= tiles) break;
        turn(odd, even);
    }
}

template <bool EXACT, bool E8, bool SPLIT>
static hipError_t direct(const MatmulArgs &a, hipStream_t s) {
    const uint32_t tiles = (a.b.rows + 15) / 16, most = SPLIT ? tiles : 256 * kDirectGroups;
    const uint32_t grid = SPLIT ? tiles : (tiles + kDirectWaves - 1) / kDirectWaves;
    const size_t lds = direct_lds(a.a.rows, a.dim);
    const auto kernel = k_fp8_direct<EXACT, E8, SPLIT>;
    if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), lds); e != hipSuccess) return e;
    return launch(kernel, grid < most ? grid : most, kDirectThreads, lds, s, a);
}
// Many rows of a: a workgroup to a tile of TM rows of a and TN of b, WM x WN waves.  A block's codes of both go to LDS, as they are,
// while the block before is multiplied; a wave reads each operand once and keeps its part of the tile in registers.
//
// A row's block is 128 bytes in LDS, its eight runs of 16 swapped about by the row's number: eight neighbouring lanes, which read
// the same run of eight rows, find it in different banks.  Loads that go past the registers write lane l at 16 l, so each lane asks for the
// run that belongs there.
//
// Bound by the matrix unit and what feeds it: 4096 rows by 4096 of 4096 coordinates into bfloat16 56 us with e8m0 scales (2.4 PFLOP/s) and
// 69 to 76 with floats (1.8 to 2.0, the matrix units busy for 48 %: the multiply-adds of a row step follow all its products), where the library's 8-bit product
// of that size, one scale for all of it, takes 49.  1024 by 100000 of 1536 into floats 316 to 336 us, 0.94 to 1.0 PFLOP/s; the library's bfloat16 product of a
// large size reaches 1.16.
enum { kScaleBytes = 0, kScaleRows = 1, kScaleTiles = 2 };      // e8m0; floats of each row of b; floats of 128 rows of b

__device__ __forceinline__ void load16_to_lds(uint32_t lds, const uint8_t *base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <int TM, int TN, int WM, int WN> constexpr size_t tile_lds() { return 2 * (size_t(TM + TN) * kScaleBlock + 64 * WM * WN * 4); }

// A strip of 16 rows and COLS columns in LDS, with 16 bytes between rows so that lanes of neighbouring rows write to different banks.
template <typename T, int COLS> constexpr int kStripBytes = 16 * (COLS * int(sizeof(T)) + 16);

// A wave's results, whose lane l holds columns 4 * (l / 16) .. + 3 of row l % 16 of each tile, to rows from m on and columns from n on.
// (16 bytes at a time wherever a row starts: an element at a time, 1730 by 41540 of 98 into float16 took 146 us where it takes 50.)
template <typename T, int COLS, int MT, int NT>
__device__ __forceinline__ void store_strips(const MatmulArgs &p, const v4f (&acc)[MT][NT], uint8_t *strip, uint32_t m, uint32_t n, int lane) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int kEach = 16 / int(sizeof(T)), kLanes = COLS / kEach, kRowsAtOnce = 64 / kLanes, kRow = COLS * int(sizeof(T)) + 16;
    const int col = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j) *reinterpret_cast<T4 *>(strip + col * kRow + (j * 16 + 4 * g) * int(sizeof(T))) = __builtin_convertvector(acc[i][j], T4);
#pragma unroll
        for (int r = 0; r < 16; r += kRowsAtOnce) {
            const int row = r + lane / kLanes, at = lane % kLanes * kEach;
            const v4i x = *reinterpret_cast<const v4i *>(strip + row * kRow + at * int(sizeof(T)));
            const uint32_t om = m + uint32_t(i * 16 + row), on = n + uint32_t(at);
            if (om >= p.a.rows || on >= p.b.rows) continue;
            T *const to = static_cast<T *>(p.out) + size_t(om) * p.out_stride + on;
            if (on + kEach <= p.b.rows) {
                *reinterpret_cast<v4i_any *>(to) = x;
            } else {
                T e[kEach];
                __builtin_memcpy(e, &x, 16);
#pragma unroll
                for (int l = 0; l < kEach; ++l)
                    if (on + l < p.b.rows) to[l] = e[l];
            }
        }
    }
}

template <bool EXACT, int SC, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_fp8_tile(MatmulArgs p, uint32_t m_tiles, uint32_t n_tiles, bool by_n, bool direct16) {
    extern __shared__ uint8_t smem[];
    constexpr int kWaves = WM * WN, kRows = TM + TN, kGroups = kRows / 8 / kWaves, MT = TM / WM / 16, NT = TN / WN / 16, kEach = (kGroups + MT - 1) / MT;
    constexpr uint32_t kBuffer = kRows * kScaleBlock, kScales = 64 * kWaves;
    static_assert(kWaves * kStripBytes<float, TN / WN> <= int(2 * kBuffer), "strips of all waves at once");
    static_assert(kRows <= 64 * kWaves && kRows % (8 * kWaves) == 0, "a thread to a row's scale, whole groups of eight rows to a wave");
    // Tiles of one strip follow each other on one XCD (workgroups go to the eight in turn), so that they find it in that one's L2.
    uint32_t tm, tn;
    {
        const uint32_t xcd = blockIdx.x & 7u, i = blockIdx.x >> 3;
        if (by_n) { tn = i / m_tiles * 8u + xcd; tm = i % m_tiles; }
        else { tm = i / n_tiles * 8u + xcd; tn = i % n_tiles; }
        if (tm >= m_tiles || tn >= n_tiles) return;
    }
    const uint32_t m0 = tm * TM, n0 = tn * TN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), col = lane & 15, g = lane >> 4;
    const uint32_t blocks = (p.dim + kScaleBlock - 1) / kScaleBlock;
    const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) uint8_t *)smem));
    float *const scales = reinterpret_cast<float *>(smem + 2 * kBuffer);

    // Of the rows of a and, after them, of b, wave w loads groups w, w + kWaves, ...: lane l row l / 8 of the group, run (l % 8) ^ (l / 8).
    // (Rows past the end are the last one: their results are not stored.)
    const uint8_t *const a0 = p.a.codes + size_t(m0) * p.a.stride, *const b0 = p.b.codes + size_t(n0) * p.b.stride;
    const uint32_t run16 = uint32_t((lane & 7) ^ (lane >> 3)) * 16u;
    uint32_t offset[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const uint32_t row = uint32_t((i * kWaves + wave) * 8 + (lane >> 3));
        const bool of_a = row < uint32_t(TM);
        const uint32_t r = of_a ? min(row, p.a.rows - 1 - m0) : min(row - TM, p.b.rows - 1 - n0);
        offset[i] = r * uint32_t(of_a ? p.a.stride : p.b.stride) + run16;
    }
    const uint32_t whole = direct16 ? p.dim / kScaleBlock : 0u;      // blocks that go to LDS past the registers: the first ones
    auto load_group = [&](uint32_t k, uint32_t buffer, int i) {
        const uint32_t group = uint32_t(i * kWaves + wave);
        load16_to_lds(lds0 + buffer * kBuffer + group * 1024u, (group * 8 < TM ? a0 : b0) + size_t(k) * kScaleBlock, offset[i]);
    };
    auto copy_groups = [&](uint32_t k, uint32_t buffer) {
#pragma unroll 1
        for (int i = 0; i < kGroups; ++i) {
            const uint32_t group = uint32_t(i * kWaves + wave), row = group * 8 + uint32_t(lane >> 3);
            const uint8_t *at = row < uint32_t(TM) ? a0 + size_t(min(row, p.a.rows - 1 - m0)) * p.a.stride : b0 + size_t(min(row - TM, p.b.rows - 1 - n0)) * p.b.stride;
            *reinterpret_cast<v4i *>(smem + buffer * kBuffer + group * 1024u + lane * 16) = codes16(at, k * kScaleBlock + run16, p.dim);
        }
    };
    // A thread to a row's scale; threads beyond the rows load the last one's and put it where nobody looks.
    const uint32_t t = threadIdx.x;
    const bool scale_a = t < uint32_t(TM);
    const size_t scale_at = scale_a ? size_t(min(m0 + t, p.a.rows - 1)) * p.a.scale_stride
                                    : size_t(min(n0 + min(t, uint32_t(kRows - 1)) - TM, p.b.rows - 1) >> p.b.group_shift) * p.b.scale_stride;
    const void *const scale_of_row = scale_a ? p.a.scales : p.b.scales;
    auto load_scale = [&](uint32_t k) -> uint32_t {
        if (SC == kScaleBytes) return static_cast<const uint8_t *>(scale_of_row)[scale_at + k];
        return static_cast<const uint32_t *>(scale_of_row)[scale_at + k];
    };
    auto put_scale = [&](uint32_t x, uint32_t buffer) {
        scales[buffer * kScales + t] = EXACT && SC == kScaleBytes ? e8_value(x) : __uint_as_float(x);
    };

    const int wm = wave % WM * (TM / WM), wn = wave / WM * (TN / WN);
    v4f acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0, 0, 0, 0};
    // (rows of a tile of 16 start at a multiple of 8, so a lane's place within them decides the swap)
    const uint32_t lo = uint32_t(col) * kScaleBlock + uint32_t(g ^ (col & 7)) * 16u, hi = uint32_t(col) * kScaleBlock + uint32_t((g + 4) ^ (col & 7)) * 16u;

    // (Straight-line code, with loads of the next block or without: across a branch the compiler moves products behind the
    // wait for those loads.)
    auto multiply = [&](uint32_t k, uint32_t buffer, auto loads) {
        const uint8_t *const ca = smem + buffer * kBuffer + wm * kScaleBlock, *const cb = smem + buffer * kBuffer + (TM + wn) * kScaleBlock;
        const float *const sa = scales + buffer * kScales + wm, *const sb = scales + buffer * kScales + TM + wn;
        Operand<EXACT> y[NT];
        int ys[NT];
        v4f yf[NT];
        // (a wave's rows of b lie in one group)
        uint32_t power = kUnitScale;
        const float shared = SC == kScaleTiles ? shared_scale(__uint_as_float(uint32_t(__builtin_amdgcn_readfirstlane(__float_as_int(sb[0])))), power) : 1.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float s = __uint_as_float(power << 23);
            ys[j] = int(power);
            if (SC == kScaleBytes) { s = sb[j * 16 + col]; ys[j] = __float_as_int(s); }
            if (SC == kScaleRows) yf[j] = *reinterpret_cast<const v4f *>(sb + j * 16 + 4 * g);
            y[j].set(*reinterpret_cast<const v4i *>(cb + j * 16 * kScaleBlock + lo), *reinterpret_cast<const v4i *>(cb + j * 16 * kScaleBlock + hi), s);
        }
        // (the next 16 rows' codes are requested before the products of these, and no sooner: the tile fills the registers)
        v4i xlo = *reinterpret_cast<const v4i *>(ca + lo), xhi = *reinterpret_cast<const v4i *>(ca + hi);
        float xs = sa[col];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const float s = xs;
            Operand<EXACT> x;
            x.set(xlo, xhi, SC == kScaleBytes ? s : 1.0f);
            if (i + 1 < MT) {
                xlo = *reinterpret_cast<const v4i *>(ca + (i + 1) * 16 * kScaleBlock + lo);
                xhi = *reinterpret_cast<const v4i *>(ca + (i + 1) * 16 * kScaleBlock + hi);
                xs = sa[(i + 1) * 16 + col];
            }
            // the next block's loads one by one, between products: all at once they hold up the wave until the last is accepted
            if constexpr (decltype(loads)::value) {
#pragma unroll
                for (int l = i * kEach; l < (i + 1) * kEach && l < kGroups; ++l) load_group(k + 1, buffer ^ 1u, l);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (SC == kScaleBytes) {
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = block_product(y[j], x, acc[i][j], ys[j], __float_as_int(s));
            } else {
                const float tile = s * shared;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const v4f part = block_product(y[j], x, v4f{0, 0, 0, 0}, ys[j], kUnitScale);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] = SC == kScaleTiles ? fmaf(part[r], tile, acc[i][j][r]) : fmaf(part[r] * s, yf[j][r], acc[i][j][r]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (whole != 0) {
#pragma unroll
        for (int i = 0; i < kGroups; ++i) load_group(0, 0, i);
        put_scale(load_scale(0), 0);
    }
    uint32_t k = 0;
    for (; k + 1 < whole; ++k) {
        wait_loads();
        __syncthreads();
        const uint32_t next_scale = load_scale(k + 1);
        multiply(k, k & 1u, IntC<1>{});
        put_scale(next_scale, (k & 1u) ^ 1u);
    }
    for (; k < blocks; ++k) {      // the last whole block, and one that ends early; all of them where rows start anywhere
        if (k >= whole) {
            __syncthreads();
            copy_groups(k, k & 1u);
            put_scale(load_scale(k), k & 1u);
        }
        wait_loads();
        __syncthreads();
        multiply(k, k & 1u, IntC<0>{});
    }
    // Sixteen rows of a wave's results at a time go through LDS, so that they leave in runs of whole cache lines.
    __syncthreads();
    if (EXACT) store_strips<float, TN / WN, MT, NT>(p, acc, smem + wave * kStripBytes<float, TN / WN>, m0 + wm, n0 + wn, lane);
    else if (p.out_type == kF16) store_strips<f16, TN / WN, MT, NT>(p, acc, smem + wave * kStripBytes<f16, TN / WN>, m0 + wm, n0 + wn, lane);
    else store_strips<bf16, TN / WN, MT, NT>(p, acc, smem + wave * kStripBytes<bf16, TN / WN>, m0 + wm, n0 + wn, lane);
}

template <bool EXACT, int SC, int TM, int TN, int WM, int WN>
static hipError_t tile(const MatmulArgs &a, hipStream_t s) {
    static_assert(SC != kScaleTiles || (kScaleBlock % (TN / WN) == 0 && TN % (TN / WN) == 0), "a wave's rows of b lie in one group");
    const uint32_t mt = (a.a.rows + TM - 1) / TM, nt = (a.b.rows + TN - 1) / TN;
    const bool by_n = nt >= mt;
    const uint64_t grid = by_n ? (uint64_t(nt) + 7) / 8 * 8 * mt : (uint64_t(mt) + 7) / 8 * 8 * nt;
    // 16 bytes at a time past the registers: rows at multiples of 16 bytes, and a tile's offsets in 32 bits
    const bool direct16 = ((uintptr_t(a.a.codes) | uintptr_t(a.b.codes) | a.a.stride | a.b.stride) & 15) == 0 && a.a.stride < (1u << 23) && a.b.stride < (1u << 23);
    if ((grid * (64 * WM * WN)) >> 32) return hipErrorInvalidConfiguration;      // (a result of 130 GB, or a narrow one of a billion columns)
    const auto kernel = k_fp8_tile<EXACT, SC, TM, TN, WM, WN>;
    if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), tile_lds<TM, TN, WM, WN>()); e != hipSuccess) return e;
    return launch(kernel, uint32_t(grid), 64 * WM * WN, tile_lds<TM, TN, WM, WN>(), s, a, mt, nt, by_n, direct16);
}

template <bool EXACT, int SC>
static hipError_t matmul(const MatmulArgs &a, hipStream_t s) {
    if (a.a.rows <= 16 && a.dim >= 16) {
        // Sixteen rows to a wave leave waves without any.  One row against 4096 and 16384 of 1536: 9 us either way; 65536: 22 shared out, 19 with a
        // wave to sixteen.  In tiles of 64, sixteen rows of a against 100000 take 31 us where these take 33, one row 36 where it takes 28.
        const bool few = a.b.rows < 256 * 4 * 16;
        if (size_t(a.a.rows) * direct_row(a.dim) <= kDirectLds) return few ? direct<EXACT, SC == kScaleBytes, true>(a, s) : direct<EXACT, SC == kScaleBytes, false>(a, s);
        // More of a than that leaves a compute unit one workgroup or two: as long as none waits for its turn.  (8 rows of 16384 against 4000, 8000
        // and 16000 into bfloat16: 30, 55 and 109 us; in tiles 65, 65 and 93.)
        const size_t lds = direct_lds(a.a.rows, a.dim);
        if (lds <= kMostLds && (a.b.rows + 15) / 16 <= 256 * (kMostLds / lds)) return direct<EXACT, SC == kScaleBytes, true>(a, s);
    }
    // Up to 32 rows of a into floats: a tile that does not convert rows that are not there.  (32 by 77777 of 1000 22 us, by 1M of 1536 343; in tiles of 64
    // 27 and 371.  Into bfloat16 it is 23 and 24, 303 and 319, but 30 and 27 by 100000 of 1536.)
    if constexpr (EXACT) {
        if (a.a.rows <= 32) return tile<EXACT, SC, 32, 128, 1, 4>(a, s);
    }
    // A CU's time: the tiles it gets, which come in rounds of as many as it holds at a time, times what one takes.  The rates come from 26 sizes of 65 to 6000 rows
    // by 1500 to 200000, of 384 to 4096, each scale kind: at three rounds and more 128 x 128 has 0.88 of the rate of 256 x 256 into floats on the mean
    // (0.79 to 1.10), 0.86 into 16 bits (0.58 to 1.00), 64 x 128 0.75 and 0.76, 64 x 64 0.70 and 0.61; those taken lose least over all sizes, 1.5 and
    // 2.3 % of the best tile's time.  6000 by 6000 of 4096 into floats: 321 us in tiles of 256, 282 of 128, 346 of 64 x 128; 1024 by 100000 of 1536 333, 366 and 444
    // of 64.  A started round costs a whole one: 64 by 100000 takes 28 us in tiles of 64, 32 of 64 x 128, by 77777 of 1000 29 and 26.  Where few tiles fill the card
    // the small ones win: 300 by 3000 36, 18 and 10 us, 64 by 20000 18 in tiles of 64 x 128 and 14 of 64.  (Float scales and bfloat16 operands of
    // a 256 x 256 tile do not fit the registers.)
    auto tiles = [&](uint32_t tm, uint32_t tn) { return uint64_t((a.a.rows + tm - 1) / tm) * ((a.b.rows + tn - 1) / tn); };
    auto time = [&](uint32_t tm, uint32_t tn, uint32_t held, double rate) {
        const uint64_t n = tiles(tm, tn), one = 256 * held;
        return double(n <= one ? (n + 255) / 256 : (n + one - 1) / one * held) * tm * tn / rate;
    };
    const double l = EXACT && SC != kScaleBytes ? HUGE_VAL : time(256, 256, 1, 1.0), m = time(128, 128, 2, EXACT ? 0.88 : 0.8), sm = time(64, 64, 4, EXACT ? 0.75 : 0.58);
    const double wide = tiles(64, 128) < 512 ? HUGE_VAL : time(64, 128, 3, EXACT ? 0.78 : 0.72);
    if constexpr (!EXACT || SC == kScaleBytes) {
        if (l <= m && l <= sm && l <= wide) return tile<EXACT, SC, 256, 256, 2, 4>(a, s);
    }
    if (m <= sm && m <= wide) return tile<EXACT, SC, 128, 128, 2, 2>(a, s);
    return wide <= sm ? tile<EXACT, SC, 64, 128, 2, 2>(a, s) : tile<EXACT, SC, 64, 64, 2, 2>(a, s);
}
template <bool EXACT>
static hipError_t matmul_as(const MatmulArgs &a, int scale_type, hipStream_t s) {
    if (scale_type == kScaleE8M0) return matmul<EXACT, kScaleBytes>(a, s);
    return a.b.group_shift == 0 ? matmul<EXACT, kScaleRows>(a, s) : matmul<EXACT, kScaleTiles>(a, s);
}
hipError_t launch_fp8_matmul(const MatmulArgs &a, int scale_type, hipStream_t s) {
    return a.out_type == kF32 ? matmul_as<true>(a, scale_type, s) : matmul_as<false>(a, scale_type, s);
}

}  // namespace tv
