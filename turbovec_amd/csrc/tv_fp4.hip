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

// A thread to eight coordinates, four neighbours to a block.  Bound by memory: 400000 rows of 1536 floats 482 to 520 us, 5.3 to 5.8 TB/s, an eighth of it written; of bfloat16 286 to 327, 4.8 to 5.4.
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

// (400000 rows of 1536 into bfloat16 291 to 300 us, 5.2 TB/s, four fifths of it written.)
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

// Sixteen bytes of a row's codes from byte k on without the half byte behind an odd dimension.
__device__ __forceinline__ v4i without_half(v4i v, uint32_t k, uint32_t dim) {
    if (dim & 1u) {
        const uint32_t last = (dim + 1u) / 2u - 1u - k;          // (of no word where the row ends elsewhere)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (last / 4u == uint32_t(i)) v[i] &= int(~(0xf0u << (last % 4u * 8u)));
    }
    return v;
}
// The 32 codes from byte k of a row on, those past the row's end zero.
__device__ __forceinline__ v4i codes32(const uint8_t *row, uint32_t k, uint32_t dim) {
    const uint32_t bytes = (dim + 1u) / 2u;
    return k >= bytes ? v4i{0, 0, 0, 0} : without_half(codes16(row, k, bytes), k, dim);
}
// Four scale bytes of a row from block k on, k < blocks; those past the end are 0 (2^-127, of codes that are 0).
__device__ __forceinline__ uint32_t scales4(const uint8_t *row, uint32_t k, uint32_t blocks) {
    uint32_t s = 0;
    if (blocks >= 4u) {
        const uint32_t at = min(k, blocks - 4u);
        __builtin_memcpy(&s, row + at, 4);
        return s >> (8u * (k - at));
    }
    for (uint32_t i = 0; k + i < blocks; ++i) s |= uint32_t(row[k + i]) << (8 * i);
    return s;
}
__device__ __forceinline__ v8i operand4(v4i v) { return v8i{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

__device__ __forceinline__ void store_out4(void *out, size_t at, float v, int type) {
    if (type == kF32) static_cast<float *>(out)[at] = v;
    else if (type == kF16) static_cast<f16 *>(out)[at] = f16(v);
    else static_cast<bf16 *>(out)[at] = bf16(v);
}

// Up to sixteen rows of a: bound by reading b once.  A wave streams 16 rows of b from memory into registers, STEPS steps of 128 coordinates while those
// before are multiplied, and goes on to its next 16 rows without a pause; a lies in LDS, and comes there behind the first of b.  Where there are few rows of b (SPLIT), the waves of
// a workgroup share 16 rows, each taking every WAVES-th turn, and their sums are added in the waves' order.
constexpr size_t kDirect4Lds = 64 << 10, kMostLds4 = 160 << 10;

__host__ __device__ inline uint32_t direct4_row(uint32_t dim) { return (dim + 127u) / 128u * 64u + 16u; }     // (rows of a a few banks apart)
inline size_t direct4_lds(uint32_t rows, uint32_t dim, int waves) { return size_t(rows) * direct4_row(dim) + (dim + 127) / 128 * 64 + size_t(waves) * 64 * 16; }

template <bool SPLIT, int WAVES, int STEPS>
__global__ __launch_bounds__(64 * WAVES, 4) void k_fp4_direct(Matmul4Args p) {
    extern __shared__ uint8_t smem[];
    constexpr int kThreads = 64 * WAVES;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const uint32_t blocks = (p.dim + 31u) / 32u, steps = (p.dim + 127u) / 128u, whole = p.dim / 128u, bytes = (p.dim + 1u) / 2u, row_bytes = direct4_row(p.dim), m = p.a.rows;
    uint32_t *const a_scales = reinterpret_cast<uint32_t *>(smem + m * row_bytes);       // [step][16]: a byte for each block of the step
    v4f *const sums = reinterpret_cast<v4f *>(a_scales + steps * 16);                    // SPLIT: [wave][lane]
    // (rows past the end are the last one: their results are not stored)
    const uint8_t *const a = smem + min(uint32_t(col), m - 1) * row_bytes + g * 16;

    const uint32_t tiles = (p.b.rows + 15) / 16, turns = (steps + STEPS - 1) / STEPS;
    const uint32_t tile_stride = SPLIT ? gridDim.x : gridDim.x * WAVES, turn_stride = SPLIT ? WAVES : 1, first_turn = SPLIT ? wave : 0;
    struct Place {
        uint32_t tile, turn;
        const uint8_t *codes, *scales;
    };
    auto go_to = [&](Place &at, uint32_t tile) {
        const uint32_t row = min(tile * 16u + uint32_t(col), p.b.rows - 1);
        at = Place{tile, first_turn, p.b.codes + size_t(row) * p.b.stride, p.b.scales + size_t(row) * p.b.scale_stride};
    };
    struct Turn {
        v4i codes[STEPS];
        uint32_t scales[STEPS];
    };
    auto load = [&](Turn &s, const Place &at) {
        if (at.tile >= tiles || at.turn >= turns) return;
        const uint32_t first = at.turn * STEPS;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) s.codes[i] = *reinterpret_cast<const v4i_any *>(at.codes + min((first + i) * 64u + uint32_t(g) * 16u, bytes - 16u));
        if (first * 4u + sizeof(s.scales) <= blocks) {
            __builtin_memcpy(s.scales, at.scales + first * 4u, sizeof(s.scales));
        } else {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) s.scales[i] = (first + i) * 4u < blocks ? scales4(at.scales, (first + i) * 4u, blocks) : 0u;
        }
    };
    v4f acc = v4f{0, 0, 0, 0};
    auto step = [&](uint32_t k, const v4i &y, uint32_t ys) {
        const v4i x = *reinterpret_cast<const v4i *>(a + k * 64u);
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand4(x), operand4(y), acc, 4, 4, 0, int(a_scales[k * 16 + col] >> (8 * g)), 0, int(ys >> (8 * g)));
    };
    auto multiply = [&](const Turn &s, const Place &at) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const uint32_t k = at.turn * STEPS + i, from = k * 64u + uint32_t(g) * 16u;
            if (k < whole) step(k, s.codes[i], s.scales[i]);
            else if (k < steps)               // (the row ends in this step: what was loaded are its last 16 bytes)
                step(k, without_half(bytes_down(s.codes[i], from - min(from, bytes - 16u)), from, p.dim), s.scales[i]);
        }
    };
    auto finish = [&](const Place &at) {
        if (SPLIT) {
            sums[threadIdx.x] = acc;
            __syncthreads();
            if (wave != 0) return;
#pragma unroll
            for (int w = 1; w < WAVES; ++w) acc += sums[w * 64 + lane];
        }
        const uint32_t n = at.tile * 16u + uint32_t(col);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (uint32_t(4 * g + r) < m && n < p.b.rows) store_out4(p.out, size_t(4 * g + r) * p.out_stride + n, acc[r], p.out_type);
        acc = v4f{0, 0, 0, 0};
    };
    Place here, next;
    Turn even, odd;
    go_to(here, SPLIT ? blockIdx.x : blockIdx.x * WAVES + wave);
    load(even, here);
    // a, eight runs to a thread on their way at a time, behind the first rows of b.
    constexpr int kRuns = 8;
    const uint32_t a_runs = m * steps * 4u;
    for (uint32_t first = threadIdx.x; first < a_runs; first += kRuns * kThreads) {
        v4i run[kRuns];
        uint32_t r[kRuns], c[kRuns];
#pragma unroll
        for (int l = 0; l < kRuns; ++l) {
            const uint32_t i = first + uint32_t(l * kThreads);
            r[l] = i / (steps * 4u);
            c[l] = i % (steps * 4u) * 16u;
            if (i < a_runs) run[l] = *reinterpret_cast<const v4i_any *>(p.a.codes + size_t(r[l]) * p.a.stride + min(c[l], bytes - 16u));
        }
#pragma unroll
        for (int l = 0; l < kRuns; ++l)
            if (first + uint32_t(l * kThreads) < a_runs) *reinterpret_cast<v4i *>(smem + r[l] * row_bytes + c[l]) = without_half(bytes_down(run[l], c[l] - min(c[l], bytes - 16u)), c[l], p.dim);
    }
    for (uint32_t first = threadIdx.x; first < steps * 16u; first += 4 * kThreads) {
        uint32_t four[4];
#pragma unroll
        for (int l = 0; l < 4; ++l)
            if (const uint32_t i = first + uint32_t(l * kThreads); i < steps * 16u) four[l] = scales4(p.a.scales + size_t(min(i & 15u, m - 1)) * p.a.scale_stride, (i >> 4) * 4u, blocks);
#pragma unroll
        for (int l = 0; l < 4; ++l)
            if (const uint32_t i = first + uint32_t(l * kThreads); i < steps * 16u) a_scales[i] = four[l];
    }
    __syncthreads();
    auto turn = [&](const Turn &now, Turn &then) {
        next = here;
        next.turn += turn_stride;
        if (next.turn >= turns) go_to(next, SPLIT ? tiles : here.tile + tile_stride);
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
template <bool SPLIT, int WAVES, int STEPS>
static hipError_t direct4(const Matmul4Args &a, hipStream_t s) {
    const uint32_t tiles = (a.b.rows + 15) / 16, grid = SPLIT ? tiles : min((tiles + WAVES - 1) / WAVES, 256u * 16u / WAVES);
    const size_t lds = direct4_lds(a.a.rows, a.dim, WAVES);
    const auto kernel = k_fp4_direct<SPLIT, WAVES, STEPS>;
    if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), lds); e != hipSuccess) return e;
    return launch(kernel, grid, 64 * WAVES, lds, s, a);
}

// Many rows of a: a workgroup to a tile of TM rows of a and TN of b, WM x WN waves, each with 32 x 32 x 64 products.  (Those reach 6.2 to 6.6 PFLOP/s on registers
// alone, where the chip's power ends it, 16 x 16 x 128 ones 4.6 to 5.5.)  Stages of 256 coordinates of both, a cache line of 128 bytes a row, come into registers a stage
// ahead, go from there to one half of LDS while the other is multiplied, and so reach the matrix units two stages later.  (Loads past the registers, into a ring
// of stages of 64 bytes a row, take whole lines for half of them: 29 bytes a clock and compute unit where these take 58.)
//
// A row's eight runs of 16 bytes are swapped about by the row's number: lanes that read the same run of neighbouring rows find it in different banks.  A row's eight scale
// bytes lie in LDS as two words, of even and of odd blocks: a lane's four steps find theirs in the bytes of one word, which the instruction picks.
//
// A stage has four steps of 64 coordinates.  Operands of a step are read from LDS while the step before is multiplied; the barrier between two stages
// stands before the last step of the first, whose operands are in registers by then, so that the matrix units have work across it.
constexpr uint32_t kStage4 = 256, kStageBytes4 = kStage4 / 2;
constexpr size_t kMostTileStride4 = size_t(1) << 23;      // a tile's offsets have 32 bits
template <int TM, int TN> constexpr size_t tile4_lds() { return 2 * size_t(TM + TN) * (kStageBytes4 + 8); }
template <typename T, int COLS> constexpr int kStrip4 = 32 * (COLS * int(sizeof(T)) + 16);

// Ways of results to memory: through the L2, past it with eight of a wave's reads from LDS on their way, past it one read and one store after the other.
enum { kThroughL2 = 0, kPastL2 = 1, kPaced = 2 };
// A wave's results, whose lane l holds, of row l % 32 of each tile, columns 8 q + 4 (l / 32) .. + 3, to rows from m on and columns from n on: 32 rows at a time
// through LDS, so that they leave in runs of whole cache lines.
template <typename T, int WAY, int COLS, int MT, int NT>
__device__ __forceinline__ void store_strips4(const Matmul4Args &p, const v16f (&acc)[MT][NT], uint8_t *strip, uint32_t m, uint32_t n, int lane) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int kEach = 16 / int(sizeof(T)), kLanes = COLS / kEach, kRowsAtOnce = 64 / kLanes, kRow = COLS * int(sizeof(T)) + 16;
    const int row32 = lane & 31, half = lane >> 5;
    const bool inside = m + MT * 32 <= p.a.rows && n + COLS <= p.b.rows;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const v4f x = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                *reinterpret_cast<T4 *>(strip + row32 * kRow + (j * 32 + q * 8 + half * 4) * int(sizeof(T))) = __builtin_convertvector(x, T4);
            }
        const uint32_t at = uint32_t(lane % kLanes * kEach), on = n + at;
        const T *const from = reinterpret_cast<const T *>(strip + lane / kLanes * kRow) + at;
        constexpr int kRounds = 32 / kRowsAtOnce, kTogether = kRounds < 8 ? kRounds : 8;
        if constexpr (WAY == kPaced) {
            const uint32_t first = m + uint32_t(i * 32 + lane / kLanes);
            const bool whole = on + kEach <= p.b.rows;
            T *to = static_cast<T *>(p.out) + size_t(first) * p.out_stride + on;
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                if (inside || (whole && first + uint32_t(r * kRowsAtOnce) < p.a.rows))
                    __builtin_nontemporal_store(*reinterpret_cast<const v4i *>(reinterpret_cast<const uint8_t *>(from) + r * kRowsAtOnce * kRow), reinterpret_cast<v4i_any *>(to));
                to += kRowsAtOnce * p.out_stride;
            }
            if (inside || whole || on >= p.b.rows) continue;
#pragma unroll 1
            for (uint32_t r = 0; r < 32 && first + r < p.a.rows; r += kRowsAtOnce) {          // (the last columns, fewer than a lane stores at once)
                const T *const x = reinterpret_cast<const T *>(reinterpret_cast<const uint8_t *>(from) + r * kRow);
                T *const row = static_cast<T *>(p.out) + size_t(first + r) * p.out_stride + on;
#pragma unroll 1
                for (uint32_t l = 0; on + l < p.b.rows; ++l) row[l] = x[l];
            }
            continue;
        }
        if (inside) {          // (a wave waits for eight reads once, not for each of them)
            T *to = static_cast<T *>(p.out) + size_t(m + uint32_t(i * 32 + lane / kLanes)) * p.out_stride + on;
#pragma unroll
            for (int r = 0; r < kRounds; r += kTogether) {
                v4i x[kTogether];
#pragma unroll
                for (int l = 0; l < kTogether; ++l) x[l] = *reinterpret_cast<const v4i *>(reinterpret_cast<const uint8_t *>(from) + (r + l) * kRowsAtOnce * kRow);
#pragma unroll
                for (int l = 0; l < kTogether; ++l) {
                    if constexpr (WAY == kPastL2) __builtin_nontemporal_store(x[l], reinterpret_cast<v4i_any *>(to));
                    else *reinterpret_cast<v4i_any *>(to) = x[l];
                    to += kRowsAtOnce * p.out_stride;
                }
            }
            continue;
        }
#pragma unroll 1
        for (int r = 0; r < 32; r += kRowsAtOnce) {
            const uint32_t om = m + uint32_t(i * 32 + r + lane / kLanes);
            if (om >= p.a.rows || on >= p.b.rows) continue;
            const T *const x = reinterpret_cast<const T *>(reinterpret_cast<const uint8_t *>(from) + r * kRow);
            T *const to = static_cast<T *>(p.out) + size_t(om) * p.out_stride + on;
            if (on + kEach <= p.b.rows) {
                *reinterpret_cast<v4i_any *>(to) = *reinterpret_cast<const v4i *>(x);
            } else {
#pragma unroll 1
                for (uint32_t l = 0; on + l < p.b.rows; ++l) to[l] = x[l];
            }
        }
    }
}

template <typename T, int TM, int TN, int WM, int WN, int HELD, int KS>
__global__ __launch_bounds__(64 * WM * WN * KS, (HELD * KS * WM * WN + 3) / 4) void k_fp4_tile(Matmul4Args p, uint32_t m_tiles, uint32_t n_tiles, uint32_t each_xcd, int way) {
    extern __shared__ uint8_t smem[];
    constexpr int kWaves = WM * WN, kThreads = 64 * kWaves, kRows = TM + TN, kGroups = kRows / 8 / kWaves, MT = TM / WM / 32, NT = TN / WN / 32;
    constexpr uint32_t kBuffer = kRows * kStageBytes4;
    static_assert(TM % (8 * kWaves) == 0 && TN % (8 * kWaves) == 0, "whole groups of eight rows of either side to a wave");
    static_assert(size_t(kWaves) * kStrip4<T, TN / WN> <= tile4_lds<TM, TN>(), "strips of all waves at once");
    // An XCD (workgroups go to the eight in turn) has tiles that follow each other: eight rows of tiles by as many columns as there are, column by column, so that its
    // thirty-two compute units find most of what they read in its L2.
    uint32_t tm, tn;
    {
        const uint32_t id = (blockIdx.x & 7u) * each_xcd + (blockIdx.x >> 3);
        if (id >= m_tiles * n_tiles) return;
        const uint32_t band = id / (8u * n_tiles), in = id % (8u * n_tiles), high = min(8u, m_tiles - band * 8u);
        tm = band * 8u + in % high;
        tn = in / high;
    }
    const uint32_t m0 = tm * TM, n0 = tn * TN;
    const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), wave = all_waves % kWaves, row32 = lane & 31, half = lane >> 5;
    const uint32_t blocks = (p.dim + 31u) / 32u, stages = (p.dim + kStage4 - 1) / kStage4, whole = p.dim / kStage4, bytes = (p.dim + 1u) / 2u;
    // KS groups of waves, with LDS of their own, take every KS-th stage; where a group has one less it multiplies zeros.
    const uint32_t group = uint32_t(all_waves / kWaves), thread = threadIdx.x % kThreads, turns = (stages + KS - 1) / KS;
    auto stage = [&](uint32_t k) { return KS == 1 ? k : k * KS + group; };
    uint8_t *const mine = smem + group * uint32_t(tile4_lds<TM, TN>());
    uint32_t *const scales = reinterpret_cast<uint32_t *>(mine + 2 * kBuffer);                  // [buffer][even or odd blocks][row]

    // Of the rows of a and, after them, of b, wave w has groups of eight w, w + kWaves, ...: lane l row l / 8 of the group, run l % 8.
    // (Rows past the end are the last one: their results are not stored.)
    const uint8_t *const a0 = p.a.codes + size_t(m0) * p.a.stride, *const b0 = p.b.codes + size_t(n0) * p.b.stride;
    const uint32_t run16 = uint32_t(lane & 7) * 16u;
    uint32_t offset[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const uint32_t row = uint32_t((i * kWaves + wave) * 8 + (lane >> 3));
        offset[i] = i * kWaves * 8 < TM ? min(row, p.a.rows - 1 - m0) * uint32_t(p.a.stride) : min(row - TM, p.b.rows - 1 - n0) * uint32_t(p.b.stride);
    }
    v4i held[kGroups];
    // (A run that the row ends in or before is the row's last 16 bytes, for ending() to put right.)
    auto load_group = [&](uint32_t k, auto i) {
        constexpr int I = decltype(i)::value;
        held[I] = *reinterpret_cast<const v4i_any *>((I * kWaves * 8 < TM ? a0 : b0) + (offset[I] + min(stage(k) * kStageBytes4 + run16, bytes - 16u)));
    };
    uint8_t *const my_run = mine + uint32_t(wave) * 1024u + uint32_t(lane >> 3) * kStageBytes4 + uint32_t((lane & 7) ^ (lane >> 3)) * 16u;
    auto put_group = [&](uint32_t k, auto i) {
        constexpr int I = decltype(i)::value;
        *reinterpret_cast<v4i *>(my_run + (k & 1u) * kBuffer + I * kWaves * 1024) = held[I];
    };
    // A thread to the scales of every kThreads-th row.
    constexpr int kScaleRounds = (kRows + kThreads - 1) / kThreads;
    uint64_t held_scales[kScaleRounds];
    const uint8_t *scale_row[kScaleRounds];
    const uint32_t last_eight = blocks >= 8u ? blocks - 8u : 0u;
#pragma unroll
    for (int i = 0; i < kScaleRounds; ++i) {
        const uint32_t row = min(uint32_t(i * kThreads) + thread, uint32_t(kRows - 1));
        scale_row[i] = row < uint32_t(TM) ? p.a.scales + size_t(min(m0 + row, p.a.rows - 1)) * p.a.scale_stride : p.b.scales + size_t(min(n0 + row - TM, p.b.rows - 1)) * p.b.scale_stride;
        // (rows of fewer than eight blocks have one stage)
        held_scales[i] = 0;
        if (blocks < 8u)
            for (uint32_t l = 0; l < blocks; ++l) held_scales[i] |= uint64_t(scale_row[i][l]) << (8 * l);
        if (blocks < 8u) scale_row[i] = a0;
    }
    auto load_scales = [&](uint32_t k) {
#pragma unroll
        for (int i = 0; i < kScaleRounds; ++i) __builtin_memcpy(&held_scales[i], scale_row[i] + min(stage(k) * 8u, last_eight), 8);
    };
    auto put_scales = [&](uint32_t k) {
#pragma unroll
        for (int i = 0; i < kScaleRounds; ++i) {
            const uint32_t row = uint32_t(i * kThreads) + thread, lo = uint32_t(held_scales[i]), hi = uint32_t(held_scales[i] >> 32);
            if (kRows % kThreads != 0 && row >= uint32_t(kRows)) continue;
            uint32_t *const to = scales + (k & 1u) * 2 * kRows + row;
            to[0] = __builtin_amdgcn_perm(hi, lo, 0x06040200u);
            to[kRows] = __builtin_amdgcn_perm(hi, lo, 0x07050301u);
        }
    };
    // The stage that rows end in, as it stands in registers: runs moved down to where they belong, zeros behind the end, scales too (2^-127, of codes that are 0).
    auto ending = [&](uint32_t at) {
        const uint32_t from = at * kStageBytes4 + run16;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) held[i] = without_half(bytes_down(held[i], from - min(from, bytes - 16u)), from, p.dim);
        if (blocks >= 8u) {
#pragma unroll
            for (int i = 0; i < kScaleRounds; ++i) held_scales[i] = at * 8u >= blocks ? 0u : held_scales[i] >> (8u * (at * 8u - min(at * 8u, last_eight)));
        }
    };

    const int wm = wave % WM * (TM / WM), wn = wave / WM * (TN / WN);
    v16f acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    struct Operands {
        v4i a[MT], b[NT];
    };
    struct Scales {
        int a[MT], b[NT];
    };
    const uint8_t *const my_a = mine + (wm + row32) * kStageBytes4, *const my_b = mine + (TM + wn + row32) * kStageBytes4;
    // What goes on between a step's products, in front of each a part: reads of the next step's operands, in the order that it wants them, of the next stage's scales, stores
    // into LDS and loads.  (A wave has its SIMD alone in the largest tiles: between two products it can give a handful of instructions; more of them in one place
    // leave the matrix unit idle.)
    constexpr int kSlots = MT * NT, kReads = MT + NT;
    auto read = [&](Operands &o, uint32_t k, int t, int slot) {
        const uint32_t at = (k & 1u) * kBuffer + uint32_t((2 * t + half) ^ (row32 & 7)) * 16u;
#pragma unroll
        for (int l = 0; l < kReads; ++l) {
            if (l * kSlots / kReads != slot) continue;
            if (l == 0) o.a[0] = *reinterpret_cast<const v4i *>(my_a + at);
            else if (l <= NT) o.b[l - 1] = *reinterpret_cast<const v4i *>(my_b + at + (l - 1) * 32 * kStageBytes4);
            else o.a[l - NT] = *reinterpret_cast<const v4i *>(my_a + at + (l - NT) * 32 * kStageBytes4);
        }
    };
    auto read_scales = [&](Scales &s, uint32_t k, int slot) {
        const int *const from = reinterpret_cast<const int *>(scales) + ((k & 1u) * 2u + uint32_t(half)) * kRows + row32;
#pragma unroll
        for (int l = 0; l < kReads; ++l) {
            if ((l * kSlots + kSlots / 2) / kReads != slot) continue;
            if (l < MT) s.a[l] = from[wm + l * 32];
            else s.b[l - MT] = from[TM + wn + (l - MT) * 32];
        }
    };
    // In three steps' slots, group by group: what is held goes to LDS, and the next stage's takes its place.
    auto pass_on = [&](uint32_t k, int slot) {
        static_for<kGroups>([&](auto l) {
            if ((decltype(l)::value * 3 * kSlots + kSlots / 2) / kGroups != slot) return;
            put_group(k + 1, l);
            load_group(k + 2, l);
        });
        if (slot == 3 * kSlots - 1) {
            put_scales(k + 1);
            load_scales(k + 2);
        }
    };
    auto multiply = [&](const Operands &o, const Scales &s, auto t, auto &&before) {
        constexpr int kByte = decltype(t)::value;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                before(i * NT + j);
                __builtin_amdgcn_sched_barrier(0);
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand4(o.b[j]), operand4(o.a[i]), acc[i][j], 4, 4, kByte, s.b[j], kByte, s.a[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    Operands even, odd;
    Scales sc, sc_next;
    static_for<kGroups>([&](auto i) { load_group(0, i); });
    if (blocks >= 8u) load_scales(0);
    if (stage(0) >= whole) ending(stage(0));
    static_for<kGroups>([&](auto i) {
        put_group(0, i);
        load_group(1, i);
    });
    put_scales(0);
    load_scales(1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
        read(even, 0, 0, i);
        read_scales(sc, 0, i);
    }
#pragma unroll 1
    for (uint32_t k = 0; k < turns; ++k) {
        if (KS == 1 ? k + 1 == whole : stage(k + 1) >= whole) ending(stage(k + 1));      // (where rows end with a stage, nobody looks at the next)
        // (The same for every stage, without a branch: across one the compiler moves products about.  Behind the last stage what is loaded and read is not used.)
        multiply(even, sc, IntC<0>{}, [&](int slot) {
            read(odd, k, 1, slot);
            pass_on(k, slot);
        });
        multiply(odd, sc, IntC<1>{}, [&](int slot) {
            read(even, k, 2, slot);
            pass_on(k, kSlots + slot);
        });
        multiply(even, sc, IntC<2>{}, [&](int slot) {
            read(odd, k, 3, slot);
            pass_on(k, 2 * kSlots + slot);
        });
        __syncthreads();
        multiply(odd, sc, IntC<3>{}, [&](int slot) {
            read(even, k + 1, 0, slot);
            read_scales(sc_next, k + 1, slot);
        });
        sc = sc_next;
    }
    __syncthreads();
    if constexpr (KS > 1) {          // (the groups' sums, added in their order)
        float *const sums = reinterpret_cast<float *>(smem + tile4_lds<TM, TN>());
        constexpr uint32_t kEach = MT * NT * 16;
        if (group != 0) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sums[((group - 1) * kEach + uint32_t((i * NT + j) * 16 + r)) * kThreads + thread] = acc[i][j][r];
        }
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int g = 1; g < KS; ++g)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][j][r] += sums[(uint32_t(g - 1) * kEach + uint32_t((i * NT + j) * 16 + r)) * kThreads + thread];
    }
    uint8_t *const strip = smem + wave * kStrip4<T, TN / WN>;
    if (way == kPaced) store_strips4<T, kPaced, TN / WN, MT, NT>(p, acc, strip, m0 + wm, n0 + wn, lane);
    else if (way == kPastL2) store_strips4<T, kPastL2, TN / WN, MT, NT>(p, acc, strip, m0 + wm, n0 + wn, lane);
    else store_strips4<T, kThroughL2, TN / WN, MT, NT>(p, acc, strip, m0 + wm, n0 + wn, lane);
}

// Results of rows below kStreamDim4 leave past the L2: they would push out what other tiles read there.  (1024 by 98304 of 1536 into floats 134 to 139 us, through it 154; of 2048 177 and 171, 4096 by
// 16384 of 4096 172 and 172, into bfloat16 157 and 148.)  Where the result's rows start in the middle of a cache line and there is little to do between two tiles' results, a wave gives eight stores at a
// time (1000 by 50001 of 768 into floats 55 us and 87, into bfloat16 45 and 64; 1000 by 50000, every other row in the middle of a line, 48 and 53; 1024 by 100001 of 1536 191 and 166, 156 and 136; rows
// at whole lines, 1024 by 98304 of 1536, 152 and 137).
constexpr size_t kLine = 128;
constexpr uint32_t kStreamDim4 = 2048, kPacedDim4 = 1280;
template <typename T, int TM, int TN, int WM, int WN, int HELD, int KS = 1>
static hipError_t tile4(const Matmul4Args &a, hipStream_t s) {
    const uint64_t mt = (a.a.rows + TM - 1) / TM, nt = (a.b.rows + TN - 1) / TN, each_xcd = (mt * nt + 7) / 8;
    if ((each_xcd * 8 * (64 * WM * WN * KS)) >> 32) return hipErrorInvalidConfiguration;      // (a result of hundreds of GB, or a narrow one of a billion columns)
    const bool lines = (a.out_stride * sizeof(T) % kLine | reinterpret_cast<uintptr_t>(a.out) % kLine) == 0;
    const int way = a.dim >= kStreamDim4 ? kThroughL2 : lines || TM < 128 || a.dim >= kPacedDim4 ? kPaced : kPastL2;
    const auto kernel = k_fp4_tile<T, TM, TN, WM, WN, HELD, KS>;
    constexpr size_t kLds = KS * tile4_lds<TM, TN>();
    if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), kLds); e != hipSuccess) return e;
    return launch(kernel, uint32_t(each_xcd * 8), 64 * WM * WN * KS, kLds, s, a, uint32_t(mt), uint32_t(nt), uint32_t(each_xcd), way);
}

// Rows of fewer than 16 bytes, or 8 MB and more apart: a wave to a tile of 16 by 16, its operands read where they lie.  (Bound by its waves, 390 vector instructions for
// 256 results, and half of the time they wait: 1024 by 100000 of 16 into floats 275 us, 1.5 TB/s, one by 1M of 24 64; 64 by 200 of 1536, rows 8 MB apart, 8.2, close together 5.5 in tiles.)
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
        const int xs = block < blocks ? as[block] : 0, ys = block < blocks ? bs[block] : 0;
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand4(x), operand4(y), acc, 4, 4, 0, xs, 0, ys);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t m = m0 + 4u * g + r, n = n0 + col;
        if (m < p.a.rows && n < p.b.rows) static_cast<T *>(p.out)[size_t(m) * p.out_stride + n] = T(acc[r]);
    }
}
template <typename T>
static hipError_t small4(const Matmul4Args &a, hipStream_t s) {
    const uint64_t mt = (a.a.rows + 15u) / 16u, nt = (a.b.rows + 15u) / 16u;
    if (mt * nt * 64u >> 32) return hipErrorInvalidConfiguration;
    return launch(k_fp4_small<T>, uint32_t(mt * nt), 64, 0, s, a, uint32_t(nt));
}

// The tiles, and what one takes a compute unit that holds so many of them, in microseconds: for a stage, in front and behind, and for a byte of the result's type.  Fitted to 56 sizes of 17 to
// 8192 rows by 100 to 1M, of 74 to 8192, into floats and bfloat16.  Of these and 44 others, timed with the tiles as they are now, the tile taken is the fastest or within 6 % of it but for twelve, 28 % at worst (6262
// by 7351 of 768: results whose rows start anywhere cost tiles of 256 more than this knows), 2.0 % on the mean; constants fitted anew to all of them do as well, 1.9 %.  A compute unit's tiles come in rounds of as
// many as it holds, and a started round costs a whole one.
struct TileTime {
    uint32_t tm, tn, held;
    double stage, once, byte;
};
constexpr TileTime kTiles4[] = {{256, 256, 1, 1.44, 4.3, 1.4}, {128, 128, 2, 0.59, 0.34, 0.42}, {64, 64, 4, 0.23, 0.24, 0.14}, {64, 128, 3, 0.39, 0.18, 0.3}, {32, 128, 3, 0.27, 0.33, 0.19}};
static double tile_time4(const TileTime &t, uint32_t m, uint32_t n, uint32_t dim, size_t size) {
    const uint64_t tiles = uint64_t((m + t.tm - 1) / t.tm) * ((n + t.tn - 1) / t.tn), one = 256 * t.held;
    const double each = double(tiles <= one ? (tiles + 255) / 256 : (tiles + one - 1) / one * t.held);
    return each * ((dim + kStage4 - 1) / kStage4 * t.stage + t.once + t.byte * double(size));
}
static int best_tile4(uint32_t m, uint32_t n, uint32_t dim, size_t size, double &time) {
    int best = 0;
    for (int i = 0; i < (m <= 32 ? 5 : 4); ++i)
        if (const double t = tile_time4(kTiles4[i], m, n, dim, size); i == 0 || t < time) {
            best = i;
            time = t;
        }
    return best;
}
template <typename T>
static hipError_t tiled4(const Matmul4Args &a, int tile, hipStream_t s) {
    if (tile == 0) return tile4<T, 256, 256, 2, 2, 1>(a, s);
    if (tile == 1) return tile4<T, 128, 128, 2, 2, 2>(a, s);
    if (tile == 2) return tile4<T, 64, 64, 2, 2, 4>(a, s);
    return tile == 3 ? tile4<T, 64, 128, 1, 4, 3>(a, s) : tile4<T, 32, 128, 1, 4, 3>(a, s);
}

template <typename T>
static hipError_t matmul4(const Matmul4Args &a, hipStream_t s) {
    if (a.a.rows <= 16 && a.dim >= 31) {
        // Sixteen rows to a wave leave waves without any; shared out over four, one row against 4096 to 16384 of 1536 takes 4 us.  (One row against 1M of 1536 141 us, in tiles of 64 165;
        // sixteen against 100000 18 and 20.)  Over eight where a compute unit has two workgroups at most: sixteen rows against 8192 of 8192 13 us and 15 over four, 4096 of 16384 14 and 18;
        // against 14000 of 4096 13 and 11.
        const uint32_t groups = (a.b.rows + 15) / 16;
        const bool few = a.b.rows < 256 * 4 * 16, wide = groups <= 512;
        const size_t lds = direct4_lds(a.a.rows, a.dim, wide ? 8 : 4);
        // (More of a than 64 KB leaves a compute unit one workgroup or two: as long as none waits for its turn.)
        const bool fits = size_t(a.a.rows) * direct4_row(a.dim) <= kDirect4Lds;
        if (fits && !few) return direct4<false, 4, 2>(a, s);
        if (fits || (lds <= kMostLds4 && groups <= 256 * (kMostLds4 / lds))) return wide ? direct4<true, 8, 2>(a, s) : direct4<true, 4, 4>(a, s);
    }
    if (a.dim < 31 || a.a.stride >= kMostTileStride4 || a.b.stride >= kMostTileStride4) return small4<T>(a, s);
    // Few tiles leave compute units idle, and one alone takes in no more than 25 to 50 GB a second: smaller ones, whose stages groups of waves share.  (64 rows against 8192 of 8192 10.9 us so and 14.5 in tiles of
    // 64, 32 against 4096 of 16384 11.4 and 24.6, 17 against 4096 of 4096 5.4 and 8.3, 128 against 4096 of 4096 6.9 and 8.6; two tiles to a compute unit, 64 against 16384 of 8192, 17.3 and 15.8.)
    const uint32_t stages = (a.dim + kStage4 - 1) / kStage4;
    const auto tiles4 = [&](uint32_t tm, uint32_t tn) { return uint64_t((a.a.rows + tm - 1) / tm) * ((a.b.rows + tn - 1) / tn); };
    if (stages >= 8 && tiles4(32, 32) <= 256) return tile4<T, 32, 32, 1, 1, 2, 4>(a, s);
    if (stages >= 6 && tiles4(64, 32) <= 256) return tile4<T, 64, 32, 2, 1, 2, 2>(a, s);
    double whole = 0;
    const int tile = best_tile4(a.a.rows, a.b.rows, a.dim, sizeof(T), whole);
    const uint32_t mt = (a.a.rows + 255) / 256, nt = (a.b.rows + 255) / 256;
    const uint64_t tiles = uint64_t(mt) * nt;
    if (tile == 0 && tiles > 256 && nt >= mt) {
        // The tiles of 256 that start a last round and do not fill it: their columns in a launch of their own, of smaller tiles, where that is less than the round.  (1024 by 100000
        // of 1536 into floats 145 us with it and 151 without, into bfloat16 120 and 126.)
        const uint32_t columns = uint32_t(tiles / 256 * 256 / mt) * 256;
        if (columns < a.b.rows) {
            Matmul4Args first = a, rest = a;
            first.b.rows = columns;
            rest.b = Rows4{a.b.codes + size_t(columns) * a.b.stride, a.b.scales + size_t(columns) * a.b.scale_stride, a.b.stride, a.b.scale_stride, a.b.rows - columns};
            rest.out = static_cast<T *>(a.out) + columns;
            double more = 0;
            const int rest_tile = best_tile4(rest.a.rows, rest.b.rows, a.dim, sizeof(T), more);
            if (tile_time4(kTiles4[0], a.a.rows, columns, a.dim, sizeof(T)) + more + 3.0 < whole) {
                const hipError_t e = tiled4<T>(first, 0, s);
                return e == hipSuccess ? tiled4<T>(rest, rest_tile, s) : e;
            }
        }
    }
    return tiled4<T>(a, tile, s);
}
hipError_t launch_fp4_matmul(const Matmul4Args &a, hipStream_t s) {
    if (a.out_type == kF32) return matmul4<float>(a, s);
    return a.out_type == kF16 ? matmul4<f16>(a, s) : matmul4<bf16>(a, s);
}

}  // namespace tv
