// Re-scoring: a query against the 8-bit rows of its own candidate slots, and the k best of them in order.
//
// score = sum over blocks of scale * (sum over the block of q * code), in 64 bits, rounded once: candidates of one query lie close
// together, and their order must not depend on the order of the additions.  Bound by the gather of whole rows; the 64-bit
// multiply-adds (at the rate of 32-bit ones) and the two conversions before each take a third of that.  1024 queries, 100
// candidates each of 1M rows of 1536: 44 us, 3.6 TB/s, where a bare gather of those rows takes 26; one query 12 us.
#include "tv_device.h"
#include "tv_ops.h"

namespace tv {

constexpr uint32_t kPair = 2;                // candidates that half a wave scores at a time, against one reading of the query
constexpr uint32_t kStep = 512, kSteps = 3;  // coordinates that half a wave covers with 16 a lane; steps whose codes are requested at once
constexpr uint32_t kMostSorts = 1 << 20;     // workgroups of a launch: a grid of 2^32 threads is not allowed
constexpr uint32_t kRanked = 256;            // candidates whose places are counted; more are sorted
constexpr uint32_t kMostEach = 512;          // candidates of a workgroup
constexpr uint32_t kAbsent = ~0u;
constexpr int kBestThreads = 1024;

template <bool E8>
__device__ __forceinline__ uint32_t scale_bits(const Rows8 &r, size_t at) {
    return E8 ? uint32_t(static_cast<const uint8_t *>(r.scales)[at]) : static_cast<const uint32_t *>(r.scales)[at];
}
template <bool E8>
__device__ __forceinline__ double scale_value(uint32_t bits) {
    if (!E8) return double(__uint_as_float(bits));
    return bits == 255u ? __longlong_as_double(0x7ff8000000000000ll) : __hiloint2double(int((bits - 127u + 1023u) << 20), 0);
}

// The key that sorts a candidate: score falling, slot rising; 0 where there is none.  NaN scores go behind -infinity.
__device__ __forceinline__ uint64_t candidate_key(float s, uint32_t slot) {
    return s == s ? sort_key(s, slot) : uint64_t(((0x7fffffffu - slot) << 1) | 1u);
}
__device__ __forceinline__ void write_best(const RescoreArgs &p, uint32_t q, uint32_t place, uint64_t key) {
    float s = -__int_as_float(0x7f800000);
    int64_t slot = -1;
    if (key != 0ull) {
        uint32_t at;
        sort_unkey(key, s, at);
        if (uint32_t(key >> 32) == 0u) s = __int_as_float(0x7fc00000);
        slot = int64_t(at);
    }
    p.out_scores[size_t(q) * p.k + place] = s;
    p.out_slots[size_t(q) * p.k + place] = slot;
}
// The candidates whose keys lie in LDS to their places: as many keys above, or equal and earlier.
__device__ __forceinline__ void write_ranked(const RescoreArgs &p, uint32_t q, const uint64_t *key) {
    for (uint32_t i = threadIdx.x; i < p.m; i += blockDim.x) {
        const uint64_t mine = key[i];
        uint32_t place = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < p.m; ++j) place += uint32_t(key[j] > mine || (key[j] == mine && j < i));
        if (place < p.k) write_best(p, q, place, mine);
    }
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double plus_moved(double v) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, false);
    return v + __hiloint2double(hi, lo);
}
// The sum over half a wave, in its last lane.
__device__ __forceinline__ double half_wave_sum(double v) {
    v = plus_moved<0x111, 0xf>(v);      // row_shr 1, 2, 4, 8
    v = plus_moved<0x112, 0xf>(v);
    v = plus_moved<0x114, 0xf>(v);
    v = plus_moved<0x118, 0xf>(v);
    return plus_moved<0x142, 0xa>(v);   // row_bcast 15 into rows 1 and 3
}

// A workgroup to `each` candidates of a query.  WHOLE: those are all of them, and it puts them in order too.
template <typename T, bool E8, bool WHOLE, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void k_rescore_scores(RescoreArgs p, uint32_t each) {
    // The query in 64 bits, coordinate step * 512 + lane * 16 + i at (step * 16 + i) * 32 + lane: the lanes of half a wave read neighbours.
    extern __shared__ double query[];
    const uint32_t steps = (p.dim + kStep - 1) / kStep;
    uint32_t *const slots = reinterpret_cast<uint32_t *>(query + steps * kStep);       // kMostEach of them
    uint64_t *const keys = reinterpret_cast<uint64_t *>(slots + kMostEach);            // WHOLE: m of them
    const uint32_t lane = threadIdx.x & 31u, half = threadIdx.x >> 5;
    for (uint32_t q = blockIdx.y; q < p.nq; q += gridDim.y) {
        for (uint32_t i = threadIdx.x; i < steps * kStep; i += uint32_t(THREADS)) {
            const double x = i < p.dim ? double(float(static_cast<const T *>(p.queries)[size_t(q) * p.q_stride + i])) : 0.0;
            query[i / kStep * kStep + (i & 15u) * 32u + i / 16u % 32u] = x;
        }
        const uint32_t first = blockIdx.x * each, end = min(first + each, p.m);
        for (uint32_t i = threadIdx.x; first + i < end; i += uint32_t(THREADS)) {
            const int64_t slot = p.slots[size_t(q) * p.slot_stride + first + i];
            slots[i] = uint64_t(slot) < uint64_t(p.rows.rows) ? uint32_t(slot) : kAbsent;
        }
        __syncthreads();
        // Pair after pair, kSteps steps at a time; what comes next is requested before this is multiplied.
        struct Place { uint32_t c, step; };
        struct Part {
            v4i codes[kPair][kSteps];
            uint32_t scale[kPair];       // of block l % 16 of the part, in lane l
        };
        const auto load = [&](Part &x, const Place &at) {
            if (at.c >= end) return;
#pragma unroll
            for (uint32_t j = 0; j < kPair; ++j) {
                // (an absent candidate, and one past the end, reads row 0, where there is one: its sum is not used)
                const uint32_t slot = at.c + j < end ? slots[at.c + j - first] : kAbsent;
                const size_t r = slot == kAbsent ? 0 : slot;
                if (p.rows.rows == 0) continue;
                const uint8_t *const row = p.rows.codes + r * p.rows.stride;
                const size_t scales = (r >> p.rows.group_shift) * p.rows.scale_stride;
#pragma unroll
                for (uint32_t s = 0; s < kSteps; ++s) {
                    if (at.step + s >= steps) break;
                    // (past the row's end its last 16 codes: against zeros of the query, or moved to their place below)
                    const uint32_t c = (at.step + s) * kStep + lane * 16u;
                    x.codes[j][s] = p.dim >= 16u ? *reinterpret_cast<const v4i_any *>(row + min(c, p.dim - 16u)) : codes16(row, c, p.dim);
                }
                x.scale[j] = scale_bits<E8>(p.rows, scales + min(at.step * (kStep / kScaleBlock) + (lane & 15u), (p.dim - 1) / kScaleBlock));
            }
        };
        double sum[kPair] = {};
        const auto multiply = [&](const Part &x, const Place &at) {
#pragma unroll
            for (uint32_t s = 0; s < kSteps; ++s) {
                if (at.step + s >= steps) break;
                const double *const from = query + (at.step + s) * kStep + lane;
                double part[kPair] = {};
                v4i codes[kPair];
#pragma unroll
                for (uint32_t j = 0; j < kPair; ++j) codes[j] = x.codes[j][s];
                if (p.dim % 16u != 0u && p.dim >= 16u && at.step + s + 1 == steps) {
                    const uint32_t c = (at.step + s) * kStep + lane * 16u;
#pragma unroll
                    for (uint32_t j = 0; j < kPair; ++j) codes[j] = bytes_down(codes[j], c - min(c, p.dim - 16u));
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const double q0 = from[(w * 4 + 0) * 32], q1 = from[(w * 4 + 1) * 32], q2 = from[(w * 4 + 2) * 32], q3 = from[(w * 4 + 3) * 32];
#pragma unroll
                    for (uint32_t j = 0; j < kPair; ++j) {
                        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes[j][w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes[j][w], true);
                        part[j] = fma(double(lo[0]), q0, part[j]);
                        part[j] = fma(double(lo[1]), q1, part[j]);
                        part[j] = fma(double(hi[0]), q2, part[j]);
                        part[j] = fma(double(hi[1]), q3, part[j]);
                    }
                }
#pragma unroll
                for (uint32_t j = 0; j < kPair; ++j) sum[j] = fma(part[j], scale_value<E8>(__shfl(x.scale[j], int(s * (kStep / kScaleBlock) + lane / 8u), 32)), sum[j]);
            }
        };
        const auto finish = [&](const Place &at) {
#pragma unroll
            for (uint32_t j = 0; j < kPair; ++j) {
                const double all = half_wave_sum(sum[j]);
                sum[j] = 0.0;
                if (lane != 31u || at.c + j >= end) continue;
                const uint32_t slot = slots[at.c + j - first];
                const uint64_t key = slot == kAbsent ? 0ull : candidate_key(float(all), slot);
                if (WHOLE) keys[at.c + j] = key;
                else p.keys[size_t(q) * p.m + at.c + j] = key;
            }
        };
        Place here{first + half * kPair, 0}, next;
        Part even, odd;
        load(even, here);
        const auto turn = [&](const Part &now, Part &then) {
            next = Place{here.c, here.step + kSteps};
            if (next.step >= steps) next = Place{here.c + (THREADS / 32) * kPair, 0};
            load(then, next);
            multiply(now, here);
            if (next.step == 0) finish(here);
            here = next;
        };
        while (here.c < end) {
            turn(even, odd);
            if (here.c >= end) break;
            turn(odd, even);
        }
        __syncthreads();
        if (WHOLE) {
            write_ranked(p, q, keys);
            __syncthreads();
        }
    }
}

// The k largest keys of a query, in order.
__global__ __launch_bounds__(kBestThreads) void k_rescore_best(RescoreArgs p, uint32_t size) {
    extern __shared__ uint64_t key[];        // size: m, or the power of two not below it
    for (uint32_t q = blockIdx.x; q < p.nq; q += gridDim.x) {
        for (uint32_t i = threadIdx.x; i < size; i += blockDim.x) key[i] = i < p.m ? p.keys[size_t(q) * p.m + i] : 0ull;
        if (p.m <= kRanked) {
            __syncthreads();
            write_ranked(p, q, key);
            __syncthreads();
            continue;
        }
        for (uint32_t run = 2; run <= size; run <<= 1) {
            for (uint32_t step = run >> 1; step > 0; step >>= 1) {
                __syncthreads();
                for (uint32_t i = threadIdx.x; i < size / 2; i += blockDim.x) {
                    const uint32_t lo = 2 * i - (i & (step - 1)), hi = lo + step;
                    const uint64_t x = key[lo], y = key[hi];
                    if ((x < y) == ((lo & run) == 0)) { key[lo] = y; key[hi] = x; }
                }
            }
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < p.k; i += blockDim.x) write_best(p, q, i, key[i]);
        __syncthreads();
    }
}

static size_t rescore_lds(size_t dim) { return (dim + kStep - 1) / kStep * kStep * sizeof(double) + kMostEach * 4; }
// One launch where a workgroup to a query is enough: for few queries, few candidates (rows of 1536; one query, 128 candidates 16 us against
// 17 in two launches, 200 candidates 22 against 17; 255 queries, 200 candidates 30 against 34).
static bool one_launch(size_t nq, size_t m, size_t dim) { return m <= (nq >= 128 ? kRanked : 128u) && rescore_lds(dim) + m * 8 <= 65536; }
// Sixteen waves to a query as long as a compute unit gets no second one (256 queries, 100 candidates 17 us against 24 with four; 1024
// queries 60 against 42).
static bool many_waves(size_t nq) { return nq <= 256; }
size_t rescore_workspace(size_t nq, size_t m, size_t dim) { return one_launch(nq, m, dim) ? 0 : nq * m * sizeof(uint64_t); }

template <typename T, bool E8>
static hipError_t rescore(const RescoreArgs &a, hipStream_t s) {
    const uint32_t queries = a.nq < 65535u ? a.nq : 65535u;
    const size_t lds = rescore_lds(a.dim);
    if (one_launch(a.nq, a.m, a.dim)) {
        if (!many_waves(a.nq)) return launch(k_rescore_scores<T, E8, true, 256>, dim3(1, queries), 256, lds + a.m * 8u, s, a, a.m);
        return launch(k_rescore_scores<T, E8, true, 1024>, dim3(1, queries), 1024, lds + a.m * 8u, s, a, a.m);
    }
    uint32_t each = 256 / 32 * kPair;
    while (each < a.m && each < kMostEach && uint64_t(a.nq) * ((a.m + each - 1) / each) > 2048) each *= 2;
    const auto kernel = k_rescore_scores<T, E8, false, 256>;
    if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), lds); e != hipSuccess) return e;
    if (const hipError_t e = launch(kernel, dim3((a.m + each - 1) / each, queries), 256, lds, s, a, each); e != hipSuccess) return e;
    uint32_t size = a.m;
    if (a.m > kRanked)
        for (size = 2; size < a.m;) size <<= 1;
    if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(k_rescore_best), size * 8u); e != hipSuccess) return e;
    return launch(k_rescore_best, a.nq < kMostSorts ? a.nq : kMostSorts, a.m > kRanked ? kBestThreads : 256, size * 8u, s, a, size);
}
template <typename T>
static hipError_t rescore(const RescoreArgs &a, int scale_type, hipStream_t s) {
    return scale_type == kScaleE8M0 ? rescore<T, true>(a, s) : rescore<T, false>(a, s);
}
hipError_t launch_fp8_rescore(const RescoreArgs &a, int q_type, int scale_type, hipStream_t s) {
    if (q_type == kF32) return rescore<float>(a, scale_type, s);
    return q_type == kF16 ? rescore<f16>(a, scale_type, s) : rescore<bf16>(a, scale_type, s);
}

}  // namespace tv
