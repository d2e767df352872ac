// Re-scoring: a query against the 8-bit rows of its own candidate slots, and the k best of them in order.
//
// score = sum over blocks of scale * (sum over the block of q * code), in 64 bits, rounded once: candidates of one query lie close
// together, and their order must not depend on the order of the additions.
#include "tv_device.h"
#include "tv_ops.h"

namespace tv {

constexpr int kRescoreThreads = 256;
constexpr uint32_t kMostSorts = 1 << 20;     // workgroups of a launch: a grid of 2^32 threads is not allowed
constexpr uint32_t kRescoreEach = 16;        // candidates of a workgroup

__device__ __forceinline__ double scale_at(const Rows8 &r, uint32_t row, uint32_t block, bool e8) {
    const size_t at = size_t(row >> r.group_shift) * r.scale_stride + block;
    if (!e8) return double(static_cast<const float *>(r.scales)[at]);
    const int e = static_cast<const uint8_t *>(r.scales)[at];
    return e == 255 ? __longlong_as_double(0x7ff8000000000000ll) : __longlong_as_double((long long)(e - 127 + 1023) << 52);
}

// The key that sorts a candidate: score falling, slot rising; 0 where there is none.  NaN scores go behind -infinity.
__device__ __forceinline__ uint64_t candidate_key(float s, uint32_t slot) {
    return s == s ? sort_key(s, slot) : uint64_t(((0x7fffffffu - slot) << 1) | 1u);
}

template <typename T, bool E8>
__global__ __launch_bounds__(kRescoreThreads) void k_rescore_scores(RescoreArgs p) {
    extern __shared__ double query[];        // dim rounded up to 16 values
    for (uint32_t q = blockIdx.y; q < p.nq; q += gridDim.y) {
    const uint32_t padded = (p.dim + 15u) / 16u * 16u;
    for (uint32_t i = threadIdx.x; i < padded; i += kRescoreThreads)
        query[i] = i < p.dim ? double(float(static_cast<const T *>(p.queries)[size_t(q) * p.q_stride + i])) : 0.0;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const uint32_t end = min((blockIdx.x + 1u) * kRescoreEach, p.m);
    for (uint32_t c = blockIdx.x * kRescoreEach + (threadIdx.x >> 5); c < end; c += kRescoreThreads / 32) {
        const int64_t slot = p.slots[size_t(q) * p.slot_stride + c];
        const bool there = uint64_t(slot) < uint64_t(p.rows.rows);
        double sum = 0.0;
        if (there) {
            const uint8_t *row = p.rows.codes + size_t(slot) * p.rows.stride;
            for (uint32_t at = lane * 16u; at < p.dim; at += 512u) {
                uint32_t w[4] = {0, 0, 0, 0};
                if (at + 16u <= p.dim) __builtin_memcpy(w, row + at, 16);
                else
                    for (uint32_t i = 0; at + i < p.dim; ++i) w[i / 4] |= uint32_t(row[at + i]) << (8 * (i % 4));
                double part = 0.0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[i]), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[i]), true);
                    part = fma(double(lo[0]), query[at + 4 * i], part);
                    part = fma(double(lo[1]), query[at + 4 * i + 1], part);
                    part = fma(double(hi[0]), query[at + 4 * i + 2], part);
                    part = fma(double(hi[1]), query[at + 4 * i + 3], part);
                }
                sum = fma(part, scale_at(p.rows, uint32_t(slot), at / kScaleBlock, E8), sum);
            }
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor(sum, d);
        if (lane == 0) p.keys[size_t(q) * p.m + c] = there ? candidate_key(float(sum), uint32_t(slot)) : 0ull;
    }
    __syncthreads();
    }
}

// The k largest keys of a query, in order.
__global__ __launch_bounds__(kRescoreThreads) void k_rescore_best(RescoreArgs p, uint32_t size) {
    extern __shared__ uint64_t key[];        // size: the power of two not below m
    for (uint32_t q = blockIdx.x; q < p.nq; q += gridDim.x) {
    for (uint32_t i = threadIdx.x; i < size; i += kRescoreThreads) key[i] = i < p.m ? p.keys[size_t(q) * p.m + i] : 0ull;
    for (uint32_t run = 2; run <= size; run <<= 1) {
        for (uint32_t step = run >> 1; step > 0; step >>= 1) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < size / 2; i += kRescoreThreads) {
                const uint32_t lo = 2 * i - (i & (step - 1)), hi = lo + step;
                const uint64_t x = key[lo], y = key[hi];
                if ((x < y) == ((lo & run) == 0)) { key[lo] = y; key[hi] = x; }
            }
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < p.k; i += kRescoreThreads) {
        const uint64_t x = key[i];
        float s = -__int_as_float(0x7f800000);
        int64_t slot = -1;
        if (x != 0ull) {
            uint32_t at;
            sort_unkey(x, s, at);
            if (uint32_t(x >> 32) == 0u) s = __int_as_float(0x7fc00000);
            slot = int64_t(at);
        }
        p.out_scores[size_t(q) * p.k + i] = s;
        p.out_slots[size_t(q) * p.k + i] = slot;
    }
    __syncthreads();
    }
}

template <typename T, bool E8>
static hipError_t rescore(const RescoreArgs &a, hipStream_t s) {
    const dim3 grid((a.m + kRescoreEach - 1) / kRescoreEach, a.nq < 65535u ? a.nq : 65535u);
    const uint32_t lds = (a.dim + 15) / 16 * 16 * sizeof(double);
    if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(k_rescore_scores<T, E8>), lds); e != hipSuccess) return e;
    if (const hipError_t e = launch(k_rescore_scores<T, E8>, grid, kRescoreThreads, lds, s, a); e != hipSuccess) return e;
    uint32_t size = 2;
    while (size < a.m) size <<= 1;
    if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(k_rescore_best), size * 8u); e != hipSuccess) return e;
    return launch(k_rescore_best, a.nq < kMostSorts ? a.nq : kMostSorts, kRescoreThreads, size * 8u, s, a, size);
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
