// Log probabilities of given slots under a softmax of rows of scores, the softmax's entropy, its best slots, and the gradient of the scores.
//
// With m the largest score that counts, d = (score - m) / T, S = sum of exp(d) and U = sum of exp(d) d: log p = d - log S, and the entropy is
// log S - U / S, two terms that are not below 0.  Exponentials are of base 2, with log2(e) / T as the factor.
#include <cfloat>

#include "tv_device.h"
#include "tv_ops.h"

namespace tv {

constexpr float kInf = __builtin_inff(), kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint64_t kMostGroups = 1 << 20;    // workgroups of a launch: a grid of 2^32 threads is not allowed

// A row's temperature: the factors of a distance to the best score, in natural logarithms and in those of base 2.  A temperature that is not above 0 has the
// largest that there is: distances other than 0 are then infinite for all purposes.
struct Heat {
    float t, factor2;
    bool limit;
    __device__ __forceinline__ Heat(const float *temperature, uint32_t row) {
        t = temperature == nullptr ? 1.0f : temperature[row];
        limit = !(t > 0.0f);
        factor2 = limit ? FLT_MAX : fminf(kLog2e / t, FLT_MAX);
    }
    // log p of a slot at distance d <= 0, of a sum whose logarithm is log_sum
    __device__ __forceinline__ float log_p(float d, float log_sum) const { return (limit ? (d < 0.0f ? -kInf : d) : d / t) - log_sum; }
};
// Whether a score counts: allowed, and not -infinity.  (NaN counts: it shows.)
__device__ __forceinline__ bool counts(const uint64_t *mask, uint32_t i, float s) {
    return (mask == nullptr || ((mask[i >> 6] >> (i & 63u)) & 1u)) && !(s == -kInf);
}
// The order of alternatives, 0 for what is none.
__device__ __forceinline__ uint64_t slot_key(const uint64_t *mask, uint32_t i, float s) { return counts(mask, i, s) && s == s ? sort_key(s, i) : 0ull; }

// Sums of exp(d) and exp(d) log2(exp(d)) in d's own base.
struct Sums {
    float s = 0.0f, u = 0.0f;
    __device__ __forceinline__ void add(float t) {
        const float e = __builtin_amdgcn_exp2f(t);
        s += e;
        u = fmaf(e, fmaxf(t, -200.0f), u);       // (2^-200 is 0 here, an infinity times that is not)
    }
};

constexpr int kLogThreads = 256;
template <typename F>
__device__ __forceinline__ float over_group(float v, float *part, F &&f) {
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) v = f(v, __shfl_xor(v, i));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < kLogThreads / 64; ++i) v = f(v, part[i]);
    return v;
}

template <typename T>
__global__ __launch_bounds__(kLogThreads) void k_log_probs(LogProbArgs a) {
    __shared__ float part[kLogThreads / 64];
    __shared__ uint64_t best[kLogThreads / 64];
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *const scores = static_cast<const T *>(a.scores) + size_t(row) * a.stride;
        const uint64_t *const mask = a.mask == nullptr ? nullptr : a.mask + size_t(row) * a.mask_stride;
        const Heat heat(a.temperature, row);
        float m = -kInf;
        for (uint32_t i = threadIdx.x; i < a.n; i += kLogThreads) {
            const float s = float(scores[i]);
            if (counts(mask, i, s)) m = fmaxf(m, s);
        }
        m = over_group(m, part, [](float x, float y) { return fmaxf(x, y); });
        if (m == -kInf) m = 0.0f;
        Sums sums;
        for (uint32_t i = threadIdx.x; i < a.n; i += kLogThreads) {
            const float s = float(scores[i]);
            if (counts(mask, i, s)) sums.add((s - m) * heat.factor2);
        }
        const float s = over_group(sums.s, part, [](float x, float y) { return x + y; }), u = over_group(sums.u, part, [](float x, float y) { return x + y; });
        const float log_sum = logf(s), entropy = s == 0.0f ? 0.0f : log_sum - kLn2 * (u / s);
        if (threadIdx.x == 0) {
            a.out_entropy[row] = entropy;
            if (a.stats != nullptr) {
                float *const to = a.stats + size_t(row) * 4;
                to[0] = m; to[1] = log2f(s); to[2] = entropy; to[3] = 0.0f;
            }
        }
        for (uint32_t i = threadIdx.x; i < a.given; i += kLogThreads) {
            const int64_t slot = a.slots[size_t(row) * a.slot_stride + i];
            float lp = -kInf;
            if (slot >= 0 && slot < int64_t(a.n)) {
                const float v = float(scores[slot]);
                if (counts(mask, uint32_t(slot), v)) lp = heat.log_p(v - m, log_sum);
            }
            a.out_log_probs[size_t(row) * a.given + i] = lp;
        }
        uint64_t below = ~0ull;
        for (uint32_t k = 0; k < a.top; ++k) {
            uint64_t mine = 0;
            if (below != 0)
                for (uint32_t i = threadIdx.x; i < a.n; i += kLogThreads) {
                    const uint64_t key = slot_key(mask, i, float(scores[i]));
                    if (key < below && key > mine) mine = key;
                }
#pragma unroll
            for (int i = 32; i > 0; i >>= 1) mine = max(mine, uint64_t(__shfl_xor((unsigned long long)(mine), i)));
            __syncthreads();
            if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = mine;
            __syncthreads();
            for (int i = 0; i < kLogThreads / 64; ++i) mine = max(mine, best[i]);
            below = mine;
            if (threadIdx.x == 0) {
                float v = 0.0f;
                uint32_t slot = 0;
                sort_unkey(mine, v, slot);
                a.out_top_slots[size_t(row) * a.top + k] = mine == 0 ? -1 : int64_t(slot);
                a.out_top_log_probs[size_t(row) * a.top + k] = mine == 0 ? -kInf : heat.log_p(v - m, log_sum);
            }
        }
    }
}
size_t log_probs_workspace(size_t, size_t, size_t) { return 0; }
template <typename T>
static hipError_t log_probs(const LogProbArgs &a, hipStream_t s) {
    return launch(k_log_probs<T>, uint32_t(a.rows < kMostGroups ? a.rows : kMostGroups), kLogThreads, 0, s, a);
}
hipError_t launch_log_probs(const LogProbArgs &a, int score_type, hipStream_t s) {
    if (score_type == kF32) return log_probs<float>(a, s);
    return score_type == kF16 ? log_probs<f16>(a, s) : log_probs<bf16>(a, s);
}

// The gradient of a score that counts: (picked - G p - g p (log p + H)) / T, picked the sum of the gradients of the given slots that are this one.
template <typename T>
__global__ __launch_bounds__(kLogThreads) void k_log_probs_grad(LogProbGradArgs a) {
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *const scores = static_cast<const T *>(a.scores) + size_t(row) * a.stride;
        const uint64_t *const mask = a.mask == nullptr ? nullptr : a.mask + size_t(row) * a.mask_stride;
        T *const grad = static_cast<T *>(a.grad) + size_t(row) * a.grad_stride;
        const Heat heat(a.temperature, row);
        const float m = a.stats[size_t(row) * 4], log2_sum = a.stats[size_t(row) * 4 + 1], entropy = a.stats[size_t(row) * 4 + 2];
        const float *const g = a.grad_log_probs + size_t(row) * a.given;
        const int64_t *const slots = a.slots + size_t(row) * a.slot_stride;
        float all = 0.0f;
        for (uint32_t k = 0; k < a.given; ++k)
            if (slots[k] >= 0 && slots[k] < int64_t(a.n) && counts(mask, uint32_t(slots[k]), float(scores[slots[k]]))) all += g[k];
        const float g_entropy = a.grad_entropy == nullptr ? 0.0f : a.grad_entropy[row];
        for (uint32_t i = threadIdx.x; i < a.n; i += kLogThreads) {
            const float s = float(scores[i]);
            float d = 0.0f;
            if (counts(mask, i, s) && !heat.limit) {
                const float l = fmaf(s - m, heat.factor2, -log2_sum), p = __builtin_amdgcn_exp2f(l);
                for (uint32_t k = 0; k < a.given; ++k)
                    if (slots[k] == int64_t(i)) d += g[k];
                d = (d - p * (all + g_entropy * fmaf(kLn2, fmaxf(l, -200.0f), entropy))) / heat.t;
            }
            grad[i] = T(d);
        }
    }
}
template <typename T>
static hipError_t log_probs_grad(const LogProbGradArgs &a, hipStream_t s) {
    return launch(k_log_probs_grad<T>, uint32_t(a.rows < kMostGroups ? a.rows : kMostGroups), kLogThreads, 0, s, a);
}
hipError_t launch_log_probs_grad(const LogProbGradArgs &a, int score_type, hipStream_t s) {
    if (score_type == kF32) return log_probs_grad<float>(a, s);
    return score_type == kF16 ? log_probs_grad<f16>(a, s) : log_probs_grad<bf16>(a, s);
}

}  // namespace tv
