// Drawing a slot from rows of scores, with temperature, top-k, top-p and min-p, from given random numbers.
//
// The weight of a slot is exp((score - max) / T), taken in 64 bits and held as a whole number of 2^-shift, shift = 63 -
// ceil(log2 n): sums of any number of them fit 64 bits and do not depend on the order of the additions, so that a draw is the same
// whatever order threads arrive in.  What top-k, top-p and min-p leave is the slots above some score, and the first few by
// index of those that have it: a threshold score is found bit by bit, a byte at a time, from the highest, and the draw
// itself walks the slots in the order of their index.
#include "tv_device.h"
#include "tv_ops.h"

namespace tv {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr uint32_t kNoKey = 0x007fffffu;     // -infinity's; what is not allowed has it too

// The scores' order as unsigned numbers; -0 counts as +0, NaN as -infinity.
__device__ __forceinline__ uint32_t score_key(float s) {
    return s > -__int_as_float(0x7f800000) ? uint32_t(order_key(s + 0.0f)) ^ 0x80000000u : kNoKey;
}

template <typename T>
struct SampleRow {
    const T *scores;
    const uint64_t *mask;
    uint32_t n;
    double top, inverse;      // the largest score, 1 / T
    int shift;
    __device__ __forceinline__ uint32_t key(uint32_t i) const {
        const uint32_t k = score_key(float(scores[i]));
        return mask == nullptr || ((mask[i >> 6] >> (i & 63u)) & 1u) ? k : kNoKey;
    }
    // exp((score - max) / T); for scores whose largest is +infinity, 1 for those that have it
    __device__ __forceinline__ double weight(uint32_t k) const {
        const double s = double(order_unkey(int(k ^ 0x80000000u)));
        return s == top ? 1.0 : exp((s - top) * inverse);
    }
    __device__ __forceinline__ uint64_t units(double w) const { return uint64_t(__double2ull_rn(ldexp(w, shift))); }
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

struct SampleShared {
    uint64_t mass[256];
    uint32_t count[256];
    uint64_t part[kSampleWaves];
    uint64_t found, before;
    uint32_t word, base_count;
};

// In index order, the first i whose f summed over 0..i exceeds target(total); all threads return it.  total > 0.
template <typename F, typename G>
__device__ uint32_t locate(uint32_t n, SampleShared &sh, F &&f, G &&target, uint64_t &total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t lo = 0, len = n;
    uint64_t want = 0;
    bool first = true;
    while (first || len > uint32_t(kSampleThreads)) {
        const uint32_t seg = ((len + kSampleWaves - 1) / kSampleWaves + 63u) & ~63u;
        const uint32_t from = min(len, wave * seg), to = min(len, from + seg);
        uint64_t sum = 0;
        for (uint32_t i = from + lane; i < to; i += 64u) sum += f(lo + i);
        sum = wave_sum64(sum);
        __syncthreads();
        if (lane == 0) sh.part[wave] = sum;
        __syncthreads();
        if (first) {
            total = 0;
            for (int w = 0; w < kSampleWaves; ++w) total += sh.part[w];
            want = target(total);
            first = false;
        }
        uint32_t w = 0;
        uint64_t upto = sh.part[0], before = 0;
        while (w + 1 < uint32_t(kSampleWaves) && upto <= want) {
            before = upto;
            upto += sh.part[++w];
        }
        want -= before;
        lo += min(len, w * seg);
        len = min(seg, len - min(len, w * seg));
    }
    // at most one slot to a thread
    const uint64_t mine = threadIdx.x < len ? f(lo + threadIdx.x) : 0;
    uint64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up(upto, d);
        if (int(lane) >= d) upto += o;
    }
    __syncthreads();
    if (lane == 63u) sh.part[wave] = upto;
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) upto += sh.part[w];
    if (upto > want && upto - mine <= want) sh.found = threadIdx.x;
    __syncthreads();
    return lo + uint32_t(sh.found);
}

// The key of the class, in falling order, that `stop` picks, byte by byte: stop(count before, mass before, count, mass) is asked of
// every class that has slots, from the highest, and the last one it says yes to is it.  MASS: whether masses are wanted.
template <bool MASS, typename T, typename F>
__device__ uint32_t select_class(const SampleRow<T> &row, SampleShared &sh, F &&reaches, uint64_t &count_before, uint64_t &mass_before, uint32_t &count) {
    uint32_t prefix = 0;
    count_before = mass_before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 256u; i += kSampleThreads) { sh.mass[i] = 0; sh.count[i] = 0; }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < row.n; i += kSampleThreads) {
            const uint32_t k = row.key(i);
            if (k == kNoKey || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
            atomicAdd(&sh.count[(k >> shift) & 255u], 1u);
            if (MASS) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[(k >> shift) & 255u]), (unsigned long long)row.units(row.weight(k)));
        }
        __syncthreads();
        uint32_t pick = 0;
        uint64_t c = count_before, m = mass_before, pc = c, pm = m;
        for (int b = 255; b >= 0; --b) {
            if (sh.count[b] == 0) continue;
            if (!reaches(c, m)) break;
            pick = uint32_t(b); pc = c; pm = m;
            c += sh.count[b];
            m += sh.mass[b];
        }
        count_before = pc; mass_before = pm;
        count = sh.count[pick];
        prefix = (prefix << 8) | pick;
    }
    return prefix;
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample(SampleArgs p) {
    __shared__ SampleShared sh;
    for (uint32_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        SampleRow<T> row;
        row.scores = static_cast<const T *>(p.scores) + size_t(r) * p.stride;
        row.mask = p.mask == nullptr ? nullptr : p.mask + size_t(r) * p.mask_stride;
        row.n = p.n;
        uint32_t most = kNoKey;
        for (uint32_t i = threadIdx.x; i < p.n; i += kSampleThreads) most = max(most, row.key(i));
        most = wave_umax(most);
        __syncthreads();
        if ((threadIdx.x & 63u) == 0) sh.part[threadIdx.x >> 6] = most;
        __syncthreads();
        for (int w = 0; w < kSampleWaves; ++w) most = max(most, uint32_t(sh.part[w]));
        if (most == kNoKey) {
            if (threadIdx.x == 0) { p.out_slots[r] = -1; p.out_probs[r] = 0.0f; }
            continue;
        }
        const float t = p.temperature == nullptr ? 1.0f : p.temperature[r];
        uint64_t total;
        if (!(t > 0.0f)) {       // the best alone
            const uint32_t at = locate(p.n, sh, [&](uint32_t i) { return uint64_t(row.key(i) == most); }, [](uint64_t) { return uint64_t(0); }, total);
            if (threadIdx.x == 0) { p.out_slots[r] = at; p.out_probs[r] = 1.0f; }
            continue;
        }
        row.top = double(order_unkey(int(most ^ 0x80000000u)));
        row.inverse = 1.0 / double(t);
        row.shift = 63 - (32 - __clz(int(p.n - 1 | 1)));
        const int32_t top_k = p.top_k == nullptr ? 0 : p.top_k[r];
        const float top_p = p.top_p == nullptr ? 1.0f : p.top_p[r];
        const double min_p = p.min_p != nullptr && p.min_p[r] > 0.0f ? fmin(double(p.min_p[r]), 1.0) : 0.0;
        uint32_t least = kNoKey + 1u, ties = ~0u, tie_last = ~0u;      // slots of a higher key stay, and of those of this one so many
        uint32_t equal = 0;
        uint64_t count_before, mass_before;
        const bool limit_k = top_k > 0 && uint32_t(top_k) < p.n, limit_p = top_p < 1.0f;
        if (limit_k) {
            least = select_class<false>(row, sh, [&](uint64_t c, uint64_t) { return c < uint64_t(top_k); }, count_before, mass_before, equal);
            ties = min(equal, uint32_t(uint64_t(top_k) - count_before));
        }
        if (limit_p) {
            // of the mass that top-k leaves
            uint64_t sum = 0;
            for (uint32_t i = threadIdx.x; i < p.n; i += kSampleThreads) {
                const uint32_t k = row.key(i);
                if (k >= least && k != kNoKey && (!limit_k || k != least)) sum += row.units(row.weight(k));
            }
            sum = wave_sum64(sum);
            __syncthreads();
            if ((threadIdx.x & 63u) == 0) sh.part[threadIdx.x >> 6] = sum;
            __syncthreads();
            sum = limit_k ? row.units(row.weight(least)) * ties : 0;
            for (int w = 0; w < kSampleWaves; ++w) sum += sh.part[w];
            const double limit = double(top_p) * double(sum);
            const uint32_t key = select_class<true>(row, sh, [&](uint64_t c, uint64_t m) { return c == 0 || double(m) < limit; }, count_before, mass_before, equal);
            const uint64_t each = row.units(row.weight(key));
            const double fit = each == 0 ? double(equal) : ceil((limit - double(mass_before)) / double(each));
            const uint32_t stay = fit < 1.0 ? 1u : fit < double(equal) ? uint32_t(fit) : equal;
            // (never below top-k's class: the mass up to its end is all that top-k left, or more)
            ties = limit_k && key == least ? min(stay, ties) : stay;
            least = key;
        }
        if ((limit_k || limit_p) && ties < equal) {
            uint64_t all;
            tie_last = locate(p.n, sh, [&](uint32_t i) { return uint64_t(row.key(i) == least); }, [&](uint64_t) { return uint64_t(ties - 1u); }, all);
        }
        const float u = p.u[r];
        const uint32_t at = locate(p.n, sh,
            [&](uint32_t i) {
                const uint32_t k = row.key(i);
                if (k < least || k == kNoKey || (k == least && i > tie_last)) return uint64_t(0);
                const double w = row.weight(k);
                return w >= min_p ? row.units(w) : uint64_t(0);
            },
            [&](uint64_t sum) {
                const double want = double(u) * double(sum);
                return want >= double(sum) ? sum - 1 : want > 0.0 ? uint64_t(want) : uint64_t(0);
            }, total);
        if (threadIdx.x == 0) {
            p.out_slots[r] = at;
            p.out_probs[r] = float(ldexp(row.weight(row.key(at)), row.shift) / double(total));
        }
    }
}

size_t sample_workspace(size_t, size_t) { return 0; }

template <typename T>
static hipError_t sample(const SampleArgs &a, hipStream_t s) {
    return launch(k_sample<T>, a.rows < 65536u ? a.rows : 65536u, kSampleThreads, 0, s, a);
}
hipError_t launch_sample(const SampleArgs &a, int score_type, hipStream_t s) {
    if (score_type == kF32) return sample<float>(a, s);
    return score_type == kF16 ? sample<f16>(a, s) : sample<bf16>(a, s);
}

}  // namespace tv
