// Drawing a slot from rows of scores, with temperature, top-k, top-p and min-p, from given random numbers.
//
// The weight of a slot is exp((score - max) / T), taken in 64 bits and held as a whole number of 2^-shift, shift = 63 -
// ceil(log2 n): sums of any number of them fit 64 bits and do not depend on the order of the additions, so that a draw is the same
// whatever order threads arrive in.  What top-k, top-p and min-p leave is a prefix of the slots ranked by score, ties to the lower
// slot: the slots above some score, and the first few of those that have it.
//
// A histogram over the distance to the best score, whose bins widen with it, finds the bin that top-k or top-p end in.  Where the slots
// down to that bin are few, they are gathered, sorted, and everything else happens among them.  Where they are many, the bin is
// divided again until what is left in it is one score or few slots; then the row is walked once more to draw from what stays.
#include "tv_device.h"
#include "tv_ops.h"

namespace tv {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr uint32_t kNoKey = 0x007fffffu;     // -infinity's; what is not allowed has it too
constexpr uint32_t kBins = 1024;             // a bin to a thread
constexpr uint32_t kListed = 4096, kListedEach = kListed / kSampleThreads;     // slots that are gathered and sorted, at most

// The scores' order as unsigned numbers; -0 counts as +0, NaN as -infinity.
__device__ __forceinline__ uint32_t score_key(float s) {
    return s > -__int_as_float(0x7f800000) ? uint32_t(order_key(s + 0.0f)) ^ 0x80000000u : kNoKey;
}
__device__ __forceinline__ float key_score(uint32_t k) { return order_unkey(int(k ^ 0x80000000u)); }

template <typename T>
struct SampleRow {
    static constexpr int kEach = 16 / int(sizeof(T));
    const T *scores;
    const uint64_t *mask;
    uint32_t n, most;         // most: the key of the largest score
    double top, inverse;      // that score, 1 / T
    int shift;
    struct Load {
        T v[kEach];
        uint32_t bits;
    };
    // Scores i .. i + kEach - 1, those past the end not allowed; i is a multiple of kEach.
    __device__ __forceinline__ void load(Load &l, uint32_t i) const {
        l.bits = mask == nullptr ? ~0u : uint32_t(mask[i >> 6] >> (i & 63u));
        if (i + kEach <= n) {
            __builtin_memcpy(l.v, scores + i, 16);
            return;
        }
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            l.v[j] = T(0.0f);
            if (i + j < n) l.v[j] = scores[i + j];
            else l.bits &= ~(1u << j);
        }
    }
    __device__ __forceinline__ uint32_t key(const Load &l, int j) const { return (l.bits >> j) & 1u ? score_key(float(l.v[j])) : kNoKey; }
    __device__ __forceinline__ uint32_t key_at(uint32_t i) const {
        return mask == nullptr || ((mask[i >> 6] >> (i & 63u)) & 1u) ? score_key(float(scores[i])) : kNoKey;
    }
    // f(slot, key) for every slot of lo .. hi - 1 (multiples of kEach, or the end), a worker of `workers`.
    template <typename F>
    __device__ __forceinline__ void each(uint32_t lo, uint32_t hi, uint32_t worker, uint32_t workers, F &&f) const {
        constexpr int kAtOnce = 4;
        const uint32_t step = workers * kEach;
        uint32_t i = lo + worker * kEach;
        for (; i < hi && hi - i > (kAtOnce - 1) * step; i += kAtOnce * step) {
            Load l[kAtOnce];
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) load(l[a], i + a * step);
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a)
#pragma unroll
                for (int j = 0; j < kEach; ++j) f(i + a * step + j, key(l[a], j));
        }
        for (; i < hi; i += step) {
            Load l;
            load(l, i);
#pragma unroll
            for (int j = 0; j < kEach; ++j) f(i + j, key(l, j));
        }
    }
    // exp((score - max) / T); for scores whose largest is +infinity, 1 for those that have it
    __device__ __forceinline__ double weight(uint32_t k) const { return k == most ? 1.0 : exp((double(key_score(k)) - top) * inverse); }
    __device__ __forceinline__ uint64_t units(double w) const { return uint64_t(__double2ull_rn(ldexp(w, shift))); }
    // The bin of a key: 32 for each power of two that the distance to the best score spans, from 2^-20 to 2^12.
    __device__ __forceinline__ uint32_t bin(uint32_t k) const {
        const float d = key_score(most) - key_score(k);
        const int x = k == most ? 0 : int(__float_as_uint(d) >> 18) - (127 - 20) * 32;
        return uint32_t(min(max(x, 0), int(kBins) - 1));
    }
    // The least key of those in bins up to b (keys rise as bins fall).
    __device__ __forceinline__ uint32_t least_of_bin(uint32_t b) const {
        uint32_t lo = kNoKey + 1u, hi = most;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (bin(mid) <= b) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    }
    // The least key whose weight is min_p or more.
    __device__ __forceinline__ uint32_t least_of_weight(double min_p) const {
        uint32_t lo = kNoKey + 1u, hi = most;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (weight(mid) >= min_p) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    }
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

struct SampleShared {
    uint64_t mass[kBins];
    uint64_t list[kListed], held[kListed];
    uint64_t part[kSampleWaves], found_mass;
    uint32_t count[kBins];
    uint32_t part32[kSampleWaves], listed, picked, found_count;
};

__device__ uint64_t block_sum(uint64_t v, SampleShared &sh) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t all = 0;
    for (int w = 0; w < kSampleWaves; ++w) all += sh.part[w];
    return all;
}
// The sum over the threads before this one; `all` the sum over all of them.
__device__ uint64_t block_before(uint64_t v, SampleShared &sh, uint64_t &all) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint64_t upto = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up(upto, d);
        if (int(lane) >= d) upto += o;
    }
    __syncthreads();
    if (lane == 63u) sh.part[wave] = upto;
    __syncthreads();
    uint64_t before = upto - v;
    all = 0;
    for (uint32_t w = 0; w < uint32_t(kSampleWaves); ++w) {
        if (w < wave) before += sh.part[w];
        all += sh.part[w];
    }
    return before;
}

// Sorts `size` (a power of two) words, falling.
__device__ void sort_falling(uint64_t *x, uint32_t size) {
    for (uint32_t run = 2; run <= size; run <<= 1) {
        for (uint32_t step = run >> 1; step > 0; step >>= 1) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < size / 2; i += kSampleThreads) {
                const uint32_t lo = 2 * i - (i & (step - 1)), hi = lo + step;
                const uint64_t a = x[lo], b = x[hi];
                if ((a < b) == ((lo & run) == 0)) { x[lo] = b; x[hi] = a; }
            }
        }
    }
    __syncthreads();
}

// In slot order, the first slot whose f summed up to it exceeds target(total); all threads return it.  total > 0.
template <typename T, typename F, typename G>
__device__ uint32_t locate(const SampleRow<T> &row, SampleShared &sh, F &&f, G &&target, uint64_t &total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t lo = 0, len = row.n;
    uint64_t want = 0;
    bool first = true;
    while (first || len > uint32_t(kSampleThreads)) {
        const uint32_t seg = ((len + kSampleWaves - 1) / kSampleWaves + 63u) & ~63u;
        const uint32_t from = min(len, wave * seg), to = min(len, from + seg);
        uint64_t sum = 0;
        row.each(lo + from, lo + to, lane, 64u, [&](uint32_t i, uint32_t k) { if (k != kNoKey) sum += f(i, k); });
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
    const uint32_t i = lo + threadIdx.x, k = threadIdx.x < len ? row.key_at(i) : kNoKey;
    const uint64_t mine = k != kNoKey ? f(i, k) : 0;
    uint64_t all;
    const uint64_t before = block_before(mine, sh, all);
    if (threadIdx.x == 0) sh.picked = 0;
    __syncthreads();
    if (before <= want && before + mine > want) sh.picked = threadIdx.x;
    __syncthreads();
    return lo + sh.picked;
}

// What a threshold is looked for by: its keys lo .. hi, how many slots have one of them, and what lies above.
struct Range {
    uint32_t lo, hi, count;
    uint64_t count_before, mass_before;
};

// One histogram: of the slots whose keys lie in r, the bins by bin_of; then the last bin that has slots and that reaches(count before, mass
// before) says yes to, r's counts becoming that bin's.  Returns the bin; total gets the mass of all bins.
template <bool MASS, typename T, typename B, typename F>
__device__ uint32_t pick_bin(const SampleRow<T> &row, SampleShared &sh, Range &r, B &&bin_of, F &&reaches, uint64_t &total) {
    const uint32_t t = threadIdx.x;
    __syncthreads();
    sh.count[t] = 0;
    if (MASS) sh.mass[t] = 0;
    if (t == 0) sh.picked = 0;
    __syncthreads();
    row.each(0, row.n, t, kSampleThreads, [&](uint32_t, uint32_t k) {
        if (k < r.lo || k > r.hi) return;
        const uint32_t b = bin_of(k);
        atomicAdd(&sh.count[b], 1u);
        if (MASS) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[b]), (unsigned long long)row.units(row.weight(k)));
    });
    __syncthreads();
    uint64_t all;
    const uint64_t count = sh.count[t], count_before = r.count_before + block_before(count, sh, all);
    const uint64_t mass_before = MASS ? r.mass_before + block_before(sh.mass[t], sh, total) : 0;
    if (count != 0 && (t == 0 || reaches(count_before, mass_before))) atomicMax(&sh.picked, t);
    __syncthreads();
    const uint32_t pick = sh.picked;
    if (t == pick) { sh.found_count = uint32_t(count_before); sh.found_mass = mass_before; }
    __syncthreads();
    r.count = sh.count[pick];
    r.count_before = sh.found_count;
    r.mass_before = sh.found_mass;
    return pick;
}

// Gathers the slots whose keys lie in lo .. hi, kListed at most, in the order of their keys, ties to the lower slot.
template <typename T>
__device__ uint32_t gather(const SampleRow<T> &row, SampleShared &sh, uint32_t lo, uint32_t hi) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    row.each(0, row.n, threadIdx.x, kSampleThreads, [&](uint32_t i, uint32_t k) {
        if (k < lo || k > hi) return;
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kListed) sh.list[at] = uint64_t(k) << 32 | uint32_t(~i);
    });
    __syncthreads();
    const uint32_t listed = min(sh.listed, kListed);
    uint32_t size = 2;
    while (size < listed) size <<= 1;
    for (uint32_t i = listed + threadIdx.x; i < size; i += kSampleThreads) sh.list[i] = 0;
    sort_falling(sh.list, size);
    return listed;
}

// Narrows r to one key: the last, in falling order, that has slots and that reaches(count before, mass before) says yes to.
template <bool MASS, typename T, typename F>
__device__ void narrow(const SampleRow<T> &row, SampleShared &sh, Range &r, F &&reaches) {
    uint64_t total;
    while (r.lo < r.hi && r.count > kListed) {
        const uint32_t hi = r.hi, shift = uint32_t(max(0, 22 - __clz(int(r.hi - r.lo))));
        const uint32_t b = pick_bin<MASS>(row, sh, r, [=](uint32_t k) { return (hi - k) >> shift; }, reaches, total);
        r.hi = hi - (b << shift);
        r.lo = max(r.lo, r.hi - min(r.hi, (1u << shift) - 1u));
    }
    if (r.lo == r.hi) return;
    const uint32_t listed = gather(row, sh, r.lo, r.hi);
    // every slot of the list by itself: the last one that is reached has the key
    uint64_t mass[kListedEach], sum = 0, all = 0;
#pragma unroll
    for (uint32_t j = 0; j < kListedEach; ++j) {
        const uint32_t e = threadIdx.x * kListedEach + j;
        mass[j] = MASS && e < listed ? row.units(row.weight(uint32_t(sh.list[e] >> 32))) : 0;
        sum += mass[j];
    }
    uint64_t before = r.mass_before + (MASS ? block_before(sum, sh, all) : 0);
    if (threadIdx.x == 0) sh.picked = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kListedEach; ++j) {
        const uint32_t e = threadIdx.x * kListedEach + j;
        if (e < listed && (e == 0 || reaches(r.count_before + e, before))) atomicMax(&sh.picked, e);
        before += mass[j];
    }
    __syncthreads();
    const uint32_t key = uint32_t(sh.list[sh.picked] >> 32);
    // the slots above it, and those that have it
    uint64_t above = 0, equal = 0, heavier = 0;
#pragma unroll
    for (uint32_t j = 0; j < kListedEach; ++j) {
        const uint32_t e = threadIdx.x * kListedEach + j;
        if (e >= listed) continue;
        const uint32_t k = uint32_t(sh.list[e] >> 32);
        above += k > key;
        equal += k == key;
        heavier += k > key ? mass[j] : 0;
    }
    r.count_before += block_sum(above, sh);
    r.mass_before += MASS ? block_sum(heavier, sh) : 0;
    r.count = uint32_t(block_sum(equal, sh));
    r.lo = r.hi = key;
}

__device__ __forceinline__ uint64_t drawn_mass(float u, uint64_t sum) {
    const double want = double(u) * double(sum);
    return want >= double(sum) ? sum - 1 : want > 0.0 ? uint64_t(want) : uint64_t(0);
}

// Draws from the slots of sh.list, in the order of their rank, `listed` of them: the first top_k, those of them that less than `limit` of
// mass lies before, those of at least min_key.  top_p: the share that limit is of the mass of the first top_k, where it is one of the list's.
template <typename T>
__device__ void draw_from_list(const SampleRow<T> &row, SampleShared &sh, uint32_t listed, bool limit_p, bool share, double top_p, double limit, uint32_t min_key,
                               float u, int64_t &slot, float &prob) {
    uint64_t mass[kListedEach], sum = 0, all;
#pragma unroll
    for (uint32_t j = 0; j < kListedEach; ++j) {
        const uint32_t e = threadIdx.x * kListedEach + j;
        mass[j] = e < listed ? row.units(row.weight(uint32_t(sh.list[e] >> 32))) : 0;
        sum += mass[j];
    }
    uint64_t before = block_before(sum, sh, all);
    if (share) limit = top_p * double(all);
    sum = 0;
    uint32_t size = 2;
    while (size < listed) size <<= 1;
    for (uint32_t e = listed + threadIdx.x; e < size; e += kSampleThreads) sh.held[e] = 0;
#pragma unroll
    for (uint32_t j = 0; j < kListedEach; ++j) {
        const uint32_t e = threadIdx.x * kListedEach + j;
        if (e < listed) {
            const uint64_t x = sh.list[e];
            const bool stays = e == 0 || ((!limit_p || double(before) < limit) && uint32_t(x >> 32) >= min_key);
            sum += stays ? mass[j] : 0;
            // by slot, falling as its complement does: low word the rank
            sh.held[e] = stays ? uint64_t(uint32_t(x)) << 32 | e : 0;
        }
        before += mass[j];
    }
    const uint64_t total = block_sum(sum, sh), want = drawn_mass(u, total);
    sort_falling(sh.held, size);
    sum = 0;
#pragma unroll
    for (uint32_t j = 0; j < kListedEach; ++j) {
        const uint32_t e = threadIdx.x * kListedEach + j;
        const uint64_t x = e < size ? sh.held[e] : 0;
        mass[j] = x != 0 ? row.units(row.weight(uint32_t(sh.list[uint32_t(x)] >> 32))) : 0;
        sum += mass[j];
    }
    before = block_before(sum, sh, all);
    if (threadIdx.x == 0) sh.picked = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kListedEach; ++j) {
        if (before <= want && before + mass[j] > want) sh.picked = threadIdx.x * kListedEach + j;
        before += mass[j];
    }
    __syncthreads();
    const uint64_t x = sh.held[sh.picked];
    slot = int64_t(~uint32_t(x >> 32));
    prob = float(ldexp(row.weight(uint32_t(sh.list[uint32_t(x)] >> 32)), row.shift) / double(total));
}

template <typename T>
__device__ void sample_row(const SampleArgs &p, const SampleRow<T> &row, SampleShared &sh, float t, uint32_t r, int64_t &slot, float &prob) {
    int32_t top_k = p.top_k == nullptr ? 0 : p.top_k[r];
    float top_p = p.top_p == nullptr ? 1.0f : p.top_p[r];
    const float least_p = p.min_p == nullptr ? 0.0f : p.min_p[r], u = p.u[r];
    if (!(t > 0.0f)) { top_k = 1; top_p = 1.0f; }       // the best alone
    const bool limit_k = top_k > 0 && uint32_t(top_k) < row.n, limit_p = top_p < 1.0f;
    const uint32_t min_key = least_p > 0.0f ? row.least_of_weight(fmin(double(least_p), 1.0)) : kNoKey + 1u;
    const auto first_k = [&](uint64_t c, uint64_t) { return c < uint64_t(top_k); };
    uint64_t total = 0;
    uint32_t least = kNoKey + 1u, equal = 0, ties = 0;      // slots of a higher key stay, and so many of those of this one
    if (limit_k) {
        Range all{kNoKey + 1u, row.most, 0, 0, 0};
        const uint32_t b = pick_bin<false>(row, sh, all, [&](uint32_t k) { return row.bin(k); }, first_k, total);
        all.lo = row.least_of_bin(b);
        if (all.count_before + all.count <= kListed) {
            const uint32_t listed = gather(row, sh, all.lo, row.most);
            return draw_from_list(row, sh, min(listed, uint32_t(top_k)), limit_p, true, double(top_p), 0.0, min_key, u, slot, prob);
        }
        if (b != 0) all.hi = row.least_of_bin(b - 1) - 1u;
        narrow<false>(row, sh, all, first_k);
        least = all.lo;
        equal = all.count;
        ties = min(equal, uint32_t(uint64_t(top_k) - all.count_before));
    }
    if (limit_p) {
        double limit = 0.0;
        if (limit_k) {
            uint64_t sum = 0;
            row.each(0, row.n, threadIdx.x, kSampleThreads, [&](uint32_t, uint32_t k) { if (k > least) sum += row.units(row.weight(k)); });
            limit = double(top_p) * double(block_sum(sum, sh) + row.units(row.weight(least)) * ties);
        }
        const auto first_p = [&](uint64_t c, uint64_t m) { return c == 0 || double(m) < limit; };
        Range all{least, row.most, 0, 0, 0};
        // (the limit is a share of the mass that the histogram itself adds up, where top-k has left everything)
        const uint32_t b = pick_bin<true>(row, sh, all, [&](uint32_t k) { return row.bin(k); },
            [&](uint64_t c, uint64_t m) { return c == 0 || double(m) < (limit_k ? limit : double(top_p) * double(total)); }, total);
        if (!limit_k) limit = double(top_p) * double(total);
        all.lo = max(least, row.least_of_bin(b));
        if (!limit_k) {
            // of what top-p may leave, min-p leaves the slots of min_key and above
            const uint32_t from = max(all.lo, min_key);
            if (from > all.lo || all.count_before + all.count <= kListed) {
                const uint32_t listed = gather(row, sh, from, row.most);
                if (sh.listed <= kListed) return draw_from_list(row, sh, listed, true, false, 0.0, limit, min_key, u, slot, prob);
            }
        }
        if (b != 0) all.hi = row.least_of_bin(b - 1) - 1u;
        narrow<true>(row, sh, all, first_p);
        const uint64_t each = row.units(row.weight(all.lo));
        const double fit = each == 0 ? double(all.count) : ceil((limit - double(all.mass_before)) / double(each));
        const uint32_t stay = fit < 1.0 ? 1u : fit < double(all.count) ? uint32_t(fit) : all.count;
        // (never below top-k's class: the mass up to its end is all that top-k left, or more)
        ties = limit_k && all.lo == least ? min(stay, ties) : stay;
        least = all.lo;
        equal = all.count;
    }
    uint32_t tie_last = ~0u;
    if (ties < equal) {
        uint64_t all;
        tie_last = locate(row, sh, [&](uint32_t, uint32_t k) { return uint64_t(k == least); }, [&](uint64_t) { return uint64_t(ties - 1u); }, all);
    }
    const uint32_t at = locate(row, sh,
        [&](uint32_t i, uint32_t k) { return k < least || k < min_key || (k == least && i > tie_last) ? uint64_t(0) : row.units(row.weight(k)); },
        [&](uint64_t sum) { return drawn_mass(u, sum); }, total);
    slot = at;
    prob = float(ldexp(row.weight(row.key_at(at)), row.shift) / double(total));
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample(SampleArgs p) {
    extern __shared__ uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    for (uint32_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        SampleRow<T> row;
        row.scores = static_cast<const T *>(p.scores) + size_t(r) * p.stride;
        row.mask = p.mask == nullptr ? nullptr : p.mask + size_t(r) * p.mask_stride;
        row.n = p.n;
        uint32_t most = kNoKey;
        row.each(0, p.n, threadIdx.x, kSampleThreads, [&](uint32_t, uint32_t k) { most = max(most, k); });
        most = wave_umax(most);
        __syncthreads();
        if ((threadIdx.x & 63u) == 0) sh.part32[threadIdx.x >> 6] = most;
        __syncthreads();
        for (int w = 0; w < kSampleWaves; ++w) most = max(most, sh.part32[w]);
        int64_t slot = -1;
        float prob = 0.0f;
        if (most != kNoKey) {
            const float t = p.temperature == nullptr ? 1.0f : p.temperature[r];
            row.most = most;
            row.top = double(key_score(most));
            row.inverse = t > 0.0f && row.top < __longlong_as_double(0x7ff0000000000000ll) ? 1.0 / double(t) : 1.0;     // (an infinite best leaves the others nothing)
            row.shift = 63 - (32 - __clz(int((p.n - 1u) | 1u)));
            sample_row(p, row, sh, t, r, slot, prob);
        }
        if (threadIdx.x == 0) { p.out_slots[r] = slot; p.out_probs[r] = prob; }
        __syncthreads();
    }
}

size_t sample_workspace(size_t, size_t) { return 0; }

template <typename T>
static hipError_t sample(const SampleArgs &a, hipStream_t s) {
    if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(k_sample<T>), sizeof(SampleShared)); e != hipSuccess) return e;
    return launch(k_sample<T>, a.rows < 65536u ? a.rows : 65536u, kSampleThreads, sizeof(SampleShared), s, a);
}
hipError_t launch_sample(const SampleArgs &a, int score_type, hipStream_t s) {
    if (score_type == kF32) return sample<float>(a, s);
    return score_type == kF16 ? sample<f16>(a, s) : sample<bf16>(a, s);
}

}  // namespace tv
