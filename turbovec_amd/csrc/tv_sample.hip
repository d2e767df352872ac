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
constexpr uint32_t kListed = 4000, kListedEach = 4;     // slots that are gathered, at most: four to a thread, and two workgroups' LDS to a compute unit
constexpr uint32_t kSorted = 512;            // of which so many are sorted

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
    double top, inverse, inverse2;      // that score, 1 / T, and that times log2(e)
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
        const uint32_t step = workers * kEach;
        uint32_t i = lo + worker * kEach;
        if (i >= hi) return;
        Load now, next;
        load(now, i);
        while (true) {
            const bool more = hi - i > step;
            if (more) load(next, i + step);
#pragma unroll
            for (int j = 0; j < kEach; ++j) f(i + j, key(now, j));
            if (!more) return;
            now = next;
            i += step;
        }
    }
    // exp((score - max) / T); for scores whose largest is +infinity, 1 for those that have it
    __device__ __forceinline__ double weight(uint32_t k) const { return k == most ? 1.0 : exp((double(key_score(k)) - top) * inverse); }
    // The same as a whole number of 2^-shift, which is what sums are made of: 2^y = 2^e * 2^f, |f| <= 1/2, with the exponential series up to
    // its tenth power (off by 2.2e-13 at most); adding 2 leaves its value in the low 52 bits.  A library exponential and a
    // conversion to 64 bits take three times as long.
    __device__ __forceinline__ uint64_t units(uint32_t k) const {
        const double y = fmax((double(key_score(k)) - top) * inverse2, -200.0);
        const double e = rint(y), f = (y - e) * 0.69314718055994530942;
        double v = 1.0 / 3628800.0;
        v = fma(v, f, 1.0 / 362880.0);
        v = fma(v, f, 1.0 / 40320.0);
        v = fma(v, f, 1.0 / 5040.0);
        v = fma(v, f, 1.0 / 720.0);
        v = fma(v, f, 1.0 / 120.0);
        v = fma(v, f, 1.0 / 24.0);
        v = fma(v, f, 1.0 / 6.0);
        v = fma(v, f, 0.5);
        v = fma(v, f, 1.0);
        v = fma(v, f, 1.0);
        const uint64_t bits = uint64_t(__double_as_longlong(v + 2.0)) & 0xfffffffffffffull;      // v * 2^51
        const int down = 62 - shift - int(e);
        const uint64_t x = bits << 11;
        return k == most ? 1ull << shift : down >= 64 ? 0ull : (x + ((1ull << down) >> 1)) >> down;
    }
    // The bin of a key: 32 for each power of two that the distance to the best score spans, from 2^-20 to 2^12.
    __device__ __forceinline__ uint32_t bin(uint32_t k) const {
        const float d = key_score(most) - key_score(k);
        const int x = k == most ? 0 : int(__float_as_uint(d) >> 18) - (127 - 20) * 32;
        return uint32_t(min(max(x, 0), int(kBins) - 1));
    }
    // The least key of those in bins up to b (keys rise as bins fall): every lane of a wave tries one of 64 places, until a step is one key.
    __device__ __forceinline__ uint32_t least_of_bin(uint32_t b) const {
        uint32_t lo = kNoKey + 1u, left = most - lo;           // it is one of lo .. lo + left
        while (left != 0u) {
            const uint32_t step = left / 64u + 1u, mine = lo + min(left, (threadIdx.x & 63u) * step);
            const uint64_t yes = __ballot(bin(mine) <= b);
            const uint32_t first = yes == 0ull ? 64u : uint32_t(__builtin_ctzll(yes));
            if (first == 0u) return lo;
            // above the place before the first that is, and no further
            const uint32_t under = lo + min(left, (first - 1u) * step), upto = first == 64u ? lo + left : lo + min(left, first * step);
            left = upto - (under + 1u);
            lo = under + 1u;
        }
        return lo;
    }
    // The least key whose weight is min_p (above 0) or more.
    __device__ __forceinline__ uint32_t least_of_weight(double min_p, double t) const {
        if (min_p >= 1.0 || !(top < __longlong_as_double(0x7ff0000000000000ll))) return most;
        const double from = top + log(min_p) * t;
        const uint32_t k = score_key(float(from));
        return max(k + (k != kNoKey && double(float(from)) < from ? 1u : 0u), kNoKey + 1u);
    }
    // Of a row's scores, given the largest one's key.
    __device__ __forceinline__ void set(uint32_t most_, float t) {
        most = most_;
        top = double(key_score(most));
        // (an infinite best leaves the others nothing)
        inverse = t > 0.0f && top < __longlong_as_double(0x7ff0000000000000ll) ? 1.0 / double(t) : 1.0;
        inverse2 = inverse * 1.44269504088896340736;
        shift = 63 - (32 - __clz(int((n - 1u) | 1u)));
    }
};

// v plus what lane moves of both halves bring (0 where they bring nothing).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t plus_moved(uint64_t v) {
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(v)), CTRL, ROWS, 0xf, false));
    const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(v >> 32)), CTRL, ROWS, 0xf, false));
    return v + (uint64_t(hi) << 32 | lo);
}
// The sum over the lanes up to this one (all 64 active): within rows of 16, then the row ends handed on.
__device__ __forceinline__ uint64_t wave_upto(uint64_t v) {
    v = plus_moved<0x111, 0xf>(v);      // row_shr 1, 2, 4, 8
    v = plus_moved<0x112, 0xf>(v);
    v = plus_moved<0x114, 0xf>(v);
    v = plus_moved<0x118, 0xf>(v);
    v = plus_moved<0x142, 0xa>(v);      // row_bcast 15 into rows 1 and 3
    return plus_moved<0x143, 0xc>(v);   // row_bcast 31 into rows 2 and 3
}

// Scores crowd into some fifty bins: four copies of each keep the lanes of a wave from waiting for each other (ten million
// scores in one row, a histogram of masses: 17.2 ms with one copy).
constexpr uint32_t kCopies = 4;
struct SampleShared {
    uint64_t part[kSampleWaves], found_mass;
    uint32_t part32[kSampleWaves], listed, picked, found_count, last;
    uint32_t count[kBins * kCopies];
    uint64_t mass[kBins * kCopies];
    uint64_t list[kListed];       // (last: kernels that list nothing leave it out)
};

__device__ uint64_t block_sum(uint64_t v, SampleShared &sh) {
    v = wave_upto(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 63u) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t all = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) all += sh.part[w];
    return all;
}
// The sum over the threads before this one; `all` the sum over all of them.
__device__ uint64_t block_before(uint64_t v, SampleShared &sh, uint64_t &all) {
    const uint32_t wave = threadIdx.x >> 6;
    const uint64_t upto = wave_upto(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 63u) sh.part[wave] = upto;
    __syncthreads();
    uint64_t before = upto - v;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < uint32_t(kSampleWaves); ++w) {
        const uint64_t x = sh.part[w];
        before += w < wave ? x : 0;
        all += x;
    }
    return before;
}

// Sorts up to kSorted different words, none of them 0, falling, by counting those above each.
__device__ void sort_falling(uint64_t *x, uint32_t size) {
    __syncthreads();
    const uint64_t mine = threadIdx.x < size ? x[threadIdx.x] : 0;
    uint32_t above = 0;
    if (mine != 0)
        for (uint32_t i = 0; i < size; ++i) above += uint32_t(x[i] > mine);
    __syncthreads();
    if (mine != 0) x[above] = mine;
    __syncthreads();
}

// In slot order, the first slot whose f, summed up to it from lo on, exceeds `want`; it is one of the `len` from lo on.  All threads return it.
template <typename T, typename F>
__device__ uint32_t locate_in(const SampleRow<T> &row, SampleShared &sh, uint32_t lo, uint32_t len, uint64_t want, F &&f) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    while (len > uint32_t(kSampleThreads)) {
        const uint32_t seg = ((len + kSampleWaves - 1) / kSampleWaves + 63u) & ~63u;
        const uint32_t from = min(len, wave * seg), to = min(len, from + seg);
        uint64_t sum = 0;
        row.each(lo + from, lo + to, lane, 64u, [&](uint32_t i, uint32_t k) { if (k != kNoKey) sum += f(i, k); });
        sum = wave_upto(sum);
        __syncthreads();
        if (lane == 63u) sh.part[wave] = sum;
        __syncthreads();
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
// f summed over the slots lo .. hi - 1.
template <typename T, typename F>
__device__ uint64_t sum_of(const SampleRow<T> &row, SampleShared &sh, uint32_t lo, uint32_t hi, F &&f) {
    uint64_t sum = 0;
    row.each(lo, hi, threadIdx.x, kSampleThreads, [&](uint32_t i, uint32_t k) { if (k != kNoKey) sum += f(i, k); });
    return block_sum(sum, sh);
}

// What a threshold is looked for by: its keys lo .. hi, how many slots have one of them, and what lies above.
struct Range {
    uint32_t lo, hi, count;
    uint64_t count_before, mass_before;
};

template <bool MASS>
__device__ void clear_bins(SampleShared &sh) {
    __syncthreads();
#pragma unroll
    for (uint32_t c = 0; c < kCopies; ++c) {
        sh.count[c * kBins + threadIdx.x] = 0;
        if (MASS) sh.mass[c * kBins + threadIdx.x] = 0;
    }
    __syncthreads();
}
// One histogram: of the slots lo .. hi - 1 whose keys lie in r, the bins by bin_of.
template <bool MASS, typename T, typename B>
__device__ void fill_bins(const SampleRow<T> &row, SampleShared &sh, const Range &r, uint32_t lo, uint32_t hi, B &&bin_of) {
    clear_bins<MASS>(sh);
    const uint32_t copy = threadIdx.x % kCopies;
    row.each(lo, hi, threadIdx.x, kSampleThreads, [&](uint32_t, uint32_t k) {
        if (k < r.lo || k > r.hi) return;
        const uint32_t at = bin_of(k) * kCopies + copy;
        atomicAdd(&sh.count[at], 1u);
        if (MASS) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[at]), (unsigned long long)row.units(k));
    });
    __syncthreads();
}
// A thread's bin, all copies.
template <bool MASS>
__device__ __forceinline__ void own_bin(const SampleShared &sh, uint32_t &count, uint64_t &mass) {
    count = 0;
    mass = 0;
#pragma unroll
    for (uint32_t c = 0; c < kCopies; ++c) {
        count += sh.count[threadIdx.x * kCopies + c];
        if (MASS) mass += sh.mass[threadIdx.x * kCopies + c];
    }
}
// The last bin that has slots and that reaches(count before, mass before) says yes to; r's counts become that bin's, total the mass of all.
template <bool MASS, typename F>
__device__ uint32_t pick_bin(SampleShared &sh, Range &r, uint32_t count, uint64_t mass, F &&reaches, uint64_t &total) {
    const uint32_t t = threadIdx.x;
    if (t == 0) sh.picked = 0;
    uint64_t all;
    const uint64_t count_before = r.count_before + block_before(count, sh, all);
    const uint64_t mass_before = MASS ? r.mass_before + block_before(mass, sh, total) : 0;
    if (count != 0 && (t == 0 || reaches(count_before, mass_before))) atomicMax(&sh.picked, t);
    __syncthreads();
    const uint32_t pick = sh.picked;
    if (t == pick) { sh.found_count = uint32_t(count_before); sh.found_mass = mass_before; sh.listed = count; }
    __syncthreads();
    r.count = sh.listed;
    r.count_before = sh.found_count;
    r.mass_before = sh.found_mass;
    return pick;
}
template <bool MASS, typename T, typename B, typename F>
__device__ uint32_t pick_bin(const SampleRow<T> &row, SampleShared &sh, Range &r, B &&bin_of, F &&reaches, uint64_t &total) {
    fill_bins<MASS>(row, sh, r, 0, row.n, bin_of);
    uint32_t count;
    uint64_t mass;
    own_bin<MASS>(sh, count, mass);
    return pick_bin<MASS>(sh, r, count, mass, reaches, total);
}
// The keys of bin b of the histogram that narrows r, whose bins are 2^shift keys each.
__device__ __forceinline__ uint32_t narrow_shift(const Range &r) { return uint32_t(max(0, 22 - __clz(int(r.hi - r.lo)))); }
__device__ __forceinline__ void narrow_to(Range &r, uint32_t b, uint32_t shift) {
    r.hi -= b << shift;
    r.lo = max(r.lo, r.hi - min(r.hi, (1u << shift) - 1u));
}

// Lists the slots of from .. to - 1 whose keys lie in lo .. hi, kListed at most; returns how many.
template <typename T>
__device__ uint32_t list_slots(const SampleRow<T> &row, SampleShared &sh, uint32_t from, uint32_t to, uint32_t lo, uint32_t hi) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    row.each(from, to, threadIdx.x, kSampleThreads, [&](uint32_t i, uint32_t k) {
        if (k < lo || k > hi) return;
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kListed) sh.list[at] = uint64_t(k) << 32 | uint32_t(~i);
    });
    __syncthreads();
    return min(sh.listed, kListed);
}
// A thread's slots of the list.
struct Listed {
    uint32_t key[kListedEach], place[kListedEach];      // place: the complement of the slot, which falls as the slot rises
    uint64_t mass[kListedEach];
    bool in[kListedEach];
    template <bool MASS, typename T>
    __device__ __forceinline__ void take(const SampleRow<T> &row, const SampleShared &sh, uint32_t listed) {
#pragma unroll
        for (uint32_t j = 0; j < kListedEach; ++j) {
            const uint32_t e = j * kSampleThreads + threadIdx.x;
            in[j] = e < listed;
            const uint64_t x = in[j] ? sh.list[e] : 0;
            key[j] = uint32_t(x >> 32);
            place[j] = uint32_t(x);
            mass[j] = MASS && in[j] ? row.units(key[j]) : 0;
        }
    }
};
// Narrows r to one value v: the last, in falling order, that has slots that are in and that reaches(count before, mass before) says yes to.
template <bool MASS, typename F>
__device__ void narrow_listed(SampleShared &sh, const Listed &l, const uint32_t (&v)[kListedEach], Range &r, F &&reaches) {
    do {      // (once at least: r's count may not be known yet)
        const uint32_t shift = narrow_shift(r), copy = threadIdx.x % kCopies;
        clear_bins<MASS>(sh);
#pragma unroll
        for (uint32_t j = 0; j < kListedEach; ++j) {
            if (!l.in[j] || v[j] < r.lo || v[j] > r.hi) continue;
            const uint32_t at = ((r.hi - v[j]) >> shift) * kCopies + copy;
            atomicAdd(&sh.count[at], 1u);
            if (MASS) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[at]), (unsigned long long)l.mass[j]);
        }
        __syncthreads();
        uint32_t count;
        uint64_t mass, total;
        own_bin<MASS>(sh, count, mass);
        narrow_to(r, pick_bin<MASS>(sh, r, count, mass, reaches, total), shift);
    } while (r.lo < r.hi);
}
// The slot up to which `ties` of those that are in and have this key lie.
__device__ uint32_t last_tie(SampleShared &sh, Listed l, uint32_t key, uint32_t ties) {
#pragma unroll
    for (uint32_t j = 0; j < kListedEach; ++j) l.in[j] &= l.key[j] == key;
    Range r{0u, ~0u, 0, 0, 0};
    narrow_listed<false>(sh, l, l.place, r, [&](uint64_t c, uint64_t) { return c < uint64_t(ties); });
    return ~r.lo;
}

// Narrows r to one key: the last, in falling order, that has slots and that reaches(count before, mass before) says yes to.
template <bool MASS, typename T, typename F>
__device__ void narrow(const SampleRow<T> &row, SampleShared &sh, Range &r, F &&reaches) {
    uint64_t total;
    while (r.lo < r.hi && r.count > kListed) {
        const uint32_t hi = r.hi, shift = narrow_shift(r);
        const uint32_t b = pick_bin<MASS>(row, sh, r, [=](uint32_t k) { return (hi - k) >> shift; }, reaches, total);
        narrow_to(r, b, shift);
    }
    if (r.lo == r.hi) return;
    Listed l;
    l.take<MASS>(row, sh, list_slots(row, sh, 0, row.n, r.lo, r.hi));
    narrow_listed<MASS>(sh, l, l.key, r, reaches);
}

__device__ __forceinline__ uint64_t drawn_mass(float u, uint64_t sum) {
    const double want = double(u) * double(sum);
    return want >= double(sum) ? sum - 1 : want > 0.0 ? uint64_t(want) : uint64_t(0);
}

// Draws from the slots of sh.list: of the first top_k in the order of their rank (0: all), those that less than a limit of mass lies before
// (limit_p), and of those the ones of at least min_key.  The limit is top_p of the mass of the first top_k, or given.
struct ListLimits {
    uint32_t top_k, min_key;
    bool limit_p;
    double top_p, limit;
    float u;
};

// Few slots: sorted by rank, then, what stays of them, by slot.
template <typename T>
__device__ void draw_sorted(const SampleRow<T> &row, SampleShared &sh, uint32_t listed, ListLimits lim, int64_t &slot, float &prob) {
    const uint32_t t = threadIdx.x;
    sort_falling(sh.list, listed);
    if (lim.top_k != 0) listed = min(listed, lim.top_k);
    const uint64_t x = t < listed ? sh.list[t] : 0;
    const uint32_t key = uint32_t(x >> 32);
    const uint64_t mass = x != 0 ? row.units(key) : 0;
    uint64_t all, total;
    const uint64_t before = block_before(mass, sh, all);
    if (lim.top_k != 0) lim.limit = lim.top_p * double(all);
    const bool stays = x != 0 && (t == 0 || ((!lim.limit_p || double(before) < lim.limit) && key >= lim.min_key));
    // (what stays is a prefix: min-p and top-p both leave one)
    block_before(stays, sh, all);
    const uint32_t kept = uint32_t(all);
    if (stays) sh.list[t] = uint64_t(uint32_t(x)) << 32 | key;
    sort_falling(sh.list, kept);
    const uint64_t y = t < kept ? sh.list[t] : 0;
    const uint64_t own = y != 0 ? row.units(uint32_t(y)) : 0, upto = block_before(own, sh, total), want = drawn_mass(lim.u, total);
    if (t == 0) sh.picked = 0;
    __syncthreads();
    if (upto <= want && upto + own > want) sh.picked = t;
    __syncthreads();
    const uint64_t z = sh.list[sh.picked];
    slot = int64_t(~uint32_t(z >> 32));
    prob = float(ldexp(row.weight(uint32_t(z)), row.shift) / double(total));
}

template <typename T>
__device__ void draw_from_list(const SampleRow<T> &row, SampleShared &sh, uint32_t listed, ListLimits lim, int64_t &slot, float &prob) {
    if (listed <= kSorted) return draw_sorted(row, sh, listed, lim, slot, prob);
    Listed l;
    l.take<true>(row, sh, listed);
    uint64_t sum;
    const auto mass_in = [&] {
        sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < kListedEach; ++j) sum += l.in[j] ? l.mass[j] : 0;
        return block_sum(sum, sh);
    };
    const auto keep = [&](uint32_t least, uint32_t count, uint32_t ties) {
        const uint32_t last = ties < count ? last_tie(sh, l, least, ties) : ~0u;
#pragma unroll
        for (uint32_t j = 0; j < kListedEach; ++j) l.in[j] &= l.key[j] > least || (l.key[j] == least && ~l.place[j] <= last);
    };
    if (lim.top_k != 0) {
        if (listed > lim.top_k) {
            Range r{kNoKey + 1u, row.most, 0, 0, 0};
            narrow_listed<false>(sh, l, l.key, r, [&](uint64_t c, uint64_t) { return c < uint64_t(lim.top_k); });
            keep(r.lo, r.count, min(r.count, uint32_t(uint64_t(lim.top_k) - r.count_before)));
        }
        lim.limit = lim.top_p * double(mass_in());
    }
    if (lim.limit_p) {
        Range r{kNoKey + 1u, row.most, 0, 0, 0};
        narrow_listed<true>(sh, l, l.key, r, [&](uint64_t c, uint64_t m) { return c == 0 || double(m) < lim.limit; });
        if (r.lo < lim.min_key) {
            r.lo = lim.min_key;
            r.count = 0;
        }
        keep(r.lo, r.count, ties_within(row, r, lim.limit));
    } else {
        keep(lim.min_key, 0, 0);
    }
    const uint64_t total = mass_in(), want = drawn_mass(lim.u, total);
    Range r{0u, ~0u, 0, 0, 0};
    narrow_listed<true>(sh, l, l.place, r, [&](uint64_t c, uint64_t m) { return c == 0 || m <= want; });
    slot = int64_t(~r.lo);
    prob = float(ldexp(row.weight(row.key_at(~r.lo)), row.shift) / double(total));
}

// A row's parameters.
struct Limits {
    int32_t top_k;
    float top_p, u;
    bool limit_k, limit_p;
    uint32_t min_key;
    float t, min_p;
    __device__ __forceinline__ void load(const SampleArgs &p, uint32_t r) {
        t = p.temperature == nullptr ? 1.0f : p.temperature[r];
        min_p = p.min_p == nullptr ? 0.0f : p.min_p[r];
        top_k = p.top_k == nullptr ? 0 : p.top_k[r];
        top_p = p.top_p == nullptr ? 1.0f : p.top_p[r];
        u = p.u[r];
        if (!(t > 0.0f)) { top_k = 1; top_p = 1.0f; }       // the best alone
    }
    template <typename T>
    __device__ __forceinline__ void set(SampleRow<T> &row, uint32_t most) {
        row.set(most, t);
        limit_k = top_k > 0 && uint32_t(top_k) < row.n;
        limit_p = top_p < 1.0f;
        min_key = min_p > 0.0f ? row.least_of_weight(double(min_p), double(t)) : kNoKey + 1u;
    }
};

// How many of r's slots, which all have its one key, stay: those that less than `limit` of mass lies before.
template <typename T>
__device__ __forceinline__ uint32_t ties_within(const SampleRow<T> &row, const Range &r, double limit) {
    const uint64_t each = row.units(r.lo);
    const double fit = each == 0 ? double(r.count) : ceil((limit - double(r.mass_before)) / double(each));
    return fit < 1.0 ? 1u : fit < double(r.count) ? uint32_t(fit) : r.count;
}

template <typename T>
__device__ void sample_row(const SampleRow<T> &row, SampleShared &sh, const Limits &lim, int64_t &slot, float &prob) {
    const int32_t top_k = lim.top_k;
    const float top_p = lim.top_p, u = lim.u;
    const bool limit_k = lim.limit_k, limit_p = lim.limit_p;
    const uint32_t min_key = lim.min_key;
    const auto first_k = [&](uint64_t c, uint64_t) { return c < uint64_t(top_k); };
    uint64_t total = 0;
    uint32_t least = kNoKey + 1u, equal = 0, ties = 0;      // slots of a higher key stay, and so many of those of this one
    if (limit_k) {
        Range all{kNoKey + 1u, row.most, 0, 0, 0};
        const uint32_t b = pick_bin<false>(row, sh, all, [&](uint32_t k) { return row.bin(k); }, first_k, total);
        all.lo = row.least_of_bin(b);
        if (all.count_before + all.count <= kListed) {
            const uint32_t listed = list_slots(row, sh, 0, row.n, all.lo, row.most);
            return draw_from_list(row, sh, listed, ListLimits{uint32_t(top_k), min_key, limit_p, double(top_p), 0.0, u}, slot, prob);
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
            const uint64_t above = sum_of(row, sh, 0, row.n, [&](uint32_t, uint32_t k) { return k > least ? row.units(k) : uint64_t(0); });
            limit = double(top_p) * double(above + row.units(least) * ties);
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
                const uint32_t listed = list_slots(row, sh, 0, row.n, from, row.most);
                if (sh.listed <= kListed) return draw_from_list(row, sh, listed, ListLimits{0u, min_key, true, 0.0, limit, u}, slot, prob);
            }
        }
        if (b != 0) all.hi = row.least_of_bin(b - 1) - 1u;
        narrow<true>(row, sh, all, first_p);
        const uint32_t stay = ties_within(row, all, limit);
        // (never below top-k's class: the mass up to its end is all that top-k left, or more)
        ties = limit_k && all.lo == least ? min(stay, ties) : stay;
        least = all.lo;
        equal = all.count;
    }
    uint32_t tie_last = ~0u;
    if (ties < equal) {
        tie_last = locate_in(row, sh, 0, row.n, ties - 1u, [&](uint32_t, uint32_t k) { return uint64_t(k == least); });
    }
    const auto kept = [&](uint32_t i, uint32_t k) { return k < least || k < min_key || (k == least && i > tie_last) ? uint64_t(0) : row.units(k); };
    total = sum_of(row, sh, 0, row.n, kept);
    const uint32_t at = locate_in(row, sh, 0, row.n, drawn_mass(u, total), kept);
    slot = at;
    prob = float(ldexp(row.weight(row.key_at(at)), row.shift) / double(total));
}

template <typename T>
__device__ __forceinline__ SampleRow<T> row_of(const SampleArgs &p, uint32_t r) {
    SampleRow<T> row;
    row.scores = static_cast<const T *>(p.scores) + size_t(r) * p.stride;
    row.mask = p.mask == nullptr ? nullptr : p.mask + size_t(r) * p.mask_stride;
    row.n = p.n;
    return row;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, SampleShared &sh) {
    v = wave_umax(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) sh.part32[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < kSampleWaves; ++w) v = max(v, sh.part32[w]);
    return v;
}

// Short rows, and many: a workgroup to a row.
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample(SampleArgs p) {
    extern __shared__ uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    for (uint32_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        SampleRow<T> row = row_of<T>(p, r);
        Limits lim;
        lim.load(p, r);
        uint32_t most = kNoKey;
        row.each(0, p.n, threadIdx.x, kSampleThreads, [&](uint32_t, uint32_t k) { most = max(most, k); });
        most = block_max(most, sh);
        int64_t slot = -1;
        float prob = 0.0f;
        if (most != kNoKey) {
            lim.set(row, most);
            sample_row(row, sh, lim, slot, prob);
        }
        if (threadIdx.x == 0) { p.out_slots[r] = slot; p.out_probs[r] = prob; }
        __syncthreads();
    }
}

// Long rows, not many: a row goes in chunks to workgroups, through six kernels that each walk it once at most.
//   max     the best score of each chunk
//   bins    the histogram, added up over the row's chunks; where nothing limits the row, the mass of each chunk
//   list    few slots down to the threshold's bin: gathered.  Many: the bin's own histogram.  Where nothing limits the row, the draw.
//   narrow  a draw from the gathered slots, by the first chunk; or the slots of the second histogram's bin.  (top-k that leaves many and
//           top-p together: the first chunk takes the row alone.)
//   mass    the threshold from the slots of that bin, by each chunk for itself; what stays in the chunk
//   draw    from those masses, by the first chunk
// A kernel's chunks add to what lies in the workspace with whole numbers, so that their order does not show.  What they hand on passes from
// kernel to kernel: handing it to the last chunk to finish, within one, takes a write-back of the XCD's cache a chunk, which made
// 256 rows of 100K take 448 us in one kernel where a launch takes 2.
struct SampleSplit {
    // zeroed by the first kernel
    uint64_t mass[2][kBins];
    uint32_t count[2][kBins];
    uint32_t listed, state, least, tie_last;
    uint64_t list[kListed];
};
constexpr uint32_t kSplitZeroed = offsetof(SampleSplit, list) / 4;
enum { kRowOpen = 0, kRowDone = 1, kRowThreshold = 2 };
struct SplitArgs {
    SampleSplit *rows;
    uint64_t *chunk_mass;     // [row][chunk]
    uint2 *chunk_cut;         // the threshold's key, and the last slot of that key that stays
    uint32_t *chunk_most;
    uint32_t chunk, chunks;   // slots of a chunk, chunks of a row
};

// A chunk of a row, and what every kernel but the first knows of the row.
template <typename T>
struct Chunk {
    SampleRow<T> row;
    Limits lim;
    SampleSplit *ws;
    uint32_t r, c, from, to, most;
    __device__ __forceinline__ Chunk(const SampleArgs &p, const SplitArgs &x)
        : row(row_of<T>(p, blockIdx.x)), ws(x.rows + blockIdx.x), r(blockIdx.x), c(blockIdx.y), from(blockIdx.y * x.chunk), to(min(p.n, from + x.chunk)) {}
    __device__ __forceinline__ bool open(const SampleArgs &p, const SplitArgs &x, SampleShared &sh) {
        lim.load(p, r);
        most = kNoKey;
        for (uint32_t i = threadIdx.x; i < x.chunks; i += kSampleThreads) most = max(most, x.chunk_most[size_t(r) * x.chunks + i]);
        most = block_max(most, sh);
        if (most == kNoKey) return false;
        lim.set(row, most);
        return true;
    }
    __device__ __forceinline__ void write(const SampleArgs &p, int64_t slot, float prob) const {
        if (threadIdx.x == 0) { p.out_slots[r] = slot; p.out_probs[r] = prob; ws->state = kRowDone; }
    }
};

template <bool MASS>
__device__ void add_bins(SampleShared &sh, SampleSplit *ws, int which) {
    uint32_t count;
    uint64_t mass;
    own_bin<MASS>(sh, count, mass);
    if (count == 0) return;
    atomicAdd(&ws->count[which][threadIdx.x], count);
    if (MASS) atomicAdd(reinterpret_cast<unsigned long long *>(&ws->mass[which][threadIdx.x]), (unsigned long long)mass);
}

// The row's draw from the masses of its chunks.
template <typename T, typename F>
__device__ void draw_by_chunks(const SampleArgs &p, const SplitArgs &x, const Chunk<T> &ch, SampleShared &sh, F &&kept) {
    const uint64_t *const masses = x.chunk_mass + size_t(ch.r) * x.chunks;
    uint64_t sum = 0;
    for (uint32_t i = threadIdx.x; i < x.chunks; i += kSampleThreads) sum += masses[i];
    const uint64_t total = block_sum(sum, sh);
    uint64_t want = drawn_mass(ch.lim.u, total), before = 0;
    if (threadIdx.x == 0) { sh.picked = 0; sh.found_mass = 0; }
    for (uint32_t i = 0; i < x.chunks; i += kSampleThreads) {
        const uint64_t mine = i + threadIdx.x < x.chunks ? masses[i + threadIdx.x] : 0;
        uint64_t all;
        const uint64_t upto = before + block_before(mine, sh, all);
        if (upto <= want && upto + mine > want) { sh.picked = i + threadIdx.x; sh.found_mass = upto; }
        before += all;
    }
    __syncthreads();
    const uint32_t c = sh.picked, lo = c * x.chunk;
    want -= sh.found_mass;
    __syncthreads();
    const uint32_t at = locate_in(ch.row, sh, lo, min(x.chunk, p.n - lo), want, kept);
    ch.write(p, at, float(ldexp(ch.row.weight(ch.row.key_at(at)), ch.row.shift) / double(total)));
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_max(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    const Chunk<T> ch(p, x);
    for (uint32_t i = ch.c * kSampleThreads + threadIdx.x; i < kSplitZeroed; i += x.chunks * kSampleThreads) reinterpret_cast<uint32_t *>(ch.ws)[i] = 0;
    uint32_t most = kNoKey;
    ch.row.each(ch.from, ch.to, threadIdx.x, kSampleThreads, [&](uint32_t, uint32_t k) { most = max(most, k); });
    most = block_max(most, sh);
    if (threadIdx.x == 0) x.chunk_most[size_t(ch.r) * x.chunks + ch.c] = most;
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_bins(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    Chunk<T> ch(p, x);
    if (!ch.open(p, x, sh)) {
        if (ch.c == 0) ch.write(p, -1, 0.0f);
        return;
    }
    const Range all{kNoKey + 1u, ch.most, 0, 0, 0};
    const auto bin_of = [&](uint32_t k) { return ch.row.bin(k); };
    if (ch.lim.limit_k) {
        fill_bins<false>(ch.row, sh, all, ch.from, ch.to, bin_of);
        add_bins<false>(sh, ch.ws, 0);
    } else if (ch.lim.limit_p) {
        fill_bins<true>(ch.row, sh, all, ch.from, ch.to, bin_of);
        add_bins<true>(sh, ch.ws, 0);
    } else {
        const uint32_t min_key = ch.lim.min_key;
        const uint64_t mass = sum_of(ch.row, sh, ch.from, ch.to, [&](uint32_t, uint32_t k) { return k < min_key ? uint64_t(0) : ch.row.units(k); });
        if (threadIdx.x == 0) x.chunk_mass[size_t(ch.r) * x.chunks + ch.c] = mass;
    }
}

// The bin b that the histogram leaves the threshold in, as keys from its least one up to the row's largest.  limit: of top-p's mass.  upto: slots
// down to that bin, or to min-p's.
template <bool MASS, typename T>
__device__ Range first_range(const Chunk<T> &ch, SampleShared &sh, double &limit, uint32_t &upto, uint32_t &b) {
    const uint32_t count = ch.ws->count[0][threadIdx.x];
    const uint64_t mass = MASS ? ch.ws->mass[0][threadIdx.x] : 0;
    uint64_t total = 0;
    Range r{kNoKey + 1u, ch.most, 0, 0, 0};
    b = pick_bin<MASS>(sh, r, count, mass,
        [&](uint64_t c, uint64_t m) { return MASS ? c == 0 || double(m) < double(ch.lim.top_p) * double(total) : c < uint64_t(ch.lim.top_k); }, total);
    limit = double(ch.lim.top_p) * double(total);
    const uint32_t down_to = MASS ? min(b, ch.row.bin(ch.lim.min_key)) : b;
    upto = uint32_t(min(block_sum(threadIdx.x <= down_to ? count : 0, sh), uint64_t(0xffffffffu)));
    r.lo = ch.row.least_of_bin(b);
    return r;
}

// Whether so few slots are left that the row is drawn from them.
__device__ __forceinline__ bool listable(uint32_t upto) { return upto <= kListed; }

// Adds the chunk's slots with keys lo .. hi to the row's list, which has room for them.
template <typename T>
__device__ void add_slots(const Chunk<T> &ch, SampleShared &sh, uint32_t lo, uint32_t hi) {
    const uint32_t listed = list_slots(ch.row, sh, ch.from, ch.to, lo, hi);
    if (threadIdx.x == 0) sh.found_count = listed == 0u ? 0u : atomicAdd(&ch.ws->listed, listed);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < listed; i += kSampleThreads)
        if (sh.found_count + i < kListed) ch.ws->list[sh.found_count + i] = sh.list[i];
}
// The row's list.
template <typename T>
__device__ uint32_t take_list(const Chunk<T> &ch, SampleShared &sh) {
    const uint32_t listed = min(ch.ws->listed, kListed);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < listed; i += kSampleThreads) sh.list[i] = ch.ws->list[i];
    __syncthreads();
    return listed;
}

template <bool MASS, typename T>
__device__ void list_chunk(Chunk<T> &ch, SampleShared &sh) {
    double limit;
    uint32_t upto, b;
    Range r = first_range<MASS>(ch, sh, limit, upto, b);
    if (listable(upto)) return add_slots(ch, sh, MASS ? max(r.lo, ch.lim.min_key) : r.lo, ch.most);
    if (ch.lim.limit_k && ch.lim.limit_p) return;
    if (b != 0) r.hi = ch.row.least_of_bin(b - 1) - 1u;
    const uint32_t shift = narrow_shift(r);
    fill_bins<MASS>(ch.row, sh, r, ch.from, ch.to, [&](uint32_t k) { return (r.hi - k) >> shift; });
    add_bins<MASS>(sh, ch.ws, 1);
}
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_list(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    Chunk<T> ch(p, x);
    if (!ch.open(p, x, sh)) return;
    if (ch.lim.limit_k) return list_chunk<false>(ch, sh);
    if (ch.lim.limit_p) return list_chunk<true>(ch, sh);
    const uint32_t min_key = ch.lim.min_key;
    if (ch.c == 0) draw_by_chunks(p, x, ch, sh, [&](uint32_t, uint32_t k) { return k < min_key ? uint64_t(0) : ch.row.units(k); });
}

// The range that the second histogram leaves.
template <bool MASS, typename T, typename F>
__device__ Range second_range(const Chunk<T> &ch, SampleShared &sh, Range r, uint32_t b, F &&reaches) {
    if (b != 0) r.hi = ch.row.least_of_bin(b - 1) - 1u;
    uint64_t total;
    const uint32_t shift = narrow_shift(r);
    narrow_to(r, pick_bin<MASS>(sh, r, ch.ws->count[1][threadIdx.x], MASS ? ch.ws->mass[1][threadIdx.x] : 0, reaches, total), shift);
    return r;
}
template <bool MASS, typename T>
__device__ __forceinline__ uint32_t ties_of(const Chunk<T> &ch, const Range &r, double limit) {
    return MASS ? ties_within(ch.row, r, limit) : min(r.count, uint32_t(uint64_t(ch.lim.top_k) - r.count_before));
}

template <bool MASS, typename T>
__device__ void narrow_chunk(const SampleArgs &p, Chunk<T> &ch, SampleShared &sh) {
    const Limits &lim = ch.lim;
    double limit;
    uint32_t upto, b;
    int64_t slot;
    float prob;
    Range r = first_range<MASS>(ch, sh, limit, upto, b);
    if (listable(upto)) {
        if (ch.c != 0) return;
        const uint32_t listed = take_list(ch, sh);
        draw_from_list(ch.row, sh, listed, MASS ? ListLimits{0u, lim.min_key, true, 0.0, limit, lim.u} : ListLimits{uint32_t(lim.top_k), lim.min_key, lim.limit_p, double(lim.top_p), 0.0, lim.u}, slot, prob);
        return ch.write(p, slot, prob);
    }
    if (lim.limit_k && lim.limit_p) {
        if (ch.c != 0) return;
        sample_row(ch.row, sh, lim, slot, prob);
        return ch.write(p, slot, prob);
    }
    const auto reaches = [&](uint64_t c, uint64_t m) { return MASS ? c == 0 || double(m) < limit : c < uint64_t(lim.top_k); };
    r = second_range<MASS>(ch, sh, r, b, reaches);
    if (r.count <= kListed) return add_slots(ch, sh, r.lo, r.hi);
    // more than that with keys next to each other: one workgroup goes on
    if (ch.c != 0) return;
    narrow<MASS>(ch.row, sh, r, reaches);
    const uint32_t ties = ties_of<MASS>(ch, r, limit), key = r.lo;
    const uint32_t last = ties < r.count ? locate_in(ch.row, sh, 0, ch.row.n, ties - 1u, [&](uint32_t, uint32_t k) { return uint64_t(k == key); }) : ~0u;
    if (threadIdx.x == 0) { ch.ws->least = key; ch.ws->tie_last = last; ch.ws->state = kRowThreshold; }
}
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_narrow(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    Chunk<T> ch(p, x);
    if (!ch.open(p, x, sh)) return;
    if (ch.lim.limit_k) narrow_chunk<false>(p, ch, sh);
    else if (ch.lim.limit_p) narrow_chunk<true>(p, ch, sh);
}

template <bool MASS, typename T>
__device__ void find_threshold(const Chunk<T> &ch, SampleShared &sh, uint32_t &least, uint32_t &tie_last) {
    const Limits &lim = ch.lim;
    double limit;
    uint32_t upto, b;
    Range r = first_range<MASS>(ch, sh, limit, upto, b);
    const auto reaches = [&](uint64_t c, uint64_t m) { return MASS ? c == 0 || double(m) < limit : c < uint64_t(lim.top_k); };
    r = second_range<MASS>(ch, sh, r, b, reaches);
    Listed l;
    l.take<MASS>(ch.row, sh, take_list(ch, sh));
    narrow_listed<MASS>(sh, l, l.key, r, reaches);
    const uint32_t ties = ties_of<MASS>(ch, r, limit);
    least = r.lo;
    tie_last = ties < r.count ? last_tie(sh, l, least, ties) : ~0u;
}
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_mass(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    Chunk<T> ch(p, x);
    if (ch.ws->state == kRowDone || !ch.open(p, x, sh)) return;
    uint32_t least, tie_last;
    if (ch.ws->state == kRowThreshold) { least = ch.ws->least; tie_last = ch.ws->tie_last; }
    else if (ch.lim.limit_k) find_threshold<false>(ch, sh, least, tie_last);
    else find_threshold<true>(ch, sh, least, tie_last);
    const uint32_t min_key = ch.lim.min_key;
    const uint64_t mass = sum_of(ch.row, sh, ch.from, ch.to,
        [&](uint32_t i, uint32_t k) { return k < least || k < min_key || (k == least && i > tie_last) ? uint64_t(0) : ch.row.units(k); });
    if (threadIdx.x != 0) return;
    x.chunk_mass[size_t(ch.r) * x.chunks + ch.c] = mass;
    x.chunk_cut[size_t(ch.r) * x.chunks + ch.c] = make_uint2(least, tie_last);
}
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_draw(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    Chunk<T> ch(p, x);
    if (ch.ws->state == kRowDone || !ch.open(p, x, sh)) return;
    const uint2 cut = x.chunk_cut[size_t(ch.r) * x.chunks];
    const uint32_t min_key = ch.lim.min_key;
    draw_by_chunks(p, x, ch, sh, [&](uint32_t i, uint32_t k) { return k < cut.x || k < min_key || (k == cut.x && i > cut.y) ? uint64_t(0) : ch.row.units(k); });
}

// Rows of more slots than this go in chunks, as long as there are no more than kSplitRows of them.
constexpr size_t kSplitSlots = 16384, kSplitRows = 512;
constexpr uint32_t kChunk = 8192;
struct Split {
    uint32_t chunk, chunks;
    size_t masses, cuts, mosts, bytes;
};
static Split split_of(size_t rows, size_t n) {
    // chunks for a thousand workgroups
    size_t chunk = kChunk;
    while (rows * ((n + chunk - 1) / chunk) > 1024 && chunk < n) chunk *= 2;
    Split x;
    x.chunk = uint32_t(chunk);
    x.chunks = uint32_t((n + chunk - 1) / chunk);
    x.masses = rows * sizeof(SampleSplit);
    x.cuts = x.masses + rows * x.chunks * 8;
    x.mosts = x.cuts + rows * x.chunks * 8;
    x.bytes = x.mosts + rows * x.chunks * 4;
    return x;
}
static bool splits(size_t rows, size_t n) { return n > kSplitSlots && rows <= kSplitRows; }
size_t sample_workspace(size_t rows, size_t n) { return splits(rows, n) ? split_of(rows, n).bytes : 0; }

template <typename T>
static hipError_t sample(const SampleArgs &a, hipStream_t s) {
    const size_t lds = sizeof(SampleShared), unlisted = offsetof(SampleShared, list);
    if (!splits(a.rows, a.n)) {
        if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(k_sample<T>), lds); e != hipSuccess) return e;
        return launch(k_sample<T>, a.rows < 65536u ? a.rows : 65536u, kSampleThreads, lds, s, a);
    }
    const Split split = split_of(a.rows, a.n);
    const SplitArgs x{reinterpret_cast<SampleSplit *>(a.ws), reinterpret_cast<uint64_t *>(a.ws + split.masses), reinterpret_cast<uint2 *>(a.ws + split.cuts),
                      reinterpret_cast<uint32_t *>(a.ws + split.mosts),
                      split.chunk, split.chunks};
    const dim3 grid(a.rows, split.chunks);      // (rows next to each other: their first chunks, which work alone at times, on all XCDs)
    const auto go = [&](void (*kernel)(SampleArgs, SplitArgs), dim3 g, size_t bytes) {
        const hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), bytes);
        return e != hipSuccess ? e : launch(kernel, g, kSampleThreads, bytes, s, a, x);
    };
    if (const hipError_t e = go(k_sample_max<T>, grid, unlisted); e != hipSuccess) return e;
    if (const hipError_t e = go(k_sample_bins<T>, grid, unlisted); e != hipSuccess) return e;
    if (const hipError_t e = go(k_sample_list<T>, grid, lds); e != hipSuccess) return e;
    if (a.top_k == nullptr && a.top_p == nullptr && a.temperature == nullptr) return hipSuccess;      // nothing limits any row
    if (const hipError_t e = go(k_sample_narrow<T>, grid, lds); e != hipSuccess) return e;
    if (const hipError_t e = go(k_sample_mass<T>, grid, lds); e != hipSuccess) return e;
    return go(k_sample_draw<T>, dim3(a.rows), unlisted);
}
hipError_t launch_sample(const SampleArgs &a, int score_type, hipStream_t s) {
    if (score_type == kF32) return sample<float>(a, s);
    return score_type == kF16 ? sample<f16>(a, s) : sample<bf16>(a, s);
}

}  // namespace tv
