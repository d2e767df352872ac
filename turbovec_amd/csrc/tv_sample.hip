// Drawing a slot from rows of scores, with temperature, top-k, top-p and min-p, from given random numbers.
//
// The weight of a slot is exp((score - max) / T), taken in 64 bits and held in whole units of 2^-shift (what is left over is dropped), shift = 63 -
// ceil(log2 n): sums of any number of them fit 64 bits and do not depend on the order of the additions, so that a draw is the same
// whatever order threads arrive in.  What top-k, top-p and min-p leave is a prefix of the slots ranked by score, ties to the lower
// slot: the slots above some score, and the first few of those that have it.
//
// All of it is one kind of search: of values in falling order (keys of scores, or complements of slots), the last one before which less
// than so many slots, or so much mass, lies.  A histogram of 1024 bins narrows the values to one bin, the next one divides that.  The first
// histogram of a row goes by the distance to the best score, its bins widening with it; where the slots down to the bin it finds are
// few, they are gathered, and everything else happens among them.  Top-k's slots are gathered without it where the best scores of the threads tell
// which (list_top), top-p's where min-p does (list_kept).  Bound by the passes over the row, two to six, and the exponentials (20 64-bit
// instructions each); a single row by what a pass takes at least, and by the fetching of its own instructions (one loop serves every
// search for that).  256 rows of 100000 bfloat16 scores, top-p 0.95 and min-p 0.001: 89 to 92 us, top-k 50 and top-p 0.9: 43; one row of 100000, top-k 50 and top-p 0.9: 29 to
// 34; ten million, half of them masked, top-p 0.5: 103.
#include <algorithm>

#include "tv_device.h"
#include "tv_ops.h"

namespace tv {

constexpr int kSampleWaves = 16, kSampleThreads = kSampleWaves * 64;      // of a row that is not short
constexpr uint32_t kNoKey = 0x007fffffu;     // -infinity's; what is not allowed has it too
constexpr uint32_t kListed = 4000;           // slots that are gathered of a row in chunks, at most: two workgroups' LDS to a compute unit

// The same value in all lanes, said to the compiler: it keeps it in scalar registers and branches on it without masks.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return uint32_t(__builtin_amdgcn_readfirstlane(int(v))); }
__device__ __forceinline__ uint64_t uniform(uint64_t v) { return uint64_t(uniform(uint32_t(v >> 32))) << 32 | uniform(uint32_t(v)); }
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(uniform(__float_as_uint(v))); }
__device__ __forceinline__ double uniform(double v) { return __longlong_as_double((long long)(uniform(uint64_t(__double_as_longlong(v))))); }

// The scores' order as unsigned numbers; -0 counts as +0, NaN as -infinity.
__device__ __forceinline__ uint32_t score_key(float s) {
    return s > -__int_as_float(0x7f800000) ? uint32_t(order_key(s + 0.0f)) ^ 0x80000000u : kNoKey;
}
__device__ __forceinline__ float key_score(uint32_t k) { return order_unkey(int(k ^ 0x80000000u)); }

// a * b + c, c the same in all lanes.  (The compiler copies each coefficient first, to add into it.)
__device__ __forceinline__ double fma_of(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

template <typename T>
struct SampleRow {
    static constexpr int kEach = 16 / int(sizeof(T));
    const T *scores;
    const uint64_t *mask;
    uint32_t n, most;         // most: the key of the largest score
    float best;               // that score
    double top, inverse, inverse2;      // the same, 1 / T, and that times log2(e)
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
    __device__ __forceinline__ uint32_t key_at(uint32_t i) const {
        return mask == nullptr || ((mask[i >> 6] >> (i & 63u)) & 1u) ? score_key(float(scores[i])) : kNoKey;
    }
    // f(slot, score, whether it counts) for the slots of lo .. hi - 1 (multiples of kEach, or the end), a worker of `workers`: those count that
    // are allowed and whose score is neither NaN nor -infinity.
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
            for (int j = 0; j < kEach; ++j) {
                const float v = float(now.v[j]);
                f(i + j, v, ((now.bits >> j) & 1u) != 0u && v > -__int_as_float(0x7f800000));
            }
            if (!more) return;
            now = next;
            i += step;
        }
    }
    // The same, four loads at a time, for a pass that does little with a score: one load at a time it waits for each.
    template <typename F>
    __device__ __forceinline__ void scan(uint32_t lo, uint32_t hi, uint32_t worker, uint32_t workers, F &&f) const {
        const uint32_t step = workers * kEach;
        uint32_t i = lo + worker * kEach;
        for (; i < hi && hi - i >= 3u * step + kEach; i += 4u * step) {
            Load l[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                l[a].bits = mask == nullptr ? ~0u : uint32_t(mask[(i + a * step) >> 6] >> ((i + a * step) & 63u));
                __builtin_memcpy(l[a].v, scores + i + a * step, 16);
            }
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int j = 0; j < kEach; ++j) {
                    const float v = float(l[a].v[j]);
                    f(i + a * step + j, v, ((l[a].bits >> j) & 1u) != 0u && v > -__int_as_float(0x7f800000));
                }
        }
        each(i, hi, 0, workers, f);
    }
    // exp((score - max) / T); for scores whose largest is +infinity, 1 for those that have it
    __device__ __forceinline__ double weight(uint32_t k) const { return k == most ? 1.0 : exp((double(key_score(k)) - top) * inverse); }
    // The same in whole units of 2^-shift, which is what sums are made of: 2^y = 2^e * 2^f, |f| <= 1/2, with the exponential series up to
    // its ninth power (off by 7e-12 at most), then its high and its low 32 bits.  A library exponential and a conversion to 64 bits
    // take three times as long.
    __device__ __forceinline__ uint64_t units(float score) const {
        if (!(best < __int_as_float(0x7f800000))) return score == best ? 1ull << shift : 0ull;
        constexpr double k1 = 0.69314718055994530942, k2 = k1 * k1 / 2, k3 = k2 * k1 / 3, k4 = k3 * k1 / 4, k5 = k4 * k1 / 5, k6 = k5 * k1 / 6, k7 = k6 * k1 / 7,
                         k8 = k7 * k1 / 8, k9 = k8 * k1 / 9;
        const double y = (double(score) - top) * inverse2, e = rint(y), f = y - e;
        double v = fma_of(k9, f, k8);
        v = fma_of(v, f, k7);
        v = fma_of(v, f, k6);
        v = fma_of(v, f, k5);
        v = fma_of(v, f, k4);
        v = fma_of(v, f, k3);
        v = fma_of(v, f, k2);
        v = fma_of(v, f, k1);
        v = ldexp(fma(v, f, 1.0), int(e) + (shift - 32));
        const uint32_t hi = uint32_t(v);
        return uint64_t(hi) << 32 | uint32_t((v - double(hi)) * 4294967296.0);
    }
    // How far a score lies below the best, as the bits of that distance: a number that rises with it.
    __device__ __forceinline__ uint32_t distance(float v) const { return v == best ? 0u : __float_as_uint(best - v); }
    // The least key no further than d (keys rise as distances fall): among the 64 around best - d, a lane each; where rounding has put it further
    // away, every lane tries one of 64 places, until a step is one key.
    __device__ __forceinline__ uint32_t least_within(uint32_t d) const {
        const uint32_t base = min(max(score_key(best - __uint_as_float(d)) - 32u, kNoKey + 1u), most);
        const uint64_t near = uniform(uint64_t(__ballot(distance(key_score(min(base + (threadIdx.x & 63u), most))) <= d)));
        if (near != 0ull && ((near & 1u) == 0u || base == kNoKey + 1u)) return base + uint32_t(__builtin_ctzll(near));
        uint32_t lo = kNoKey + 1u, left = most - lo;           // it is one of lo .. lo + left
        while (left != 0u) {
            const uint32_t step = left / 64u + 1u, mine = lo + min(left, (threadIdx.x & 63u) * step);
            const uint64_t yes = uniform(uint64_t(__ballot(distance(key_score(mine)) <= d)));
            const uint32_t first = yes == 0ull ? 64u : uint32_t(__builtin_ctzll(yes));
            if (first == 0u) return lo;
            // above the place before the first that is, and no further
            const uint32_t under = lo + min(left, (first - 1u) * step), upto = first == 64u ? lo + left : lo + min(left, first * step);
            left = upto - (under + 1u);
            lo = under + 1u;
        }
        return lo;
    }
    // The least key whose weight is min_p (above 0) or more; t is above 0.
    __device__ __forceinline__ uint32_t least_of_weight(double min_p, double t) const {
        if (min_p >= 1.0 || !(top < __longlong_as_double(0x7ff0000000000000ll))) return most;
        const double from = top + log(min_p) * t;
        const uint32_t k = score_key(float(from));
        return min(max(k + (k != kNoKey && double(float(from)) < from ? 1u : 0u), kNoKey + 1u), most);
    }
    // Of a row's scores, given the largest one's key.
    __device__ __forceinline__ void set(uint32_t most_, float t) {
        most = most_;
        best = key_score(most);
        top = uniform(double(best));
        // (an infinite best leaves the others nothing)
        inverse = t > 0.0f && top < __longlong_as_double(0x7ff0000000000000ll) ? uniform(1.0 / double(t)) : 1.0;
        inverse2 = uniform(inverse * 1.44269504088896340736);
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
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t plus_moved(uint32_t v) {
    return v + uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xf, false));
}
// The sum over the lanes up to this one (all 64 active): within rows of 16, then the row ends handed on.
template <typename N>
__device__ __forceinline__ N wave_upto(N v) {
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
// What a workgroup of W waves shares; a bin to a thread.  ROOM: for so many bins, so that fewer waves find the list in the same place.
template <int W, uint32_t MOST = kListed, uint32_t ROOM = 64 * W>
struct SampleShared {
    static constexpr uint32_t kThreads = 64 * W, kBins = kThreads, kBits = W == 16 ? 10 : W == 4 ? 8 : 0, kMost = MOST;
    static_assert(kBins == 1u << kBits, "a bin to a thread");
    uint64_t part[ROOM / 64], found_mass;
    uint32_t part32[ROOM / 64], listed, picked, found_count, found_before, found_down, found_value;
    uint32_t count[ROOM * kCopies];
    uint64_t mass[ROOM * kCopies];
    uint64_t list[MOST];          // key, complement of the slot.  (Last: what lies within 64 KiB is addressed at no cost.)
    // The bin of a distance: 32 of 1024 for each power of two that it spans, from 2^-20 to 2^12; what is nearer or further is in the first or the
    // last.
    static constexpr int kDistance = 28 - int(kBits), kFirstBin = (127 - 20) << (int(kBits) - 5);
    __device__ __forceinline__ static uint32_t bin(uint32_t d) { return uint32_t(min(max(int(d >> kDistance) - kFirstBin, 0), int(kBins) - 1)); }
    __device__ __forceinline__ static uint32_t nearest(uint32_t bin) { return bin == 0 ? 0u : uint32_t(kFirstBin + int(bin)) << kDistance; }
    __device__ __forceinline__ static uint32_t furthest(uint32_t bin) { return bin == kBins - 1 ? 0x7f800000u : nearest(bin + 1) - 1u; }
    // That many values fall into bins of 2^this.
    __device__ __forceinline__ static uint32_t shift_of(uint32_t range) { return uint32_t(max(0, 32 - int(kBits) - __clz(int(range)))); }
};
// Slots of a thread from which on its best one tells enough for list_top.  (Top-k 10 and top-p 0.9, 256 rows: of 4000 21 us without and 18 with it, of
// 15000 26 and 22; rows of 1000 16 either way.)
constexpr uint32_t kTopEach = 4;
constexpr uint32_t kShortListed = 2048;     // five workgroups' LDS to a compute unit
constexpr uint32_t kRowListed = 8000;        // a compute unit has one workgroup of sixteen waves
using LongShared = SampleShared<kSampleWaves>;
using BinsShared = SampleShared<kSampleWaves, 1>;      // of kernels that list nothing

// The sum over the threads before this one; `all` the sum over all of them.
template <int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ uint64_t block_before(uint64_t v, SampleShared<W, MOST, ROOM> &sh, uint64_t &all) {
    const uint32_t wave = threadIdx.x >> 6;
    const uint64_t upto = wave_upto(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 63u) sh.part[wave] = upto;
    __syncthreads();
    uint64_t before = upto - v;
    all = 0;
    for (uint32_t w = 0; w < uint32_t(W); ++w) {
        const uint64_t x = sh.part[w];
        before += w < wave ? x : 0;
        all += x;
    }
    all = uniform(all);
    return before;
}
template <int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ uint64_t block_sum(uint64_t v, SampleShared<W, MOST, ROOM> &sh) {
    uint64_t all;
    block_before(v, sh, all);
    return all;
}
template <int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ uint32_t block_max(uint32_t v, SampleShared<W, MOST, ROOM> &sh) {
    v = wave_umax(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) sh.part32[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < W; ++w) v = max(v, sh.part32[w]);
    return uniform(v);
}

// A row's parameters.
struct Limits {
    int32_t top_k;
    float top_p, u, t, min_p;
    bool limit_k, limit_p;
    uint32_t min_key;
    __device__ __forceinline__ void load(const SampleArgs &p, uint32_t r) {
        t = p.temperature == nullptr ? 1.0f : uniform(p.temperature[r]);
        min_p = p.min_p == nullptr ? 0.0f : uniform(p.min_p[r]);
        top_k = p.top_k == nullptr ? 0 : int32_t(uniform(uint32_t(p.top_k[r])));
        top_p = p.top_p == nullptr ? 1.0f : uniform(p.top_p[r]);
        u = uniform(p.u[r]);
        if (!(t > 0.0f)) { top_k = 1; top_p = 1.0f; min_p = 0.0f; }       // the best alone
    }
    template <typename T>
    __device__ __forceinline__ void set(SampleRow<T> &row, uint32_t most) {
        row.set(most, t);
        limit_k = top_k > 0 && uint32_t(top_k) < row.n;
        limit_p = top_p < 1.0f;
        min_key = min_p > 0.0f ? uniform(row.least_of_weight(double(min_p), double(t))) : kNoKey + 1u;
    }
};

// What stays: slots of keys above `least`, and of those of that key the ones up to tie_last.
struct Cut {
    uint32_t least, tie_last;
};
struct CutScores {
    float least;
    uint32_t tie_last;
    __device__ __forceinline__ explicit CutScores(const Cut &c) : least(key_score(c.least)), tie_last(c.tie_last) {}
    __device__ __forceinline__ bool leaves(uint32_t i, float v) const { return v > least || (v == least && i <= tie_last); }
};
// The values that the one sought is among, in falling order from hi: keys of scores, near to far within distances `near` to `far`, or complements of
// slots.  Of a bin that was picked: its slots, and the slots and the mass before it.
struct Search {
    uint32_t lo, hi, near, far, count;
    uint64_t before, mass_before;
};

enum { kFirst, kByDistance, kByKey, kByPlace };
struct Pass {
    int mode;
    bool mass, ties;          // ties: of the cut's slots only those of its least key
};
// A histogram of the cut's slots whose values lie in s: of those of the list, or those lo .. hi - 1 of the row.
template <typename T, int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ void fill(const SampleRow<T> &row, SampleShared<W, MOST, ROOM> &sh, bool listed, uint32_t lo, uint32_t hi, const Cut &cut, const Search &s, const Pass &pass) {
    __syncthreads();
#pragma unroll
    for (uint32_t c = 0; c < kCopies; ++c) {
        sh.count[c * sh.kBins + threadIdx.x] = 0;
        if (pass.mass) sh.mass[c * sh.kBins + threadIdx.x] = 0;
    }
    __syncthreads();
    const CutScores scores(cut);
    const uint32_t by_distance = sh.shift_of(s.far - s.near), by_value = sh.shift_of(s.hi - s.lo), copy = threadIdx.x % kCopies;
    const auto add = [&](uint32_t i, float v, bool in) {
        in = in && scores.leaves(i, v);
        uint32_t bin;
        if (pass.mode <= kByDistance) {
            const uint32_t d = row.distance(v);
            bin = sh.bin(d);
            if (pass.mode == kByDistance) {
                in = in && d >= s.near && d <= s.far;
                bin = (d - s.near) >> by_distance;
            }
        } else {
            const uint32_t x = pass.mode == kByPlace ? ~i : score_key(v);
            in = in && x >= s.lo && x <= s.hi && (!pass.ties || v == scores.least);
            bin = (s.hi - x) >> by_value;
        }
        if (!in) return;
        const uint32_t at = bin * kCopies + copy;
        atomicAdd(&sh.count[at], 1u);
        if (pass.mass) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[at]), (unsigned long long)row.units(v));
    };
    if (listed) {
#pragma unroll 1
        for (uint32_t e = threadIdx.x; e < hi; e += sh.kThreads) add(~uint32_t(sh.list[e]), key_score(uint32_t(sh.list[e] >> 32)), true);
    } else {
        row.each(lo, hi, threadIdx.x, sh.kThreads, add);
    }
    __syncthreads();
}
// A thread's bin, all copies.
template <int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ void own_bin(const SampleShared<W, MOST, ROOM> &sh, bool with_mass, uint32_t &count, uint64_t &mass) {
    count = 0;
    mass = 0;
#pragma unroll
    for (uint32_t c = 0; c < kCopies; ++c) {
        count += sh.count[threadIdx.x * kCopies + c];
        if (with_mass) mass += sh.mass[threadIdx.x * kCopies + c];
    }
}

__device__ __forceinline__ uint64_t drawn_mass(float u, uint64_t sum) {
    const double want = double(u) * double(sum);
    return want >= double(sum) ? sum - 1 : want > 0.0 ? uint64_t(want) : uint64_t(0);
}
__device__ __forceinline__ uint64_t top_p_bound(const Limits &lim, uint64_t sum) { return uniform(uint64_t(ceil(fmax(double(lim.top_p), 0.0) * double(sum)))); }
// A row's searches, one after the other.
enum { kTopK, kTopP, kTies, kDraw };
struct State {
    int phase, after;         // after: the phase that ends in ties
    bool whole;               // the search has not been narrowed yet
    int histograms;           // of the row by distance so far; two, then by key
    bool listed, bin_only;    // bin_only: the list holds one bin's slots, not all from there up
    uint32_t n;               // slots in the list
    Search s;
    Cut cut;
    uint64_t bound, total;    // total: the mass of what the phase's first histogram counted
};
__device__ __forceinline__ bool by_mass(int phase) { return phase == kTopP || phase == kDraw; }

// Of the bins, a thread each, the last that has slots and that less than the bound lies before; the first one always.  `down`: the slots down to
// it, or to the bin `cap` if that comes before.
template <int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ uint32_t pick(SampleShared<W, MOST, ROOM> &sh, State &st, const Limits &lim, uint32_t count, uint64_t mass, uint32_t cap, uint32_t &down) {
    const uint32_t t = threadIdx.x, wave = t >> 6;
    const bool masses = by_mass(st.phase);
    const uint32_t counts = wave_upto(count);
    const uint64_t sums = masses ? wave_upto(mass) : 0;
    __syncthreads();
    if (t == 0) sh.picked = 0;
    if ((t & 63u) == 63u) { sh.part32[wave] = counts; sh.part[wave] = sums; }
    __syncthreads();
    uint32_t before = counts - count;
    for (uint32_t w = 0; w < wave; ++w) before += sh.part32[w];
    uint64_t upto = st.s.before + before, mass_before = 0;
    if (masses) {
        uint64_t all = 0;
        mass_before = st.s.mass_before + sums - mass;
        for (uint32_t w = 0; w < uint32_t(W); ++w) {
            const uint64_t x = sh.part[w];
            mass_before += w < wave ? x : 0;
            all += x;
        }
        upto = mass_before;
        if (st.whole) {
            st.total = all = uniform(all);
            st.bound = st.phase == kTopP ? top_p_bound(lim, all) : uniform(drawn_mass(lim.u, all)) + 1;
        }
    }
    if (count != 0 && (st.s.before + before == 0 || upto < st.bound)) atomicMax(&sh.picked, t);
    __syncthreads();
    const uint32_t bin = uniform(sh.picked);
    if (t == bin) { sh.found_count = count; sh.found_before = uint32_t(st.s.before) + before; sh.found_mass = mass_before; }
    if (t == min(bin, cap)) sh.found_down = uint32_t(st.s.before) + before + count;
    __syncthreads();
    st.s.count = uniform(sh.found_count);
    st.s.before = uniform(sh.found_before);
    st.s.mass_before = uniform(sh.found_mass);
    st.whole = false;
    down = uniform(sh.found_down);
    return bin;
}

// Lists the cut's slots of lo .. hi - 1 whose keys are from .. upto, sh.kMost at most; returns how many.
template <typename T, int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ uint32_t list_slots(const SampleRow<T> &row, SampleShared<W, MOST, ROOM> &sh, uint32_t lo, uint32_t hi, const Cut &cut, uint32_t from, uint32_t upto) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    const CutScores scores(cut);
    const float least = key_score(from), most = key_score(upto);
    row.scan(lo, hi, threadIdx.x, sh.kThreads, [&](uint32_t i, float v, bool in) {
        if (!in || v < least || v > most || !scores.leaves(i, v)) return;
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < sh.kMost) sh.list[at] = uint64_t(score_key(v)) << 32 | uint32_t(~i);
    });
    __syncthreads();
    return uniform(min(sh.listed, sh.kMost));
}
// The one value in s of the list's slots that count; where min-p has kept it out of the list, the least that would be there.
template <int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ uint32_t only_value(SampleShared<W, MOST, ROOM> &sh, const State &st) {
    if (threadIdx.x == 0) sh.found_value = st.s.lo;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < st.n; e += sh.kThreads) {
        const uint32_t k = uint32_t(sh.list[e] >> 32), place = uint32_t(sh.list[e]), v = st.phase >= kTies ? place : k;
        const bool stays = k > st.cut.least || (k == st.cut.least && ~place <= st.cut.tie_last);
        if (v >= st.s.lo && v <= st.s.hi && stays && (st.phase != kTies || k == st.cut.least)) sh.found_value = v;
    }
    __syncthreads();
    const uint32_t v = uniform(sh.found_value);
    __syncthreads();
    return v;
}

// Of the cut's slots from lo on (ties: those of its least key, each counting 1; otherwise their mass), in slot order the first that the sum up to it
// exceeds `want` at; it is one of the `len` from lo on.
template <typename T, int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ uint32_t locate(const SampleRow<T> &row, SampleShared<W, MOST, ROOM> &sh, uint32_t lo, uint32_t len, const Cut &cut, bool ties, uint64_t want, bool draws = false,
                                           float u = 0.0f, uint64_t *total = nullptr) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const CutScores scores(cut);
    const auto value = [&](uint32_t i, float v, bool in) {
        in = in && scores.leaves(i, v);
        if (__ballot(in) == 0ull) return uint64_t(0);
        const uint64_t x = ties ? uint64_t(v == scores.least) : row.units(v);
        return in ? x : uint64_t(0);
    };
    while (len > sh.kThreads) {
        const uint32_t seg = ((len + uint32_t(W) - 1) / W + 63u) & ~63u;
        const uint32_t from = min(len, wave * seg), to = min(len, from + seg);
        uint64_t sum = 0;
        row.each(lo + from, lo + to, lane, 64u, [&](uint32_t i, float v, bool in) { sum += value(i, v, in); });
        sum = wave_upto(sum);
        __syncthreads();
        if (lane == 63u) sh.part[wave] = sum;
        __syncthreads();
        if (draws) {
            uint64_t all = 0;
            for (uint32_t w = 0; w < uint32_t(W); ++w) all += uniform(sh.part[w]);
            *total = all;
            want = uniform(drawn_mass(u, all));
            draws = false;
        }
        uint32_t w = 0;
        uint64_t upto = uniform(sh.part[0]), before = 0;
        while (w + 1 < uint32_t(W) && upto <= want) {
            before = upto;
            upto += uniform(sh.part[++w]);
        }
        want -= before;
        lo += min(len, w * seg);
        len = min(seg, len - min(len, w * seg));
        __syncthreads();
    }
    uint64_t mine = 0;
    if (threadIdx.x < len) {
        const uint32_t k = row.key_at(lo + threadIdx.x);
        mine = value(lo + threadIdx.x, key_score(k), k != kNoKey);
    }
    uint64_t all;
    const uint64_t before = block_before(mine, sh, all);
    if (draws) {
        *total = all;
        want = uniform(drawn_mass(u, all));
    }
    if (threadIdx.x == 0) sh.picked = 0;
    __syncthreads();
    if (before <= want && before + mine > want) sh.picked = threadIdx.x;
    __syncthreads();
    return lo + uniform(sh.picked);
}
// The mass that the cut leaves of the slots lo .. hi - 1 that are this worker's.
template <typename T>
__device__ __forceinline__ uint64_t mass_of(const SampleRow<T> &row, uint32_t lo, uint32_t hi, uint32_t worker, uint32_t workers, const Cut &cut) {
    const CutScores scores(cut);
    uint64_t sum = 0;
    row.each(lo, hi, worker, workers, [&](uint32_t i, float v, bool in) {
        in = in && scores.leaves(i, v);
        if (__ballot(in) == 0ull) return;
        const uint64_t x = row.units(v);
        sum += in ? x : 0;
    });
    return sum;
}

template <typename T>
__device__ __forceinline__ State first_state(const SampleRow<T> &row, const Limits &lim) {
    State st;
    st.phase = lim.limit_k ? kTopK : lim.limit_p ? kTopP : kDraw;
    st.after = kDraw;
    st.whole = true;
    st.histograms = 0;
    st.listed = st.bin_only = false;
    st.n = 0;
    st.s = Search{kNoKey + 1u, row.most, 0, ~0u, 0, 0, 0};
    st.cut = Cut{kNoKey + 1u, ~0u};
    st.bound = uint64_t(lim.top_k);
    st.total = 0;
    return st;
}
// The search goes from a histogram by distance to the bin it picked.
template <typename T, int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ void to_bin(const SampleRow<T> &row, const SampleShared<W, MOST, ROOM> &sh, State &st, uint32_t bin) {
    Search &s = st.s;
    if (st.histograms++ == 0) {
        s.near = sh.nearest(bin);
        s.far = sh.furthest(bin);
    } else {
        const uint32_t shift = sh.shift_of(s.far - s.near);
        s.near += bin << shift;
        s.far = min(s.far, s.near + ((1u << shift) - 1u));
    }
    s.lo = max(st.cut.least, row.least_within(s.far));
    s.hi = s.near == 0 ? row.most : row.least_within(s.near - 1u) - 1u;
}
// The last bin of the first histogram that can matter for what is drawn.  (Min-p leaves fewer, but top-p after top-k needs all of top-k's.)
template <typename T, int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ uint32_t last_bin(const SampleRow<T> &row, const SampleShared<W, MOST, ROOM> &sh, const State &st, const Limits &lim) {
    return st.phase == kTopP ? sh.bin(row.distance(key_score(lim.min_key))) : sh.kBins - 1;
}
// From which key on a row's slots are listed.  Where min-p leaves nothing of the bin, the search is over.
__device__ __forceinline__ uint32_t list_from(State &st, const Limits &lim) {
    if (st.phase != kTopP || lim.min_key <= st.s.lo) return st.s.lo;
    st.s.lo = min(lim.min_key, st.s.hi);
    if (lim.min_key > st.s.hi) st.s.count = 0;
    return lim.min_key;
}

// Gathers what is in the bin, or, of few slots down to it, those from there up; where there are few.
template <typename T, int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ bool list_bin(const SampleRow<T> &row, SampleShared<W, MOST, ROOM> &sh, State &st, const Limits &lim, uint32_t down) {
    if (down > sh.kMost && st.s.count > sh.kMost) return false;
    st.bin_only = down > sh.kMost;
    const uint32_t from = list_from(st, lim), upto = st.bin_only ? st.s.hi : row.most;
    st.n = from > upto ? 0 : list_slots(row, sh, 0, row.n, st.cut, from, upto);
    st.listed = true;
    return true;
}

// Top-k's slots and a few more, without a histogram of the row: of its threads' best scores (each of slots of its own) as many as k
// reach down to some bin, so that many slots do too.  False where that leaves too many, or fewer threads than k have a slot.
template <typename T, int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ bool list_top(const SampleRow<T> &row, SampleShared<W, MOST, ROOM> &sh, const Limits &lim, State &st, float own_best) {
    __syncthreads();
#pragma unroll
    for (uint32_t c = 0; c < kCopies; ++c) sh.count[c * sh.kBins + threadIdx.x] = 0;
    __syncthreads();
    if (own_best > -__int_as_float(0x7f800000)) atomicAdd(&sh.count[sh.bin(row.distance(own_best)) * kCopies + threadIdx.x % kCopies], 1u);
    __syncthreads();
    uint32_t count, down;
    uint64_t mass;
    own_bin(sh, false, count, mass);
    State of_threads = st;
    const uint32_t bin = pick(sh, of_threads, lim, count, 0, sh.kBins - 1, down);
    if (down < uint32_t(lim.top_k)) return false;
    to_bin(row, sh, of_threads, bin);
    st.n = list_slots(row, sh, 0, row.n, st.cut, of_threads.s.lo, row.most);
    if (uniform(sh.listed) > sh.kMost) return false;
    st.s.lo = of_threads.s.lo;
    st.listed = true;
    return true;
}

// What min-p leaves, listed along with the sum of all masses, which is what top-p goes by.  False where that is too much.
template <typename T, int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ bool list_kept(const SampleRow<T> &row, SampleShared<W, MOST, ROOM> &sh, const Limits &lim, State &st) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    const float least = key_score(lim.min_key);
    uint64_t sum = 0;
    row.each(0, row.n, threadIdx.x, sh.kThreads, [&](uint32_t i, float v, bool in) {
        if (__ballot(in) == 0ull) return;
        const uint64_t x = row.units(v);
        sum += in ? x : 0;
        if (!in || v < least) return;
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < sh.kMost) sh.list[at] = uint64_t(score_key(v)) << 32 | uint32_t(~i);
    });
    const uint64_t total = block_sum(sum, sh);
    const uint32_t listed = uniform(sh.listed);
    if (listed > sh.kMost) return false;
    st.total = total;
    st.bound = top_p_bound(lim, total);
    st.n = listed;
    st.listed = true;
    st.whole = false;
    st.s.lo = lim.min_key;
    st.s.count = listed;
    return true;
}

// The searches that are left, to the draw, or (to_cut) to the end of the one that st is in, or (to_list) to where the slots that can still be drawn
// are listed: then false.
template <typename T, int W, uint32_t MOST, uint32_t ROOM>
__device__ __forceinline__ bool search(const SampleRow<T> &row, SampleShared<W, MOST, ROOM> &sh, const Limits &lim, State &st, bool to_cut, bool to_list, int64_t &slot, float &prob) {
    while (true) {
        if (st.phase >= kTies && !st.listed) {
            // slots next to each other fall into one bin, a row's are walked instead
            st.s.lo = st.s.hi = ~locate(row, sh, 0, row.n, st.cut, st.phase == kTies, st.bound - 1, st.phase == kDraw, lim.u, &st.total);
        } else if (st.whole || (st.s.lo < st.s.hi && st.s.count != 0)) {
            const bool distances = !st.listed && st.histograms < 2, first = distances && st.histograms == 0;
            if (!st.whole && st.listed && st.s.count == 1) {
                st.s.lo = st.s.hi = only_value(sh, st);
                continue;
            }
            const int mode = first ? kFirst : distances ? kByDistance : st.phase >= kTies ? kByPlace : kByKey;
            fill(row, sh, st.listed, 0, st.listed ? st.n : row.n, st.cut, st.s, Pass{mode, by_mass(st.phase), st.phase == kTies});
            uint32_t count;
            uint64_t mass;
            own_bin(sh, by_mass(st.phase), count, mass);
            uint32_t down;
            const uint32_t bin = pick(sh, st, lim, count, mass, first ? last_bin(row, sh, st, lim) : sh.kBins - 1, down);
            if (!distances) {
                const uint32_t shift = sh.shift_of(st.s.hi - st.s.lo);
                st.s.hi -= bin << shift;
                st.s.lo = max(st.s.lo, st.s.hi - min(st.s.hi, (1u << shift) - 1u));
                continue;
            }
            to_bin(row, sh, st, bin);
            if (list_bin(row, sh, st, lim, down)) {
                if (to_list && !st.bin_only) return false;
            }
            continue;
        }
        // one value is left
        if (st.phase == kDraw) {
            slot = int64_t(~st.s.lo);
            prob = float(ldexp(row.weight(row.key_at(~st.s.lo)), row.shift) / double(st.total));
            return true;
        }
        int next = kDraw;
        if (st.phase == kTies) {
            st.cut.tie_last = ~st.s.lo;
            next = st.after;
        } else {
            next = st.phase == kTopK && lim.limit_p ? kTopP : kDraw;
            uint32_t ties = uint32_t(min(uint64_t(st.s.count), st.bound - min(st.bound, st.s.before)));
            if (st.phase == kTopP) {
                const uint64_t each = row.units(key_score(st.s.lo));
                const double fit = each == 0 ? double(st.s.count) : ceil((double(st.bound) - double(st.s.mass_before)) / double(each));
                ties = uniform(fit < 1.0 ? min(1u, st.s.count) : fit < double(st.s.count) ? uint32_t(fit) : st.s.count);
            }
            st.cut = Cut{st.s.lo, st.s.lo == st.cut.least ? st.cut.tie_last : ~0u};
            if (ties < st.s.count) {
                st.after = next;
                next = kTies;
                st.bound = ties;
            }
        }
        if (to_cut && next != kTies) return true;
        if (next == kDraw && lim.min_key > st.cut.least) st.cut = Cut{lim.min_key, ~0u};
        st.phase = next;
        if (next != kTies && st.bin_only) st.listed = st.bin_only = false;
        st.whole = true;
        st.histograms = 0;
        st.s = Search{st.cut.least, row.most, 0, ~0u, 0, 0, 0};
        if (next >= kTies) { st.s.lo = ~(row.n - 1u); st.s.hi = ~0u; }
    }
}

template <typename T>
__device__ __forceinline__ SampleRow<T> row_of(const SampleArgs &p, uint32_t r) {
    SampleRow<T> row;
    row.scores = static_cast<const T *>(p.scores) + size_t(r) * p.stride;
    row.mask = p.mask == nullptr ? nullptr : p.mask + size_t(r) * p.mask_stride;
    row.n = p.n;
    return row;
}

// Short rows, and many: a workgroup of W waves to a row.
template <typename T, int W, uint32_t MOST>
__global__ __launch_bounds__(64 * W) void k_sample(SampleArgs p) {
    extern __shared__ uint8_t smem[];
    SampleShared<W, MOST> &sh = *reinterpret_cast<SampleShared<W, MOST> *>(smem);
    for (uint32_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        SampleRow<T> row = row_of<T>(p, r);
        Limits lim;
        lim.load(p, r);
        float best = -__int_as_float(0x7f800000);
        row.scan(0, p.n, threadIdx.x, sh.kThreads, [&](uint32_t, float v, bool in) {
            if (in) best = fmaxf(best, v);
        });
        const uint32_t most = block_max(score_key(best), sh);
        int64_t slot = -1;
        float prob = 0.0f;
        if (most != kNoKey) {
            lim.set(row, most);
            State st = first_state(row, lim);
            if (st.phase == kDraw && lim.min_key > st.cut.least) st.cut.least = lim.min_key;
            const bool last = W == kSampleWaves && r + gridDim.x >= p.rows;
            const bool top = st.phase == kTopK && uint32_t(lim.top_k) <= sh.kThreads / 2 && p.n >= kTopEach * sh.kThreads && list_top(row, sh, lim, st, best);
            const bool kept = st.phase == kTopP && lim.min_key > kNoKey + 1u && list_kept(row, sh, lim, st);
            if (((top || kept) && last) || !search(row, sh, lim, st, false, last, slot, prob)) {
                // Four waves go on: they wait less for each other, and a barrier counts the waves that have not ended.
                SampleShared<4, MOST, 64 * W> &few = *reinterpret_cast<SampleShared<4, MOST, 64 * W> *>(smem);
                __syncthreads();
                if (threadIdx.x >= few.kThreads) return;
                search(row, few, lim, st, false, false, slot, prob);
            }
        }
        if (threadIdx.x == 0) { p.out_slots[r] = slot; p.out_probs[r] = prob; }
        __syncthreads();
    }
}

// Long rows, not many: a row goes in chunks to workgroups, through six kernels that each walk it once at most.
//   max     the best score of each chunk
//   bins    the first histogram, added up over the row's chunks; where nothing limits the row, the mass of each part of a chunk
//   list    few slots down to the bin it leaves: gathered.  Many: the bin's own histogram.  Where nothing limits the row, the draw.
//   narrow  the rest of the search among the gathered slots, by the first chunk; or, where the second histogram was made, its bin's slots
//   mass    the threshold from the slots of that bin, by each chunk for itself; what stays in the chunk.  Where that was top-k's and top-p follows,
//           top-p's first histogram
//   draw    from those masses, by the first chunk; or the rest of top-p's search (ten million, top-k 20000 and top-p 0.9: 3.3 of 3.4 ms)
// A kernel's chunks add to what lies in the workspace with whole numbers, so that their order does not show.  What they hand on passes from
// kernel to kernel: handing it to the last chunk to finish, within one, takes a write-back of the XCD's cache a chunk, which made
// 256 rows of 100K take 448 us in one kernel where a launch takes 2.
// Where a row's search stands between kernels.
struct Kept {
    uint32_t most, down;      // the key of the largest score, 0 where there is nothing to search; slots down to the bin (first_bin)
    Search s;
    uint64_t bound, total;
};
struct SampleSplit {
    // zeroed by the first kernel
    uint64_t mass[3][LongShared::kBins];
    uint32_t count[3][LongShared::kBins];
    uint32_t listed, state;
    Cut cut;
    Kept kept[2];             // after the first histogram; after the second, or the first where its bin's slots are listed
    uint64_t list[kListed];
};
constexpr uint32_t kSplitZeroed = offsetof(SampleSplit, list) / 4;
enum { kRowOpen = 0, kRowDone = 1, kRowCut = 2 };
struct SplitArgs {
    SampleSplit *rows;
    uint64_t *part_mass;      // [row][part]: kSampleWaves parts a chunk, a wave each
    Cut *chunk_cut;           // [row][chunk]
    uint32_t *chunk_most;
    uint32_t chunk, chunks;   // slots of a chunk, chunks of a row
};

// A chunk of a row, and what every kernel but the first knows of the row.
template <typename T>
struct Chunk {
    SampleRow<T> row;
    Limits lim;
    SampleSplit *ws;
    uint32_t r, c, from, to, most, count;
    uint64_t mass;            // count, mass: a thread's bin of the first histogram
    __device__ __forceinline__ Chunk(const SampleArgs &p, const SplitArgs &x)
        : row(row_of<T>(p, blockIdx.x)), ws(x.rows + blockIdx.x), r(blockIdx.x), c(blockIdx.y), from(blockIdx.y * x.chunk), to(min(p.n, from + x.chunk)) {}
    template <uint32_t MOST>
    __device__ __forceinline__ bool open(const SampleArgs &p, const SplitArgs &x, SampleShared<kSampleWaves, MOST> &sh, bool bins) {
        lim.load(p, r);
        most = kNoKey;
        count = bins ? ws->count[0][threadIdx.x] : 0;
        mass = bins ? ws->mass[0][threadIdx.x] : 0;
        for (uint32_t i = threadIdx.x; i < x.chunks; i += kSampleThreads) most = max(most, x.chunk_most[size_t(r) * x.chunks + i]);
        most = block_max(most, sh);
        if (most == kNoKey) return false;
        lim.set(row, most);
        return true;
    }
    __device__ __forceinline__ void keep(int at, const State &st, uint32_t down) const {
        if (c == 0 && threadIdx.x == 0) ws->kept[at] = Kept{most, down, st.s, st.bound, st.total};
    }
    // Instead of open() and first_bin(), in a kernel behind the one that kept it.
    __device__ __forceinline__ bool open_kept(const SampleArgs &p, int at, State &st, uint32_t &down) {
        const Kept k = ws->kept[at];
        most = uniform(k.most);
        if (most == 0u) return false;
        lim.load(p, r);
        lim.set(row, most);
        st = first_state(row, lim);
        st.whole = false;
        st.histograms = 1;
        st.s = Search{uniform(k.s.lo), uniform(k.s.hi), uniform(k.s.near), uniform(k.s.far), uniform(k.s.count), uniform(k.s.before), uniform(k.s.mass_before)};
        st.bound = uniform(k.bound);
        st.total = uniform(k.total);
        down = uniform(k.down);
        return true;
    }
    __device__ __forceinline__ void write(const SampleArgs &p, int64_t slot, float prob) const {
        if (threadIdx.x == 0) { p.out_slots[r] = slot; p.out_probs[r] = prob; ws->state = kRowDone; }
    }
    // After the first histogram.
    __device__ __forceinline__ State first_bin(LongShared &sh, uint32_t &down) {
        State st = first_state(row, lim);
        const uint32_t bin = pick(sh, st, lim, count, mass, last_bin(row, sh, st, lim), down);
        to_bin(row, sh, st, bin);
        return st;
    }
    __device__ __forceinline__ bool limited() const { return lim.limit_k || lim.limit_p; }
    __device__ __forceinline__ bool both() const { return lim.limit_k && lim.limit_p; }
};
// Top-p's search after top-k's cut.
template <typename T>
__device__ __forceinline__ State second_state(const Chunk<T> &ch, const Cut &cut) {
    State st = first_state(ch.row, ch.lim);
    st.phase = kTopP;
    st.cut = cut;
    st.s.lo = cut.least;
    return st;
}

template <typename T, uint32_t MOST>
__device__ __forceinline__ void add_bins(const Chunk<T> &ch, SampleShared<kSampleWaves, MOST> &sh, int which, bool with_mass) {
    uint32_t count;
    uint64_t mass;
    own_bin(sh, with_mass, count, mass);
    if (count == 0) return;
    atomicAdd(&ch.ws->count[which][threadIdx.x], count);
    if (with_mass) atomicAdd(reinterpret_cast<unsigned long long *>(&ch.ws->mass[which][threadIdx.x]), (unsigned long long)mass);
}
// Adds the chunk's slots with keys from .. upto to the row's list, which has room for them.
template <typename T>
__device__ __forceinline__ void add_slots(const Chunk<T> &ch, LongShared &sh, uint32_t from, uint32_t upto) {
    const uint32_t listed = list_slots(ch.row, sh, ch.from, ch.to, Cut{kNoKey + 1u, ~0u}, from, upto);
    if (threadIdx.x == 0) sh.found_count = listed == 0u ? 0u : atomicAdd(&ch.ws->listed, listed);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < listed; i += kSampleThreads)
        if (sh.found_count + i < kListed) ch.ws->list[sh.found_count + i] = sh.list[i];
}
// The search goes on among the row's list.
template <typename T, int W>
__device__ __forceinline__ void take_list(const Chunk<T> &ch, SampleShared<W> &sh, State &st) {
    st.n = uniform(min(ch.ws->listed, kListed));
    st.listed = true;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < st.n; i += sh.kThreads) sh.list[i] = ch.ws->list[i];
    __syncthreads();
}

// The mass of each part of the chunk.
template <typename T>
__device__ __forceinline__ void put_masses(const SplitArgs &x, const Chunk<T> &ch, const Cut &cut) {
    const uint32_t part = x.chunk / kSampleWaves, wave = threadIdx.x >> 6, lo = min(ch.to, ch.from + wave * part);
    const uint64_t mass = wave_upto(mass_of(ch.row, lo, min(ch.to, lo + part), threadIdx.x & 63u, 64u, cut));
    if ((threadIdx.x & 63u) == 63u) x.part_mass[(size_t(ch.r) * x.chunks + ch.c) * kSampleWaves + wave] = mass;
}
// The row's draw from those of its chunks.
template <typename T>
__device__ __forceinline__ void draw_by_parts(const SampleArgs &p, const SplitArgs &x, const Chunk<T> &ch, LongShared &sh, const Cut &cut) {
    // (a thread to parts that follow each other)
    const uint32_t parts = x.chunks * kSampleWaves, part = x.chunk / kSampleWaves, each = (parts + kSampleThreads - 1) / kSampleThreads;
    const uint64_t *const masses = x.part_mass + size_t(ch.r) * parts;
    uint32_t at_part = min(parts, threadIdx.x * each);
    uint64_t sum = 0, total;
    for (uint32_t i = at_part; i < min(parts, (threadIdx.x + 1u) * each); ++i) sum += masses[i];
    uint64_t before = block_before(sum, sh, total);
    uint64_t want = drawn_mass(ch.lim.u, total);
    if (threadIdx.x == 0) { sh.picked = 0; sh.found_mass = 0; }
    __syncthreads();
    if (before <= want && before + sum > want) {
        for (; before + masses[at_part] <= want; ++at_part) before += masses[at_part];
        sh.picked = at_part;
        sh.found_mass = before;
    }
    __syncthreads();
    const uint32_t lo = uniform(sh.picked) * part;
    want -= uniform(sh.found_mass);
    __syncthreads();
    const uint32_t at = locate(ch.row, sh, lo, min(part, p.n - lo), cut, false, want);
    ch.write(p, at, float(ldexp(ch.row.weight(ch.row.key_at(at)), ch.row.shift) / double(total)));
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_max(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    BinsShared &sh = *reinterpret_cast<BinsShared *>(smem);
    const Chunk<T> ch(p, x);
    for (uint32_t i = ch.c * kSampleThreads + threadIdx.x; i < kSplitZeroed; i += x.chunks * kSampleThreads) reinterpret_cast<uint32_t *>(ch.ws)[i] = 0;
    float best = -__int_as_float(0x7f800000);
    ch.row.scan(ch.from, ch.to, threadIdx.x, kSampleThreads, [&](uint32_t, float v, bool in) {
        if (in) best = fmaxf(best, v);
    });
    const uint32_t most = block_max(score_key(best), sh);
    if (threadIdx.x == 0) x.chunk_most[size_t(ch.r) * x.chunks + ch.c] = most;
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_bins(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    BinsShared &sh = *reinterpret_cast<BinsShared *>(smem);
    Chunk<T> ch(p, x);
    if (!ch.open(p, x, sh, false)) {
        if (ch.c == 0) ch.write(p, -1, 0.0f);
        return;
    }
    if (ch.limited()) {
        const State st = first_state(ch.row, ch.lim);
        fill(ch.row, sh, false, ch.from, ch.to, st.cut, st.s, Pass{kFirst, !ch.lim.limit_k, false});
        add_bins(ch, sh, 0, !ch.lim.limit_k);
    } else {
        put_masses(x, ch, Cut{ch.lim.min_key, ~0u});
    }
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_list(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    LongShared &sh = *reinterpret_cast<LongShared *>(smem);
    Chunk<T> ch(p, x);
    if (!ch.open(p, x, sh, true)) return;
    if (!ch.limited()) {
        if (ch.c == 0) draw_by_parts(p, x, ch, sh, Cut{ch.lim.min_key, ~0u});
        return;
    }
    uint32_t down;
    State st = ch.first_bin(sh, down);
    ch.keep(0, st, down);
    if (down <= kListed) return add_slots(ch, sh, list_from(st, ch.lim), ch.most);
    if (st.s.count <= kListed) return add_slots(ch, sh, st.s.lo, st.s.hi);
    fill(ch.row, sh, false, ch.from, ch.to, st.cut, st.s, Pass{kByDistance, by_mass(st.phase), false});
    add_bins(ch, sh, 1, by_mass(st.phase));
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_narrow(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    LongShared &sh = *reinterpret_cast<LongShared *>(smem);
    Chunk<T> ch(p, x);
    State st;
    uint32_t down;
    int64_t slot;
    float prob;
    if (!ch.open_kept(p, 0, st, down)) return;
    if (down <= kListed) {
        if (ch.c != 0) return;
        list_from(st, ch.lim);
        // Four waves go on: they wait less for each other, and a barrier counts the waves that have not ended.
        SampleShared<4> &few = *reinterpret_cast<SampleShared<4> *>(smem);
        if (threadIdx.x >= few.kThreads) return;
        take_list(ch, few, st);
        search(ch.row, few, ch.lim, st, false, false, slot, prob);
        return ch.write(p, slot, prob);
    }
    if (st.s.count <= kListed) return ch.keep(1, st, down);
    to_bin(ch.row, sh, st, pick(sh, st, ch.lim, ch.ws->count[1][threadIdx.x], ch.ws->mass[1][threadIdx.x], sh.kBins - 1, down));
    ch.keep(1, st, down);
    if (st.s.count <= kListed) return add_slots(ch, sh, st.s.lo, st.s.hi);
    // more than that with keys next to each other: one workgroup goes on
    if (ch.c != 0) return;
    search(ch.row, sh, ch.lim, st, true, false, slot, prob);
    if (threadIdx.x == 0) { ch.ws->cut = st.cut; ch.ws->state = kRowCut; }
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_mass(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    LongShared &sh = *reinterpret_cast<LongShared *>(smem);
    Chunk<T> ch(p, x);
    const uint32_t state = uniform(ch.ws->state);
    State st;
    uint32_t down;
    if (state == kRowDone || !ch.open_kept(p, 1, st, down)) return;
    Cut cut{uniform(ch.ws->cut.least), uniform(ch.ws->cut.tie_last)};
    if (state != kRowCut) {
        int64_t slot;
        float prob;
        take_list(ch, sh, st);
        search(ch.row, sh, ch.lim, st, true, false, slot, prob);
        cut = st.cut;
    }
    if (ch.both()) {
        // top-p's first histogram, of what top-k leaves
        const State after = second_state(ch, cut);
        fill(ch.row, sh, false, ch.from, ch.to, cut, after.s, Pass{kFirst, true, false});
        add_bins(ch, sh, 2, true);
    } else {
        if (ch.lim.min_key > cut.least) cut = Cut{ch.lim.min_key, ~0u};
        put_masses(x, ch, cut);
    }
    if (threadIdx.x == 0) x.chunk_cut[size_t(ch.r) * x.chunks + ch.c] = cut;
}
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_draw(SampleArgs p, SplitArgs x) {
    extern __shared__ uint8_t smem[];
    LongShared &sh = *reinterpret_cast<LongShared *>(smem);
    Chunk<T> ch(p, x);
    if (uniform(ch.ws->state) == kRowDone || !ch.open(p, x, sh, false)) return;
    Cut cut = x.chunk_cut[size_t(ch.r) * x.chunks];
    cut = Cut{uniform(cut.least), uniform(cut.tie_last)};
    if (!ch.both()) return draw_by_parts(p, x, ch, sh, cut);
    State st = second_state(ch, cut);
    uint32_t down;
    const uint32_t bin = pick(sh, st, ch.lim, ch.ws->count[2][threadIdx.x], ch.ws->mass[2][threadIdx.x], last_bin(ch.row, sh, st, ch.lim), down);
    to_bin(ch.row, sh, st, bin);
    list_bin(ch.row, sh, st, ch.lim, down);
    int64_t slot;
    float prob;
    search(ch.row, sh, ch.lim, st, false, false, slot, prob);
    ch.write(p, slot, prob);
}

// Rows of more slots than this go in chunks, as long as there are no more than kSplitRows of them.  Which limit holds is on the device; by mass the
// chunks gain more than they lose by number.  (In chunks and in one workgroup, the parameters' filling counted: top-p 0.9, one row of 32768 41 and 47
// us, of 65536 44 and 69, of 131072 45 and 106, 128 rows of 65536 64 and 72; top-k 50 and top-p 0.9, one row of 32768 43 and 30, of 65536 44 and 34,
// of 131072 44 and 42, 128 rows of 65536 52 and 38.)
constexpr size_t kSplitSlots = 40960, kSplitRows = 128;
constexpr size_t kChunk = 8192;
struct Split {
    uint32_t chunk, chunks;
    size_t masses, cuts, mosts, bytes;
};
static Split split_of(size_t rows, size_t n) {
    // chunks for a workgroup a compute unit: what a kernel does before it walks its chunk takes as long as 16384 slots
    const size_t most = rows < 128 ? 256 / rows : 2;
    const size_t chunk = std::max(kChunk, ((n + most - 1) / most + kChunk - 1) / kChunk * kChunk);
    Split x;
    x.chunk = uint32_t(chunk);
    x.chunks = uint32_t((n + chunk - 1) / chunk);
    x.masses = rows * sizeof(SampleSplit);
    x.cuts = x.masses + rows * x.chunks * kSampleWaves * 8;
    x.mosts = x.cuts + rows * x.chunks * 8;
    x.bytes = x.mosts + rows * x.chunks * 4;
    return x;
}
static bool splits(size_t rows, size_t n) { return n > kSplitSlots && rows != 0 && rows <= kSplitRows; }
size_t sample_workspace(size_t rows, size_t n) { return splits(rows, n) ? split_of(rows, n).bytes : 0; }

// A row for four waves: a short one, whose time goes into the steps that the workgroup waits in between (one row, top-k 50 and top-p 0.9: 100
// slots 26 -> 18 us, 4000 slots 28 -> 23, 8000 slots 30 -> 26 but 31 -> 34 with top-p alone, 16000 slots 34 -> 38).  And of more rows than compute units,
// four of which share one then, those not too long (1024 rows of 1000: 112 -> 26, of 25000: 165 -> 74, of 100000: 331 -> 257 but 400 -> 434 with
// top-p alone; 300 rows of 25000: 82 -> 56, of 100000: 147 -> 171).
static bool few_waves(size_t rows, size_t n) { return n <= 6144 || (rows > 256 && n <= 64 * rows); }
template <typename T>
static hipError_t sample(const SampleArgs &a, hipStream_t s) {
    const size_t lds = sizeof(LongShared), unlisted = sizeof(BinsShared), row_lds = sizeof(SampleShared<kSampleWaves, kRowListed>);
    const uint32_t grid_rows = a.rows < 65536u ? a.rows : 65536u;
    if (few_waves(a.rows, a.n)) return launch(k_sample<T, 4, kShortListed>, grid_rows, 256, sizeof(SampleShared<4, kShortListed>), s, a);
    if (!splits(a.rows, a.n)) {
        const auto kernel = k_sample<T, kSampleWaves, kRowListed>;
        if (const hipError_t e = allow_lds(reinterpret_cast<const void *>(kernel), row_lds); e != hipSuccess) return e;
        return launch(kernel, grid_rows, kSampleThreads, row_lds, s, a);
    }
    const Split split = split_of(a.rows, a.n);
    const SplitArgs x{reinterpret_cast<SampleSplit *>(a.ws), reinterpret_cast<uint64_t *>(a.ws + split.masses), reinterpret_cast<Cut *>(a.ws + split.cuts),
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
    return go(k_sample_draw<T>, dim3(a.rows), lds);
}
hipError_t launch_sample(const SampleArgs &a, int score_type, hipStream_t s) {
    if (score_type == kF32) return sample<float>(a, s);
    return score_type == kF16 ? sample<f16>(a, s) : sample<bf16>(a, s);
}

}  // namespace tv
