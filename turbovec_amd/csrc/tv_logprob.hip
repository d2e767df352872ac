// Log probabilities of given slots under a softmax of rows of scores, the softmax's entropy, its best slots, and the gradient of the scores.
//
// With m the largest score that counts, d = (score - m) / T, S = sum of exp(d) and U = sum of exp(d) d: log p = d - log S, and the entropy is
// log S - U / S, two terms that are not below 0.  Exponentials are of base 2, with log2(e) / T as the factor.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "tv_device.h"
#include "tv_ops.h"

namespace tv {

constexpr float kInf = __builtin_inff(), kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A row's temperature: the factors of a distance to the best score, in natural logarithms and in those of base 2.  One that is no normal number above 0 is the limit: every distance
// other than 0 is infinite, whatever a product says.  An infinite one has the smallest factor, not 0: what does not count lies at -infinity, and stays there.
struct Heat {
    float t, factor2;
    bool limit;
    __device__ __forceinline__ Heat(const float *temperature, uint32_t row) {
        t = temperature == nullptr ? 1.0f : temperature[row];
        limit = !(t >= FLT_MIN);
        factor2 = limit ? FLT_MAX : fmaxf(kLog2e / t, FLT_TRUE_MIN);
    }
    // log p of a slot at distance d <= 0, of a sum whose logarithm is log_sum.  (A distance that 32 bits do not hold is infinite at every temperature.)
    __device__ __forceinline__ float log_p(float d, float log_sum) const { return (limit ? (d < 0.0f ? -kInf : d) : d == -kInf ? d : d / t) - log_sum; }
};
// Whether a score counts: allowed, and not -infinity.  (NaN counts: it shows.)
__device__ __forceinline__ bool counts(const uint64_t *mask, uint32_t i, float s) {
    return (mask == nullptr || ((mask[i >> 6] >> (i & 63u)) & 1u)) && !(s == -kInf);
}
// What a set of scores adds up to: its largest score (kNone or less: it has none), and the sums of 2^t and 2^t t over it, t = (score - largest) * factor2 <= 0.
constexpr float kNone = -FLT_MAX;
struct Sums {
    float m = kNone, s = 0.0f, u = 0.0f;
    // The same, seen from a largest score that is not below its own.  (2^-10000 is 0 here; an infinity times 0 is not.)
    __device__ __forceinline__ void rise(float to, float factor2) {
        const float d = fmaxf((m - to) * factor2, -10000.0f), f = __builtin_amdgcn_exp2f(d);
        u = f * fmaf(s, d, u);
        s *= f;
        m = to;
    }
    // At the limit nothing of it is left then where its own is below.  (A NaN stays.)
    __device__ __forceinline__ void outdo(float to) {
        s = m < to ? s * 0.0f : s;
        u = m < to ? u * 0.0f : u;
    }
    __device__ __forceinline__ void add(float score, float factor2) {
        const float t = (score - m) * factor2, e = __builtin_amdgcn_exp2f(t);
        s += e;
        u = fmaf(e, fmaxf(t, -200.0f), u);
    }
    __device__ __forceinline__ void join(const Sums &other) {
        s += other.s;
        u += other.u;
    }
    __device__ __forceinline__ float entropy(float log_sum) const { return s == 0.0f ? 0.0f : log_sum - kLn2 * (u / s); }
};

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t smaller(uint64_t a, uint64_t b) { return a < b ? a : b; }

// Workgroups of kLogThreads; of kWideThreads where a row has one to itself and would need several of the others, of kShortThreads for many short rows.
constexpr int kLogThreads = 256, kLogWaves = kLogThreads / 64, kWideThreads = 1024, kShortThreads = 64;
// Sums over the workgroup, in every thread; `best` has room for a float a thread and is left holding the threads' largest scores.
template <int THREADS>
struct Reduce {
    __attribute__((aligned(16))) float best[THREADS];
    float part[2][THREADS / 64];
};
template <int THREADS>
__device__ __forceinline__ Sums group_sums(Sums v, const Heat &heat, Reduce<THREADS> &r) {
    constexpr int kWaves = THREADS / 64;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    r.best[threadIdx.x] = v.m;
    __syncthreads();
    float m = r.best[lane];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) m = fmaxf(m, r.best[i * 64 + lane]);
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor(m, i));
    if (heat.limit) v.outdo(m);
    v.rise(m, heat.factor2);
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) {
        v.s += __shfl_xor(v.s, i);
        v.u += __shfl_xor(v.u, i);
    }
    if (lane == 0) {
        r.part[0][wave] = v.s;
        r.part[1][wave] = v.u;
    }
    __syncthreads();
    v.s = v.u = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        v.s += r.part[0][i];
        v.u += r.part[1][i];
    }
    return v;
}

// The best keys of those that a workgroup has met: gathered in LDS, cut to the k best whenever the next 8 of each thread (of kMostMeet at most) might not fit.
constexpr uint32_t kKeep = 256, kInOrder = 512;
constexpr int kMostMeet = 512;
template <int THREADS>
struct Gathered {
    static constexpr uint32_t kMeet = THREADS < kMostMeet ? THREADS : kMostMeet, kGather = kKeep + 8 * kMeet;
    uint64_t keys[kGather];
    uint32_t count, part[2][THREADS / 64];
};
// Of the `count` keys, kKeep < count <= kGather: the k-th largest, bit by bit from the highest on; it and those above stay.
template <int THREADS>
__device__ __forceinline__ uint64_t cut(Gathered<THREADS> &g, uint32_t k) {
    constexpr int kEach = int(Gathered<THREADS>::kGather + THREADS - 1) / THREADS;
    const uint32_t count = g.count, wave = threadIdx.x >> 6;
    uint64_t mine[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine[i] = uint32_t(i * THREADS) + threadIdx.x < count ? g.keys[i * THREADS + threadIdx.x] : 0ull;
    uint64_t found = 0;
#pragma unroll 1
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t trial = found | 1ull << bit;
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) n += uint32_t(__popcll(__ballot(mine[i] >= trial)));
        uint32_t *const part = g.part[bit & 1];
        if ((threadIdx.x & 63u) == 0) part[wave] = n;
        __syncthreads();
        uint32_t all = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) all += part[w];
        if (all >= k) found = trial;
    }
    if (threadIdx.x == 0) g.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        if (mine[i] >= found) g.keys[atomicAdd(&g.count, 1u)] = mine[i];
    __syncthreads();
    return found;
}
// The k best in order to `out`, zeros where there are fewer.  (A thread finds its keys' places by counting.)
template <int THREADS, typename F>
__device__ __forceinline__ void in_order(Gathered<THREADS> &g, uint32_t k, F &&out) {
    uint32_t count = g.count;
    if (count > kInOrder) {
        cut(g, k);
        count = g.count;
    }
    for (uint32_t first = threadIdx.x; first < count; first += 2 * THREADS) {
        const uint64_t mine = g.keys[first], other = first + THREADS < count ? g.keys[first + THREADS] : 0ull;
        uint32_t place = 0, other_place = 0;
#pragma unroll 4
        for (uint32_t i = 0; i < count; ++i) {
            const uint64_t x = g.keys[i];
            place += x > mine;
            other_place += x > other;
        }
        if (place < k) out(place, mine);
        if (other != 0 && other_place < k) out(other_place, other);
    }
    for (uint32_t i = threadIdx.x; i < k; i += THREADS)
        if (i >= count) out(i, 0ull);
}

// A thread's given slots and their scores: asked for before the sums are known.
template <int THREADS>
struct Given {
    static constexpr int kEach = (int(kMostGiven) + THREADS - 1) / THREADS;
    float score[kEach];
    bool there[kEach];
    template <typename T>
    __device__ __forceinline__ void load(const LogProbArgs &a, uint32_t row, const T *scores, const uint64_t *mask) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t k = uint32_t(i * THREADS) + threadIdx.x;
            there[i] = false;
            if (k >= a.given) continue;
            const int64_t slot = a.slots[size_t(row) * a.slot_stride + k];
            if (slot < 0 || slot >= int64_t(a.n)) continue;
            score[i] = float(scores[slot]);
            there[i] = counts(mask, uint32_t(slot), score[i]);
        }
    }
};
// A row's results from its sums and best keys.
template <int THREADS>
__device__ __forceinline__ void finish(const LogProbArgs &a, uint32_t row, const Given<THREADS> &given, const Heat &heat, const Sums &sums, Gathered<THREADS> &g) {
    const float log_sum = logf(sums.s);
    if (threadIdx.x == 0) {
        const float entropy = sums.entropy(log_sum);
        a.out_entropy[row] = entropy;
        if (a.stats != nullptr) *reinterpret_cast<float4 *>(a.stats + size_t(row) * 4) = make_float4(sums.m, log2f(sums.s), entropy, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < given.kEach; ++i)
        if (const uint32_t k = uint32_t(i * THREADS) + threadIdx.x; k < a.given)
            a.out_log_probs[size_t(row) * a.given + k] = given.there[i] ? heat.log_p(given.score[i] - sums.m, log_sum) : -kInf;
    if (a.top != 0)
        in_order(g, a.top, [&](uint32_t place, uint64_t key) {
            float v = 0.0f;
            uint32_t slot = 0;
            sort_unkey(key, v, slot);
            a.out_top_slots[size_t(row) * a.top + place] = key == 0 ? -1 : int64_t(slot);
            a.out_top_log_probs[size_t(row) * a.top + place] = key == 0 ? -kInf : heat.log_p(v - sums.m, log_sum);
        });
}

// Scores i .. i + kEach - 1 as floats, i a multiple of kEach; what is masked and what lies behind the end is -infinity.
template <typename T>
struct Scores {
    static constexpr int kEach = 16 / int(sizeof(T));
    T v[kEach];
    uint32_t bits;
    __device__ __forceinline__ void load(const T *scores, const uint64_t *mask, uint32_t i) {
        __builtin_memcpy(v, scores + i, 16);
        bits = mask == nullptr ? ~0u : uint32_t(mask[i >> 6] >> (i & 63u));
    }
    __device__ __forceinline__ void load_end(const T *scores, const uint64_t *mask, uint32_t i, uint32_t n) {
        bits = mask == nullptr ? ~0u : uint32_t(mask[i >> 6] >> (i & 63u));
#pragma unroll
        for (int j = 0; j < kEach; ++j) v[j] = i + j < n ? scores[i + j] : T(-kInf);
    }
    template <bool MASK>
    __device__ __forceinline__ float at(int j) const {
        // (bfloat16 by its bits: the compiler takes largest ones in the narrow type, five instructions each)
        float x;
        if constexpr (sizeof(T) == 2 && !std::is_same_v<T, f16>) x = __uint_as_float(uint32_t(__builtin_bit_cast(uint16_t, v[j])) << 16);
        else x = float(v[j]);
        return !MASK || ((bits >> j) & 1u) ? x : -kInf;
    }
};

// The largest of three; a quiet NaN is passed over, a signalling one is not.  (Written as two maxima the compiler makes each operand canonical first.)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// A part of a row to a workgroup, all of it where there are rows enough.  One pass takes the sums, a thread each its own from its own largest score, which it raises once for
// four loads.  The alternatives come from the threads' largest scores: the k-th of those is one that k scores reach, and so is what its first bits say; only where a thread
// reaches that itself, a thread's part in four for itself, is the row read again.  Bound by the vector ALU: an exponential and nine to ten instructions a score, 69 us of the 79 that 2048 rows of 100000
// bfloat16 take; of floats 163, 5.0 TB/s.
struct LogPart {
    float m, s, u, none;
};
constexpr int kLogLoads = 4, kLogSegments = 4;
// Where thread t's scores lie: load l is at lo + (l * THREADS + t) * kEach, the first `segment` loads are its first segment.
struct Loads {
    uint32_t lo, hi, all, segment;
    __device__ __forceinline__ Loads(uint32_t from, uint32_t to, uint32_t step) : lo(from), hi(to) {
        all = (to - from + step - 1) / step;
        constexpr uint32_t kRounds = kLogSegments * kLogLoads;
        segment = all < 2 * kRounds ? all : (all + kRounds - 1) / kRounds * kLogLoads;
    }
};
template <int THREADS, int LOADS, typename T, bool MASK>
__device__ __forceinline__ void scan_part(const T *scores, const uint64_t *mask, const Heat &heat, const Loads &at, Sums &sums, float (&segments)[kLogSegments]) {
    constexpr int kEach = Scores<T>::kEach;
    constexpr uint32_t kStep = THREADS * kEach;
    float segment = kNone;
    auto take = [&](const Scores<T> *l, auto count) {
        constexpr int kCount = decltype(count)::value * kEach;
        float x[kCount];
#pragma unroll
        for (int i = 0; i < kCount; ++i) x[i] = l[i / kEach].template at<MASK>(i % kEach);
#pragma unroll
        for (int i = 0; i < kCount; i += 2) segment = max3(segment, x[i], x[i + 1]);
        const float largest = fmaxf(sums.m, segment);
        if (heat.limit) {
            sums.outdo(largest);
#pragma unroll
            for (int i = 0; i < kCount; ++i) x[i] = x[i] < largest ? -kInf : x[i];
        }
        sums.rise(largest, heat.factor2);
        Sums some;                      // (what is loaded at once is added for itself: the long sum loses a rounding for each of those, not for each score)
        some.m = sums.m;
#pragma unroll
        for (int i = 0; i < kCount; ++i) some.add(x[i], heat.factor2);
        sums.join(some);
    };
#pragma unroll
    for (int part = 0; part < kLogSegments; ++part) {
        const uint32_t first = at.lo + uint32_t(part) * at.segment * kStep, end = part + 1 == kLogSegments ? at.hi : min(at.lo + uint32_t(part + 1) * at.segment * kStep, at.hi);
        segment = kNone;
        if (uint32_t(part) * at.segment < at.all) {
            uint32_t i = first + threadIdx.x * kEach;
            for (; i + (LOADS - 1) * kStep + kEach <= end; i += LOADS * kStep) {
                Scores<T> l[LOADS];
#pragma unroll
                for (int j = 0; j < LOADS; ++j) l[j].load(scores, mask, i + j * kStep);
                take(l, IntC<LOADS>{});
            }
            for (; i < end; i += kStep) {
                Scores<T> l;
                if (i + kEach <= end) l.load(scores, mask, i);
                else l.load_end(scores, mask, i, end);
                take(&l, IntC<1>{});
            }
        }
        segments[part] = segment;
    }
    // A signalling NaN takes the largest score before it along, so what it stands in is read again, all of it.
    if (sums.s != sums.s) {
#pragma unroll
        for (int part = 0; part < kLogSegments; ++part) segments[part] = kInf;
    }
}
constexpr uint32_t kFewAlternatives = 24;
// One that at least k of a score a thread in `best` reach, and not far below the k-th: its first 16 bits in the scores' order.  The same in every thread.
template <int THREADS>
__device__ __forceinline__ float reached(const float *best, uint32_t k) {
    constexpr int kEach = THREADS / 64;
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t key[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) key[i] = uint32_t(order_key(best[i * 64 + lane] + 0.0f)) ^ 0x80000000u;
    uint32_t found = 0;
    if (k <= kFewAlternatives) {          // (the largest of every sixty-fourth thread: 64 of those do)
        uint32_t one = key[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) one = max(one, key[i]);
#pragma unroll
        for (int bit = 31; bit >= 16; --bit)
            if (uint32_t(__popcll(__ballot(one >= (found | 1u << bit)))) >= k) found |= 1u << bit;
    } else {
#pragma unroll
        for (int bit = 31; bit >= 16; --bit) {
            uint32_t n = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) n += uint32_t(__popcll(__ballot(key[i] >= (found | 1u << bit))));
            if (n >= k) found |= 1u << bit;
        }
    }
    return fmaxf(order_unkey(int(found ^ 0x80000000u)), kNone);      // (nothing counts below that; a key of 0 is no number)
}
template <int THREADS, typename T, bool MASK>
__device__ __forceinline__ void gather_part(const LogProbArgs &a, const T *scores, const uint64_t *mask, const Loads &at, const float (&segments)[kLogSegments], Gathered<THREADS> &g, const float *best,
                                            uint16_t *who, uint32_t *who_count) {
    constexpr int kEach = Scores<T>::kEach;
    constexpr uint32_t kStep = THREADS * kEach;
    const float least = reached<THREADS>(best, a.top);
    if (threadIdx.x == 0) g.count = *who_count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kLogSegments; ++i)
        if (segments[i] >= least && uint32_t(i) * at.segment < at.all) who[atomicAdd(who_count, 1u)] = uint16_t(i * THREADS + threadIdx.x);
    __syncthreads();
    const uint32_t items = *who_count * at.segment;
    auto place = [&](uint32_t item) {      // hi where there is nothing
        if (item >= items) return at.hi;
        const uint32_t it = who[item / at.segment], l = it / THREADS * at.segment + item % at.segment;
        const uint64_t i = at.lo + uint64_t(l) * kStep + it % THREADS * kEach;
        return l < at.all && i < at.hi ? uint32_t(i) : at.hi;
    };
    auto load = [&](Scores<T> &l, uint32_t i) {
        if (i >= at.hi) return;
        if (i + kEach <= at.hi) l.load(scores, mask, i);
        else l.load_end(scores, mask, i, at.hi);
    };
    auto put = [&](const Scores<T> &l, uint32_t i, uint64_t above) {
        if (i >= at.hi) return;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const float v = l.template at<MASK>(j);
            if (!(v >= least)) continue;
            const uint64_t key = sort_key(v, i + j);
            if (key <= above) continue;
            const uint32_t to = atomicAdd(&g.count, 1u);
            if (to < Gathered<THREADS>::kGather) g.keys[to] = key;
        }
    };
    // As a rule all that is met fits.
    for (uint32_t first = threadIdx.x; first < items; first += 2 * THREADS) {
        Scores<T> l[2];
        const uint32_t i[2] = {place(first), place(first + THREADS)};
#pragma unroll
        for (int j = 0; j < 2; ++j) load(l[j], i[j]);
#pragma unroll
        for (int j = 0; j < 2; ++j) put(l[j], i[j], 0);
    }
    __syncthreads();
    if (g.count <= Gathered<THREADS>::kGather) return;
    // Crowded scores: once more, cut to the best whenever the next loads might not fit.
    __syncthreads();
    if (threadIdx.x == 0) g.count = 0;
    __syncthreads();
    uint64_t above = 0;
    for (uint32_t first = 0; first < items; first += Gathered<THREADS>::kMeet) {
        Scores<T> l;
        const uint32_t i = threadIdx.x < Gathered<THREADS>::kMeet ? place(first + threadIdx.x) : at.hi;
        load(l, i);
        put(l, i, above);
        __syncthreads();
        const uint32_t count = g.count;
        __syncthreads();
        if (count > kKeep) above = cut(g, a.top);
    }
}
// (LOADS at once: two where a compute unit is to hold two of the wide workgroups, 64 registers a thread, nine more spilled.)
template <int THREADS, int LOADS, typename T, bool MASK>
__global__ __launch_bounds__(THREADS, THREADS == kWideThreads && LOADS < kLogLoads ? 8 : 1) void k_log_probs(LogProbArgs a, uint32_t parts, uint32_t part_size) {
    __shared__ Reduce<THREADS> reduce;
    __shared__ Gathered<THREADS> g;
    __shared__ uint16_t who[kLogSegments * THREADS];
    __shared__ uint32_t who_count;
    LogPart *const out = reinterpret_cast<LogPart *>(a.ws);
    uint64_t *const out_keys = reinterpret_cast<uint64_t *>(a.ws + size_t(a.rows) * parts * sizeof(LogPart));
    auto one = [&](uint64_t unit) {
        const uint32_t row = uint32_t(unit / parts), lo = uint32_t(unit % parts) * part_size;
        const Loads at(lo, min(part_size, a.n - lo) + lo, THREADS * Scores<T>::kEach);
        const T *const scores = static_cast<const T *>(a.scores) + size_t(row) * a.stride;
        const uint64_t *const mask = MASK ? a.mask + size_t(row) * a.mask_stride : nullptr;
        const Heat heat(a.temperature, row);
        Given<THREADS> given;
        if (parts == 1) given.load(a, row, scores, mask);
        Sums sums;
        float segments[kLogSegments];
        scan_part<THREADS, LOADS, T, MASK>(scores, mask, heat, at, sums, segments);
        sums = group_sums(sums, heat, reduce);
        if (a.top != 0) gather_part<THREADS, T, MASK>(a, scores, mask, at, segments, g, reduce.best, who, &who_count);
        if (parts == 1) {
            finish(a, row, given, heat, sums, g);
        } else {
            if (threadIdx.x == 0) out[unit] = LogPart{sums.m, sums.s, sums.u, 0.0f};
            if (a.top != 0) in_order(g, a.top, [&](uint32_t place, uint64_t key) { out_keys[unit * a.top + place] = key; });
        }
    };
    if constexpr (THREADS == kWideThreads) {
        one(blockIdx.x);
    } else {
        for (uint64_t unit = blockIdx.x; unit < uint64_t(a.rows) * parts; unit += gridDim.x) {
            one(unit);
            __syncthreads();
        }
    }
}
// The parts of a row, joined.  Keys that cannot be among the best are told from a few of each part: its last one is one that k keys reach, and so is the lowest of all parts'
// j-th where j keys of each are k, and the k-th of all parts' first.  Only parts whose first passes are read.
constexpr uint32_t kMostParts = 1024;
template <typename T>
__global__ __launch_bounds__(kLogThreads) void k_log_probs_join(LogProbArgs a, uint32_t parts) {
    __shared__ Reduce<kLogThreads> reduce;
    __shared__ Gathered<kLogThreads> g;
    __shared__ uint64_t least[2][kLogWaves];
    __shared__ uint16_t who[kMostParts];
    __shared__ uint32_t who_count;
    constexpr int kEach = kMostParts / kLogThreads;
    const uint32_t top = a.top, share = top == 0 ? 0 : (top + parts - 1) / parts;
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *const scores = static_cast<const T *>(a.scores) + size_t(row) * a.stride;
        const uint64_t *const mask = a.mask == nullptr ? nullptr : a.mask + size_t(row) * a.mask_stride;
        const LogPart *const in = reinterpret_cast<const LogPart *>(a.ws) + size_t(row) * parts;
        const uint64_t *const in_keys = reinterpret_cast<const uint64_t *>(a.ws + size_t(a.rows) * parts * sizeof(LogPart)) + size_t(row) * parts * top;
        const Heat heat(a.temperature, row);
        Given<kLogThreads> given;
        given.load(a, row, scores, mask);
        LogPart p[kEach];
        uint64_t first[kEach], last = 0, low = ~0ull;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t part = uint32_t(i * kLogThreads) + threadIdx.x;
            first[i] = 0;
            p[i] = LogPart{kNone, 0.0f, 0.0f, 0.0f};
            if (part >= parts) continue;
            p[i] = in[part];
            if (top == 0) continue;
            const uint64_t *const keys = in_keys + size_t(part) * top;
            first[i] = keys[0];
            last = larger(last, keys[top - 1]);
            low = smaller(low, keys[share - 1]);
        }
        Sums sums;
        float best = kNone;
#pragma unroll
        for (int i = 0; i < kEach; ++i) sums.m = fmaxf(sums.m, p[i].m);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            Sums more;
            more.m = p[i].m; more.s = p[i].s; more.u = p[i].u;
            if (heat.limit) more.outdo(sums.m);
            more.rise(sums.m, heat.factor2);
            sums.s += more.s;
            sums.u += more.u;
            best = fmaxf(best, first[i] == 0 ? kNone : order_unkey(int(uint32_t(first[i] >> 32) ^ 0x80000000u)));
        }
        if (top != 0) {
#pragma unroll
            for (int i = 32; i > 0; i >>= 1) {
                last = larger(last, uint64_t(__shfl_xor((unsigned long long)(last), i)));
                low = smaller(low, uint64_t(__shfl_xor((unsigned long long)(low), i)));
            }
            if ((threadIdx.x & 63) == 0) {
                least[0][threadIdx.x >> 6] = last;
                least[1][threadIdx.x >> 6] = low;
            }
            if (threadIdx.x == 0) g.count = who_count = 0;
        }
        sums = group_sums(sums, heat, reduce);
        if (top != 0) {
            uint64_t from = larger(larger(larger(least[0][0], least[0][1]), larger(least[0][2], least[0][3])), smaller(smaller(least[1][0], least[1][1]), smaller(least[1][2], least[1][3])));
            __syncthreads();
            reduce.best[threadIdx.x] = best;
            __syncthreads();
            const float reach = reached<kLogThreads>(reduce.best, top);
            from = larger(from, reach > kNone ? sort_key(reach, 0x7fffffffu) & ~1ull : 0ull);      // (the lowest key of that score)
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (first[i] != 0 && first[i] >= from) who[atomicAdd(&who_count, 1u)] = uint16_t(i * kLogThreads + threadIdx.x);
            __syncthreads();
            const uint32_t keys = who_count * top;
            for (uint32_t at = 0; at < keys; at += kLogThreads) {
                const uint32_t item = at + threadIdx.x;
                const uint64_t key = item < keys ? in_keys[size_t(who[item / top]) * top + item % top] : 0ull;
                if (key != 0 && key >= from) g.keys[atomicAdd(&g.count, 1u)] = key;
                __syncthreads();
                const uint32_t count = g.count;
                __syncthreads();
                if (count > Gathered<kLogThreads>::kGather - kLogThreads) from = cut(g, top);
            }
        }
        finish(a, row, given, heat, sums, g);
        __syncthreads();
    }
}
// Rows in parts where there are too few of them for the card: parts of a multiple of what a workgroup loads at once.
static uint32_t log_parts(size_t rows, size_t n, uint32_t &part_size) {
    constexpr size_t kOnce = 8192, kMost = kMostParts;      // scores; workgroups: four to a compute unit
    const size_t at_once = (n + kOnce - 1) / kOnce, wanted = rows >= kMost ? 1 : kMost / rows;
    const size_t each = (at_once + std::min(wanted, at_once) - 1) / std::min(wanted, at_once);
    part_size = uint32_t(std::min(each * kOnce, n));
    return uint32_t((n + part_size - 1) / part_size);
}
// Rows in parts that have a wide workgroup each all the same: rows enough for half of the card, and those that are not much longer than what a second launch takes, and the parts'
// ranking of their best where alternatives are asked for.  A second launch costs a call among others 3.7 us on the host, one that is waited for and one in a graph less: the border lies between what these
// two have.  (us so and in parts, bfloat16, in a graph / waited for.  1 row without alternatives: 64000 scores 8.2 and 7.3 / 26.9 and 28.6, 80000 9.2 and 8.3 / 27.8 and 28.6, 100000 9.9 and 7.1 / 28.6 and
// 28.4; with 1 100000 12.3 and 10.9 / 31.2 and 32.4, 128256 14.8 and 11.0 / 33.8 and 32.4; with 20 100000 13.6 and 14.7 / 32.7 and 35.9, 128256 16.5 and 14.5 / 35.3 and 35.7; with 128 151936 28 and 31 / 48 and
// 50.  64 rows: without 100000 10.8 and 11.1 / 30.1 and 31.4, 128256 13.8 and 11.1 / 32.9 and 31.6; with 20 128256 18.0 and 19.7 / 37 and 40; with 128 151936 30 and 47 / 50 and 68.  128 rows without:
// 151936 15.5 and 15.6 / 34.7 and 36.1, 200000 18.0 and 17.7 / 37 and 38; 192 rows without: 200000 20.9 and 22.0, 500000 44 and 49.  Scores of which thousands tie with the best are gathered in turns, of
// which parts have fewer each: 64 equal rows of 128256 with 20 227 and 111.  That is why many alternatives do not raise the border to where random scores have theirs, 300000 and more with 128.)
static bool log_wide(size_t rows, size_t n, size_t top) { return rows >= 160 || n <= 80000 + (top != 0 ? 20000 : 0) + 500 * top + 600 * rows; }
// Many rows of a few loads have a wave each, as long as its 64 largest scores tell the alternatives apart.  (Rows of 1000 bfloat16 scores with 5 alternatives: 1024 rows 7.9 us so and 8.5
// with workgroups of 256, 4096 rows 10.2 and 21.9, 65536 rows 88 and 275; their gradients 4096 rows 8.2 and 11.4, 65536 rows 73 and 152.)
static bool log_short(size_t rows, size_t n, size_t size, size_t top) { return rows >= 1024 && n * size <= 8192 && top <= kFewAlternatives; }
size_t log_probs_workspace(size_t rows, size_t n, size_t top) {
    if (rows == 0 || n == 0) return 0;
    uint32_t part_size;
    const size_t parts = log_parts(rows, n, part_size);
    return parts == 1 || log_wide(rows, n, top) ? 0 : rows * parts * (sizeof(LogPart) + top * sizeof(uint64_t));
}
template <typename T, bool MASK>
static hipError_t log_probs(const LogProbArgs &a, hipStream_t s) {
    uint32_t part_size;
    const uint32_t parts = log_parts(a.rows, a.n, part_size);
    if (parts > 1 && log_wide(a.rows, a.n, a.top)) {
        const auto kernel = a.rows <= 256 ? k_log_probs<kWideThreads, kLogLoads, T, MASK> : k_log_probs<kWideThreads, kLogLoads / 2, T, MASK>;
        return launch(kernel, a.rows, kWideThreads, 0, s, a, 1u, a.n);
    }
    const uint64_t units = uint64_t(a.rows) * parts;
    if (log_short(a.rows, a.n, sizeof(T), a.top))
        return launch(k_log_probs<kShortThreads, kLogLoads / 2, T, MASK>, uint32_t(units < kMostGroups ? units : kMostGroups), kShortThreads, 0, s, a, 1u, a.n);
    const hipError_t e = launch(k_log_probs<kLogThreads, kLogLoads, T, MASK>, uint32_t(units < kMostGroups ? units : kMostGroups), kLogThreads, 0, s, a, parts, part_size);
    return e != hipSuccess || parts == 1 ? e : launch(k_log_probs_join<T>, uint32_t(a.rows < kMostGroups ? a.rows : kMostGroups), kLogThreads, 0, s, a, parts);
}
template <typename T>
static hipError_t log_probs_as(const LogProbArgs &a, hipStream_t s) {
    return a.mask == nullptr ? log_probs<T, false>(a, s) : log_probs<T, true>(a, s);
}
hipError_t launch_log_probs(const LogProbArgs &a, int score_type, hipStream_t s) {
    if (score_type == kF32) return log_probs_as<float>(a, s);
    return score_type == kF16 ? log_probs_as<f16>(a, s) : log_probs_as<bf16>(a, s);
}

// The gradient of a score that counts: (picked - p (G + g (log p + H))) / T, picked the sum of the gradients of the given slots that are this one.  With l = log2 p that is
// (picked + p (A + B l)) / T, A = -(G + g H) and B = -g ln 2.  Bound by memory, a reading and a writing: 2048 rows of 100000 bfloat16 166 us, 4.9 TB/s, what a copy reaches.  What is picked is added by the thread that wrote the
// slot's own gradient, behind that.
template <int THREADS, typename T, bool MASK>
__global__ __launch_bounds__(THREADS) void k_log_probs_grad(LogProbGradArgs a, uint32_t parts, uint32_t part_size) {
    constexpr int kEach = Scores<T>::kEach;
    constexpr uint32_t kStep = THREADS * kEach;
    typedef T Run __attribute__((ext_vector_type(kEach), aligned(sizeof(T))));
    for (uint64_t unit = blockIdx.x; unit < uint64_t(a.rows) * parts; unit += gridDim.x) {
        const uint32_t row = uint32_t(unit / parts), lo = uint32_t(unit % parts) * part_size, hi = lo + min(part_size, a.n - lo);
        const T *const scores = static_cast<const T *>(a.scores) + size_t(row) * a.stride;
        const uint64_t *const mask = MASK ? a.mask + size_t(row) * a.mask_stride : nullptr;
        T *const grad = static_cast<T *>(a.grad) + size_t(row) * a.grad_stride;
        const Heat heat(a.temperature, row);
        const float4 stats = *reinterpret_cast<const float4 *>(a.stats + size_t(row) * 4);      // largest, log2 of the sum, entropy
        const float *const g = a.grad_log_probs + size_t(row) * a.given;
        const int64_t *const slots = a.slots + size_t(row) * a.slot_stride;
        float all = 0.0f;                // (a lane to a given slot, every wave the same)
        for (uint32_t k = threadIdx.x & 63u; k < a.given; k += 64u) {
            const int64_t slot = slots[k];
            if (slot >= 0 && slot < int64_t(a.n) && counts(mask, uint32_t(slot), float(scores[slot]))) all += g[k];
        }
#pragma unroll
        for (int k = 32; k > 0; k >>= 1) all += __shfl_xor(all, k);
        const float g_entropy = a.grad_entropy == nullptr ? 0.0f : a.grad_entropy[row];
        const float factor_a = -(all + g_entropy * stats.z), factor_b = -g_entropy * kLn2, inverse = heat.limit ? 0.0f : 1.0f / heat.t;
        auto at = [&](float s) {
            const float l = fmaf(s - stats.x, heat.factor2, -stats.y), d = __builtin_amdgcn_exp2f(l) * fmaf(factor_b, fmaxf(l, -200.0f), factor_a);
            return s == -kInf ? 0.0f : d;
        };
        auto whole = [&](const Scores<T> &l, uint32_t i) {
            Run r;
#pragma unroll
            for (int j = 0; j < kEach; ++j) r[j] = T(at(l.template at<MASK>(j)) * inverse);
            __builtin_nontemporal_store(r, reinterpret_cast<Run *>(grad + i));
        };
        uint32_t i = lo + threadIdx.x * kEach;
        for (; i + (kLogLoads - 1) * kStep + kEach <= hi; i += kLogLoads * kStep) {
            Scores<T> l[kLogLoads];
#pragma unroll
            for (int j = 0; j < kLogLoads; ++j) l[j].load(scores, mask, i + j * kStep);
#pragma unroll
            for (int j = 0; j < kLogLoads; ++j) whole(l[j], i + j * kStep);
        }
        for (; i < hi; i += kStep) {
            Scores<T> l;
            if (i + kEach <= hi) {
                l.load(scores, mask, i);
                whole(l, i);
            } else {
                l.load_end(scores, mask, i, hi);
#pragma unroll
                for (int j = 0; j < kEach; ++j)
                    if (i + j < hi) grad[i + j] = T(at(l.template at<MASK>(j)) * inverse);
            }
        }
        for (uint32_t k = 0; k < (heat.limit ? 0u : a.given); ++k) {
            const int64_t slot = slots[k];
            if (slot < int64_t(lo) || slot >= int64_t(hi) || (uint32_t(slot) - lo) / kEach % THREADS != threadIdx.x) continue;
            const float s = float(scores[slot]);
            if (!counts(mask, uint32_t(slot), s)) continue;
            float picked = 0.0f;               // (where the same slot stands there again, the last sum is the whole one)
            for (uint32_t l = 0; l <= k; ++l) picked += slots[l] == slot ? g[l] : 0.0f;
            grad[slot] = T((at(s) + picked) * inverse);
        }
    }
}
template <int THREADS, typename T>
static hipError_t log_probs_grad(const LogProbGradArgs &a, hipStream_t s) {
    uint32_t part_size;
    const uint32_t parts = log_parts(a.rows, a.n, part_size);
    const uint64_t units = uint64_t(a.rows) * parts;
    const uint32_t grid = uint32_t(units < kMostGroups ? units : kMostGroups);
    const auto kernel = a.mask == nullptr ? k_log_probs_grad<THREADS, T, false> : k_log_probs_grad<THREADS, T, true>;
    return launch(kernel, grid, THREADS, 0, s, a, parts, part_size);
}
template <typename T>
static hipError_t log_probs_grad_as(const LogProbGradArgs &a, hipStream_t s) {
    return log_short(a.rows, a.n, sizeof(T), 0) ? log_probs_grad<kShortThreads, T>(a, s) : log_probs_grad<kLogThreads, T>(a, s);
}
hipError_t launch_log_probs_grad(const LogProbGradArgs &a, int score_type, hipStream_t s) {
    if (score_type == kF32) return log_probs_grad_as<float>(a, s);
    return score_type == kF16 ? log_probs_grad_as<f16>(a, s) : log_probs_grad_as<bf16>(a, s);
}

}  // namespace tv
