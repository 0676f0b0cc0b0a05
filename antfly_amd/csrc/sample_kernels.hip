// A token of every row of logits from the row's random number.
//
//   w_i = exp((l_i - M) / T) = 2^y_i,   tokens in the order of falling logit (equal ones by rising index):
//   kept: rank < k;  weights before < p * (sum of the first k);  w >= m;   token: the first whose weights up to it exceed u * (sum of the kept)
//
// Each filter keeps a prefix of one order, so what they keep together is the shortest of the three, and the drawn token is found as
// a prefix's end is: everything is "the first token at which the count, or the sum, passes a target".  Nothing is sorted but the few
// tokens around such a place.
// Weights are formed in 64 bits (f64 multiply-adds run at the rate of f32 ones) and summed as whole multiples of 2^-bits: sums are
// exact, whatever their order, and hang on no atomics' order.
//
// A row is shared out over workgroups, and a call is three launches:
//   most     every part's largest logit, and the largest of every few threads' tokens
//   spread   with the row's largest known: where a cut is known that leaves few tokens, these into a list (the k-th largest of the
//            largest logits above is below the k-th largest of all; min-p's cut follows from the largest).  Otherwise a histogram of
//            counts and sums over the logits' range.  The last workgroup of a row draws from the list, or finds the bins that the
//            targets can fall into
//   settle   the tokens of these bins into a list, from which the row's last workgroup draws
// A list that would not hold what it has to (thousands of equal logits, mostly) leaves the row to one workgroup, which narrows the
// bins down and counts equal ones.
//
// Large calls are bound by reading the logits twice and by the 64-bit weights of those that may count (256 rows of 128000 f32 logits,
// a filter set each: 144 to 148 us, 131 MB of them are 26 at the rate of a copy); small ones by the three launches and the ways from
// workgroup to workgroup (one row of 32000 with top-k and top-p: 17 to 28 us by their values).
#include "quantized_launch.h"

#include <hip/hip_runtime.h>

#include "sample_search.h"

namespace afhip {

namespace {

constexpr int kThreads = kSampleThreads, kWaves = kThreads / 64;
constexpr uint32_t kBins = kSampleBins, kListed = 4096;
constexpr uint32_t kMostParts = 32, kGroups = kThreads / 4;  // parts of a row, and groups of threads of a part with a largest logit of their own
constexpr double kLog2e = 1.4426950408889634;
typedef unsigned long long u64;

// The order of falling logit and rising index as that of whole numbers.
__device__ __forceinline__ uint32_t key_of(float v) {  // rising with v
    const uint32_t bits = __builtin_bit_cast(uint32_t, v + 0.0f);  // (minus zero is zero)
    return bits ^ (static_cast<uint32_t>(static_cast<int>(bits) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key); }
__device__ __forceinline__ u64 rank_of(float v, uint32_t i) { return static_cast<u64>(~key_of(v)) << 32 | i; }
__device__ __forceinline__ float value_at(u64 rank) { return value_of(~static_cast<uint32_t>(rank >> 32)); }

// A row's weights in multiples of 2^-bits.
struct Weights {
    double largest, per_logit;  // M, and log2(e) / T
    int bits;
    float top;
    bool endless;  // the largest is infinite: the infinite ones weigh 1, others nothing
    __device__ __forceinline__ double power(float v) const {  // of two
        return (static_cast<double>(v) - largest) * per_logit;
    }
    // 2^y for y <= 0: y's fraction by the series of 2^f up to f^11 (the next term is 6e-15 at f = 1/2)
    __device__ __forceinline__ double exp2_scaled(double y, int scale) const {
        const double n = __builtin_rint(y), f = y - n;
        double r = 4.4455382718708116e-10;
        r = __builtin_fma(r, f, 7.0549116208011234e-09);
        r = __builtin_fma(r, f, 1.0178086009239700e-07);
        r = __builtin_fma(r, f, 1.3215486790144309e-06);
        r = __builtin_fma(r, f, 1.5252733804059841e-05);
        r = __builtin_fma(r, f, 1.5403530393381609e-04);
        r = __builtin_fma(r, f, 1.3333558146428443e-03);
        r = __builtin_fma(r, f, 9.6181291076284772e-03);
        r = __builtin_fma(r, f, 5.5504108664821580e-02);
        r = __builtin_fma(r, f, 2.4022650695910071e-01);
        r = __builtin_fma(r, f, 6.9314718055994531e-01);
        r = __builtin_fma(r, f, 1.0);
        return __builtin_amdgcn_ldexp(r, static_cast<int>(n) + scale);
    }
    __device__ __forceinline__ u64 of(float v) const {
        const double y = power(v);
        if (!(y > -1.0 - bits)) return endless && v == top ? 1ull << bits : 0;  // (minus infinity, and no number, among them)
        // added to 2^52 it is rounded to a whole number, which the sum's lower bits are
        return __builtin_bit_cast(u64, exp2_scaled(y, bits) + 0x1p52) & ((1ull << 52) - 1);
    }
    __device__ __forceinline__ double fraction(float v) const {
        const double y = power(v);
        return y > -1000.0 ? exp2_scaled(y, 0) : endless && v == top ? 1.0 : 0.0;
    }
};

struct __attribute__((aligned(16))) Shared {
    u64 list[kListed];
    u64 sums[kBins];
    uint32_t counts[kBins];
    u64 wave_sums[kWaves];
    uint32_t wave_counts[kWaves];
    u64 wave_ranks[kWaves];
    u64 found_sum, found_before, found_rank;
    uint32_t found_count, found_bin, listed, key_low, key_high;
};

// Sum over all threads, in all of them.
__device__ __forceinline__ u64 block_sum(u64 v, Shared& s) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) s.wave_sums[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all += s.wave_sums[w];
    __syncthreads();
    return all;
}

// Sums of counts and sums over the threads before this one, and over all.
__device__ __forceinline__ void block_before(uint32_t count, u64 sum, Shared& s, uint32_t* count_before, u64* sum_before, uint32_t* all_count, u64* all_sum) {
    const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
    uint32_t c = count;
    u64 m = sum;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t cc = __shfl_up(c, d);
        const u64 mm = __shfl_up(m, d);
        if (lane >= d) {
            c += cc;
            m += mm;
        }
    }
    if (lane == 63) {
        s.wave_counts[wave] = c;
        s.wave_sums[wave] = m;
    }
    __syncthreads();
    c -= count;
    m -= sum;
    uint32_t every_count = 0;
    u64 every_sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const uint32_t wc = s.wave_counts[w];
        const u64 wm = s.wave_sums[w];
        c += w < wave ? wc : 0;
        m += w < wave ? wm : 0;
        every_count += wc;
        every_sum += wm;
    }
    __syncthreads();
    *all_count = every_count;
    *all_sum = every_sum;
    *count_before = c;
    *sum_before = m;
}

// Tokens [begin, end) of a row (begin a multiple of eight) by f(values, first), runs of four or eight, a thread's own in rising
// order; no numbers are minus infinity, and so is what fills up the last run.
template <int kType>
constexpr int kRun = kType == 0 ? 4 : 8;
template <int kType, typename F>
__device__ __forceinline__ void each_run(const void* row, uint32_t begin, uint32_t end, F f) {
    constexpr int kPer = kRun<kType>;
    struct __attribute__((packed, aligned(kType == 0 ? 4 : 2))) Run { uint32_t words[4]; };  // (rows start at any element)
    const uint32_t runs = end / kPer;
    const auto value = [](uint32_t word, int part) {
        float v;
        if (kType == 0) v = __builtin_bit_cast(float, word);
        else if (kType == 30) v = __builtin_bit_cast(float, part == 0 ? word << 16 : word & 0xFFFF0000u);
        else v = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(word >> (16 * part))));
        return v == v ? v : -__builtin_inff();
    };
    const auto visit = [&](const Run& r, uint32_t run) {
        float values[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) values[j] = value(r.words[kType == 0 ? j : j / 2], kType == 0 ? 0 : j % 2);
        f(values, run * kPer);
    };
    const Run* from = static_cast<const Run*>(row);
    constexpr uint32_t kAhead = 4;
    uint32_t run = begin / kPer + threadIdx.x;
    for (; run + (kAhead - 1) * kThreads < runs; run += kAhead * kThreads) {
        Run held[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) held[j] = from[run + j * kThreads];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) visit(held[j], run + j * kThreads);
    }
    for (; run < runs; run += kThreads) visit(from[run], run);
    const uint32_t rest = max(runs * kPer, begin) + threadIdx.x;  // (fewer than a run: no more than one a thread)
    if (rest < end) {
        const uint32_t word = kType == 0 ? static_cast<const uint32_t*>(row)[rest] : static_cast<const uint16_t*>(row)[rest];
        float values[kPer];
        values[0] = value(word, 0);
#pragma unroll
        for (int j = 1; j < kPer; ++j) values[j] = -__builtin_inff();
        f(values, rest);
    }
}
template <int kType, typename F>
__device__ __forceinline__ void each_logit(const void* row, uint32_t begin, uint32_t end, F f) {
    each_run<kType>(row, begin, end, [&](const float (&values)[kRun<kType>], uint32_t first) {
#pragma unroll
        for (int j = 0; j < kRun<kType>; ++j) f(values[j], first + j);
    });
}

// The tokens that `wanted` says, none of them below `low` or above `high`, into the list as far as it has room; how many there are.
template <int kType, typename Wanted>
__device__ __forceinline__ uint32_t gather(const void* row, uint32_t begin, uint32_t end, Shared& s, float low, float high, Wanted wanted) {
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    each_run<kType>(row, begin, end, [&](const float (&values)[kRun<kType>], uint32_t first) {
        bool any = false;
#pragma unroll
        for (int j = 0; j < kRun<kType>; ++j) any |= values[j] >= low && values[j] <= high;
        if (!any) return;  // (as most runs)
#pragma unroll
        for (int j = 0; j < kRun<kType>; ++j) {
            if (values[j] >= low && values[j] <= high && wanted(values[j])) {
                const uint32_t at = atomicAdd(&s.listed, 1u);
                if (at < kListed) s.list[at] = rank_of(values[j], first + j);
            }
        }
    });
    __syncthreads();
    return s.listed;
}

// The list's first n entries in rising order: a bitonic sort with kOwn entries a thread, entry r * kThreads + thread in register r.
// Pairs lie in one thread, in one wavefront or, for three distances of the twelve, go through LDS.
template <uint32_t kOwn>
__device__ __forceinline__ void sort_registers(uint32_t n, uint32_t size, Shared& s) {
    const uint32_t tid = threadIdx.x;
    u64 own[kOwn];
#pragma unroll
    for (uint32_t r = 0; r < kOwn; ++r) own[r] = r * kThreads + tid < n ? s.list[r * kThreads + tid] : ~0ull;
    for (uint32_t k = 2; k <= size; k *= 2) {
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            if (j >= static_cast<uint32_t>(kThreads)) {
#pragma unroll
                for (uint32_t d = 1; d < kOwn; d *= 2) {
                    if (j != d * kThreads) continue;
#pragma unroll
                    for (uint32_t r = 0; r < kOwn; ++r) {
                        if ((r & d) != 0) continue;
                        const u64 a = own[r], b = own[r | d];
                        const bool swaps = (a > b) == (((r * kThreads + tid) & k) == 0);
                        own[r] = swaps ? b : a;
                        own[r | d] = swaps ? a : b;
                    }
                }
                continue;
            }
            u64 others[kOwn];
            if (j >= 64) {
                __syncthreads();
#pragma unroll
                for (uint32_t r = 0; r < kOwn; ++r) s.list[r * kThreads + tid] = own[r];
                __syncthreads();
#pragma unroll
                for (uint32_t r = 0; r < kOwn; ++r) others[r] = s.list[r * kThreads + (tid ^ j)];
            } else {
#pragma unroll
                for (uint32_t r = 0; r < kOwn; ++r) others[r] = __shfl_xor(own[r], static_cast<int>(j));
            }
#pragma unroll
            for (uint32_t r = 0; r < kOwn; ++r) {
                const bool smaller = ((tid & j) == 0) == (((r * kThreads + tid) & k) == 0);  // this place keeps the smaller
                own[r] = (others[r] < own[r]) == smaller ? others[r] : own[r];
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < kOwn; ++r) s.list[r * kThreads + tid] = own[r];
    __syncthreads();
}

// Up to a token a thread: its place is the number of those before it.  (88 tokens take 1.4 us and 359 4.8; sorted in pairs, 70 take 3.7
// and 160 4.7.)
__device__ __forceinline__ void rank_list(uint32_t n, Shared& s) {
    const uint32_t tid = threadIdx.x;
    const u64 own = tid < n ? s.list[tid] : ~0ull;
    if (tid == 0 && (n & 1) != 0) s.list[n] = ~0ull;
    __syncthreads();
    uint32_t place = 0;
    if ((tid & ~63u) < n) {
        typedef u64 Pair __attribute__((ext_vector_type(2)));
        const Pair* pairs = reinterpret_cast<const Pair*>(s.list);
#pragma unroll 8
        for (uint32_t i = 0; i < (n + 1) / 2; ++i) {
            const Pair two = pairs[i];
            place += two[0] < own;
            place += two[1] < own;
        }
    }
    __syncthreads();
    if (tid < n) s.list[place] = own;
    __syncthreads();
}

__device__ __forceinline__ void sort_list(uint32_t n, Shared& s) {
    __syncthreads();
    if (n <= static_cast<uint32_t>(kThreads)) {
        rank_list(n, s);
        return;
    }
    uint32_t size = 2 * kThreads;
    while (size < n) size *= 2;
    if (size == 2u * kThreads) sort_registers<2>(n, size, s);
    else if (size == 4u * kThreads) sort_registers<4>(n, size, s);
    else sort_registers<kListed / kThreads>(n, size, s);
}

// The weights of the sorted list's n tokens, a run of `each` a thread, and their sum before the thread's.
struct Listed {
    static constexpr uint32_t kMost = kListed / kThreads;
    u64 own[kMost], before, all;
    uint32_t n, each, first;
    __device__ __forceinline__ Listed(uint32_t count, const Weights& weights, Shared& s) : n(count), each((count + kThreads - 1) / kThreads), first(threadIdx.x * each) {
        u64 sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < kMost; ++j) {
            own[j] = j < each && first + j < n ? weights.of(value_at(s.list[first + j])) : 0;
            sum += own[j];
        }
        uint32_t unused, none;
        block_before(0, sum, s, &unused, &before, &none, &all);
    }
    // The first of the tokens [from, until) at which the target is passed, counts and sums before them being given: into found_rank,
    // found_sum (with it), found_before and found_count (with it).  False: none.
    __device__ __forceinline__ bool find(uint32_t from, uint32_t until, uint32_t count0, u64 sum0, const Target& target, Shared& s) const {
        if (threadIdx.x == 0) s.found_count = 0;
        u64 base = sum0, upto = before;
        if (from != 0) {
#pragma unroll
            for (uint32_t j = 0; j < kMost; ++j) {
                if (j < each && first + j == from) s.found_before = upto;  // (of the list's)
                upto += own[j];
            }
            __syncthreads();
            base -= s.found_before;
            upto = before;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < kMost; ++j) {
            const uint32_t at = first + j, c = count0 + at - from;
            // (the one at which it passes: not before it, but with it)
            if (j < each && at >= from && at < until && target.passed(c + 1, base + upto + own[j]) && (at == from || !target.passed(c, base + upto))) {
                s.found_rank = s.list[at];
                s.found_before = base + upto;
                s.found_sum = base + upto + own[j];
                s.found_count = c + 1;
            }
            upto += own[j];
        }
        __syncthreads();
        return s.found_count != 0;
    }
};

// The j-th (from 1) of the row's tokens with this very logit, by rising index: into found_rank.
template <int kType>
__device__ __forceinline__ void find_equal(const void* row, uint32_t vocab, float value, uint32_t j, Shared& s) {
    // a run of tokens a thread, so that the threads' order is the tokens'
    const uint32_t each = (vocab + kThreads - 1) / kThreads, first = min(threadIdx.x * each, vocab), last = min(first + each, vocab);
    const auto at = [&](uint32_t i) {
        if (kType == 0) return static_cast<const float*>(row)[i];
        const uint16_t bits = static_cast<const uint16_t*>(row)[i];
        return kType == 30 ? __builtin_bit_cast(float, static_cast<uint32_t>(bits) << 16) : static_cast<float>(__builtin_bit_cast(_Float16, bits));
    };
    uint32_t count = 0, before, every;
    u64 unused, none;
    for (uint32_t i = first; i < last; ++i) count += at(i) == value;
    block_before(count, 0, s, &before, &unused, &every, &none);
    if (j > before && j <= before + count) {
        for (uint32_t i = first; i < last; ++i) {
            if (at(i) == value && ++before == j) s.found_rank = rank_of(value, i);
        }
    }
    __syncthreads();
}

struct Histogram {
    float top, low, scale;
    __device__ __forceinline__ bool holds(float v) const { return v >= low; }
    // Below all logits of the bins up to this one, and above all of those from this one on (a bin's number is off by far less than half a bin's width).
    __device__ __forceinline__ float below(uint32_t last) const {
        return scale > 0.0f && last < kBins - 1 ? fmaxf(top - (static_cast<float>(last) + 1.5f) / scale, low) : low;
    }
    __device__ __forceinline__ float above(uint32_t first) const { return scale > 0.0f && first > 0 ? top - (static_cast<float>(first) - 0.5f) / scale : top; }
    __device__ __forceinline__ uint32_t bin(float v) const { return v == top ? 0u : min(static_cast<uint32_t>((top - v) * scale), kBins - 1); }
};

__device__ __forceinline__ void clear_bins(Shared& s) {
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) {
        s.counts[b] = 0;
        s.sums[b] = 0;
    }
    __syncthreads();
}

// Counts and sums of each bin -> of the bins before it; the sums of all are returned.
__device__ __forceinline__ void scan_bins(Shared& s, uint32_t* all_count, u64* all_sum) {
    constexpr uint32_t kEach = kBins / kThreads;
    uint32_t counts[kEach], count = 0, count_before;
    u64 sums[kEach], sum = 0, sum_before;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        counts[j] = s.counts[threadIdx.x * kEach + j];
        sums[j] = s.sums[threadIdx.x * kEach + j];
        count += counts[j];
        sum += sums[j];
    }
    block_before(count, sum, s, &count_before, &sum_before, all_count, all_sum);
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        s.counts[threadIdx.x * kEach + j] = count_before;
        s.sums[threadIdx.x * kEach + j] = sum_before;
        count_before += counts[j];
        sum_before += sums[j];
    }
    __syncthreads();
}

// The first token of the row at which the target is passed (found_*), by the histogram's bins; false: none.  The bins are
// overwritten where one holds more tokens than the list: then `fresh` is cleared, and they have to be made again.
template <int kType>
__device__ bool locate(const void* row, uint32_t vocab, const Histogram& histogram, uint32_t all_count, u64 all_sum, const Target& target,
                       const Weights& weights, Shared& s, bool* fresh) {
    const uint32_t bin = find_bin(target, 0, 0, all_count, all_sum, s);
    if (bin == kBins) return false;
    uint32_t count0 = s.counts[bin];
    u64 sum0 = s.sums[bin];
    uint32_t n = gather<kType>(row, 0, vocab, s, histogram.below(bin), histogram.above(bin), [&](float v) { return histogram.bin(v) == bin; });
    if (n <= kListed) {
        sort_list(n, s);
        return Listed(n, weights, s).find(0, n, count0, sum0, target, s);
    }
    *fresh = false;
    // the bin's range of keys, halved by as many bins as there are until it holds few tokens, or one logit
    if (threadIdx.x == 0) {
        s.key_low = ~0u;
        s.key_high = 0;
    }
    __syncthreads();
    uint32_t low = ~0u, high = 0;
    each_logit<kType>(row, 0, vocab, [&](float v, uint32_t) {
        if (histogram.holds(v) && histogram.bin(v) == bin) {
            low = min(low, key_of(v));
            high = max(high, key_of(v));
        }
    });
    atomicMin(&s.key_low, low);
    atomicMax(&s.key_high, high);
    __syncthreads();
    low = s.key_low;
    high = s.key_high;
    for (;;) {
        if (low == high) {  // n tokens of one logit: the j-th of them
            const u64 w = weights.of(value_of(low));
            uint32_t first = 1, last = n;
            while (first < last) {
                const uint32_t middle = first + (last - first) / 2;
                if (target.passed(count0 + middle, sum0 + middle * w)) last = middle;
                else first = middle + 1;
            }
            if (!target.passed(count0 + first, sum0 + first * w)) return false;
            __syncthreads();
            find_equal<kType>(row, vocab, value_of(low), first, s);
            if (threadIdx.x == 0) {
                s.found_before = sum0 + (first - 1) * w;
                s.found_sum = sum0 + first * w;
                s.found_count = count0 + first;
            }
            __syncthreads();
            return true;
        }
        const int shift = max(0, 32 - __builtin_clz(high - low) - 10);  // 2^10 bins
        __syncthreads();
        clear_bins(s);
        each_logit<kType>(row, 0, vocab, [&](float v, uint32_t) {
            const uint32_t key = key_of(v);
            if (key >= low && key <= high && v > -__builtin_inff()) {
                const uint32_t b = (high - key) >> shift;
                atomicAdd(&s.counts[b], 1u);
                atomicAdd(&s.sums[b], weights.of(v));
            }
        });
        __syncthreads();
        uint32_t count;
        u64 sum;
        scan_bins(s, &count, &sum);
        const uint32_t b = find_bin(target, count0, sum0, count, sum, s);
        if (b == kBins) return false;
        count0 += s.counts[b];
        sum0 += s.sums[b];
        const uint32_t from = high - (b << shift);
        low = max(low, from - ((1u << shift) - 1));  // (the bin's lowest key)
        high = from;
        // (by keys: the value of a highest key right below zero's compares as zero)
        n = gather<kType>(row, 0, vocab, s, value_of(low), value_of(high), [&](float v) { return key_of(v) >= low && key_of(v) <= high && v > -__builtin_inff(); });
        if (n <= kListed) {
            sort_list(n, s);
            return Listed(n, weights, s).find(0, n, count0, sum0, target, s);
        }
    }
}

// What a call's launches pass on of a row.
enum : uint32_t { kDone, kWide, kNarrow };  // drawn; for one workgroup; tokens of some bins are wanted
struct Wanted {                             // bins that a target can fall into, and what is before them
    uint32_t first, last, count;
    u64 sum;
};
struct Row {
    uint32_t spread_arrived, settle_arrived, listed, state;
    float top, cut;
    Wanted of_k, of_p, of_u;
    u64 all, weighty;
    uint32_t all_count;
};
struct Scratch {
    Row* rows;
    u64* best;         // [rows][parts]: ranks
    float* groups;     // [rows][parts][kGroups]
    u64* lists;        // [rows][kListed], as the next two only where a row has several parts
    u64* sums;         // [rows][parts][kBins + 1]: the last the sum of what weighs enough for min-p
    uint32_t* counts;  // [rows][parts][kBins]
    uint32_t parts, part_len;
};

// What a row's filters ask for.
struct Wishes {
    float temperature, p, least, u;
    uint32_t k;
    bool has_p, has_least;
    __device__ __forceinline__ Wishes(const SampleArgs& a, uint32_t r) {
        temperature = a.temperatures != nullptr ? a.temperatures[r] : 1.0f;
        p = a.top_p != nullptr ? a.top_p[r] : 1.0f;
        least = a.min_p != nullptr ? a.min_p[r] : 0.0f;
        u = a.uniforms[r];
        k = a.top_k != nullptr && a.top_k[r] > 0 ? static_cast<uint32_t>(a.top_k[r]) : 0u;
        if (k >= a.vocab) k = 0;
        has_p = p < 1.0f;
        has_least = least > 0.0f;
        if (!(u > 0.0f)) u = 0.0f;
    }
    // The target of the drawn token among tokens of this sum: more than u of it, for a u of 1 or more all of it.
    __device__ __forceinline__ Target draw(u64 kept) const {
        return Target{0, u >= 1.0f ? kept : static_cast<u64>(static_cast<double>(u) * static_cast<double>(kept)) + 1};
    }
    // What a token has to weigh for min-p, as a whole number.
    __device__ __forceinline__ u64 least_sum(u64 one) const {
        return !has_least ? 0 : least >= 1.0f ? (least > 1.0f ? one + 1 : one) : static_cast<u64>(__builtin_ceil(static_cast<double>(least) * static_cast<double>(one)));
    }
    // At least p of this sum (nothing of it: the first token passes).
    __device__ __forceinline__ Target nucleus(u64 kept) const {
        return Target{0, p > 0.0f ? static_cast<u64>(__builtin_ceil(static_cast<double>(p) * static_cast<double>(kept))) : 0};
    }
};

__device__ __forceinline__ Weights weights_of(float top, float temperature, uint32_t vocab) {
    Weights w;
    w.endless = top == __builtin_inff();
    w.per_logit = kLog2e / static_cast<double>(temperature);
    w.largest = static_cast<double>(top);
    w.top = top;
    w.bits = min(46, 62 - (32 - __builtin_clz(vocab - 1 | 1)));  // (the sum of all stays below 2^62)
    return w;
}

__device__ __forceinline__ Histogram histogram_of(float top, float cut) {
    Histogram h{top, cut, 0.0f};
    h.scale = top > cut && top < __builtin_inff() ? static_cast<float>(kBins - 1) / (top - cut) : 0.0f;
    return h;
}

__device__ __forceinline__ const void* row_of(const SampleArgs& a, uint32_t r, int size) { return static_cast<const char*>(a.logits) + r * a.row_stride * size; }

__device__ __forceinline__ void put(const SampleArgs& a, uint32_t r, int token, float probability) {
    a.tokens[r] = token;
    if (a.probabilities != nullptr) a.probabilities[r] = probability;
}
__device__ __forceinline__ void put_drawn(const SampleArgs& a, uint32_t r, u64 rank, const Weights& w, u64 kept) {
    put(a, r, static_cast<int>(static_cast<uint32_t>(rank)), static_cast<float>(w.fraction(value_at(rank)) * static_cast<double>(1ull << w.bits) / static_cast<double>(kept)));
}

// What a row's workgroups tell one another within a launch goes past the caches that they do not share (relaxed atomics of the
// device's scope): a fence for all else that they wrote would write back and drop an XCD's whole L2 (the second launch
// over 256 rows of 128000 takes five times as long with such fences).
template <typename T>
__device__ __forceinline__ void tell(T* to, T v) { __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
__device__ __forceinline__ T told(const T* from) { return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The row's first token, from its parts' (a lane a part: no load waits for another).
__device__ __forceinline__ u64 best_of(const Scratch& scratch, uint32_t r) {
    const uint32_t lane = threadIdx.x & 63;
    u64 best = lane < scratch.parts ? scratch.best[static_cast<size_t>(r) * scratch.parts + lane] : ~0ull;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) best = min(best, static_cast<u64>(__shfl_xor(best, d)));
    return best;
}

// Whether this is the last of the row's workgroups to come here; all that the others told is there then.
__device__ __forceinline__ bool last_of(uint32_t* arrived, uint32_t parts, Shared& s) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what this thread told has arrived
    __syncthreads();
    if (threadIdx.x == 0) s.found_bin = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const bool last = s.found_bin == parts - 1;
    __syncthreads();
    return last;
}

// The row's tokens that `wants` says, none of them below `low` or above `high`, into the list in LDS, by its parts: true for the last of them, which has them all (as far as
// there is room; *n: how many there are).
template <int kType, typename Wants>
__device__ __forceinline__ bool list_row(const SampleArgs& a, const Scratch& scratch, uint32_t r, uint32_t part, uint32_t* arrived, Shared& s, float low, float high, Wants wants, uint32_t* n) {
    const void* row = row_of(a, r, kType == 0 ? 4 : 2);
    const uint32_t begin = part * scratch.part_len, end = min(begin + scratch.part_len, a.vocab);
    *n = gather<kType>(row, begin, end, s, low, high, wants);
    if (scratch.parts == 1) return true;
    // behind the other parts' (one addition a part: thousands to one place of memory would follow one another)
    Row* const state = scratch.rows + r;
    u64* const list = scratch.lists + static_cast<size_t>(r) * kListed;
    if (threadIdx.x == 0) s.found_count = __hip_atomic_fetch_add(&state->listed, *n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const uint32_t at = s.found_count;
    for (uint32_t i = threadIdx.x; i < min(*n, kListed) && at + i < kListed; i += kThreads) tell(list + at + i, s.list[i]);
    if (!last_of(arrived, scratch.parts, s)) return false;
    *n = told(&state->listed);
    for (uint32_t i = threadIdx.x; i < min(*n, kListed); i += kThreads) s.list[i] = told(list + i);
    __syncthreads();
    return true;
}

template <int kType>
__global__ __launch_bounds__(kThreads) void most_kernel(SampleArgs a, Scratch scratch) {
    __shared__ u64 ranks[kWaves];
    const uint32_t r = blockIdx.y, part = blockIdx.x, begin = part * scratch.part_len, end = min(begin + scratch.part_len, a.vocab);
    float most = -__builtin_inff();
    uint32_t most_at = 0xFFFFFFFFu;
    each_logit<kType>(row_of(a, r, kType == 0 ? 4 : 2), begin, end, [&](float v, uint32_t i) {
        if (v > most) {
            most = v;
            most_at = i;
        }
    });
    float four = fmaxf(most, __shfl_xor(most, 1));
    four = fmaxf(four, __shfl_xor(four, 2));
    if ((threadIdx.x & 3) == 0) scratch.groups[(static_cast<size_t>(r) * scratch.parts + part) * kGroups + threadIdx.x / 4] = four;
    u64 best = rank_of(most, most_at);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u64 other = __shfl_xor(best, d);
        best = other < best ? other : best;
    }
    if ((threadIdx.x & 63) == 0) ranks[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) best = ranks[w] < best ? ranks[w] : best;
        scratch.best[static_cast<size_t>(r) * scratch.parts + part] = best;
        if (part == 0) {
            Row* state = scratch.rows + r;
            state->spread_arrived = state->settle_arrived = state->listed = 0;
            state->state = kDone;
        }
    }
}

// Draws from a row's first tokens, all that its filters can keep, in the sorted list.
__device__ __forceinline__ void draw_listed(const SampleArgs& a, uint32_t r, const Wishes& wishes, const Weights& weights, uint32_t n, u64 best, Shared& s) {
    const u64 one = 1ull << weights.bits;
    const u64 least_sum = wishes.least_sum(one);
    const uint32_t ranked = wishes.k != 0 && wishes.k < n ? wishes.k : n;
    const Listed listed(ranked, weights, s);
    u64 kept = listed.all;
    if (wishes.has_p) {
        if (listed.find(0, ranked, 0, 0, wishes.nucleus(kept), s)) kept = s.found_sum;
        __syncthreads();
    }
    if (wishes.has_least) {
        u64 over = 0;
#pragma unroll
        for (uint32_t j = 0; j < Listed::kMost; ++j) over += listed.own[j] >= least_sum ? listed.own[j] : 0;
        kept = min(kept, block_sum(over, s));
    }
    kept = max(kept, one);
    const bool found = listed.find(0, ranked, 0, 0, wishes.draw(kept), s);
    if (threadIdx.x == 0) put_drawn(a, r, found ? s.found_rank : best, weights, kept);
}

template <int kType>
__global__ __launch_bounds__(kThreads) void spread_kernel(SampleArgs a, Scratch scratch) {
    __shared__ Shared s;
    const uint32_t r = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, parts = scratch.parts;
    const uint32_t begin = part * scratch.part_len, end = min(begin + scratch.part_len, a.vocab);
    const Wishes wishes(a, r);
    const u64 best = best_of(scratch, r);
    const float top = value_at(best);
    if (top == -__builtin_inff() || !(wishes.temperature > 0.0f)) {
        if (part == 0 && tid == 0) put(a, r, top == -__builtin_inff() ? -1 : static_cast<int>(static_cast<uint32_t>(best)), top == -__builtin_inff() ? 0.0f : 1.0f);
        return;
    }
    const Weights weights = weights_of(top, wishes.temperature, a.vocab);
    const u64 one = 1ull << weights.bits;

    // ---- below which logit no token can be kept, or count in a sum: the logits' own roundings and the division's leave a margin
    const auto cut_at = [&](double power) {
        const double v = static_cast<double>(top) + power / weights.per_logit * 1.000001;
        return static_cast<float>(v - __builtin_fabs(v) * 0x1p-22);
    };
    float cut = top == __builtin_inff() ? top : cut_at(-1.5 - weights.bits);
    bool few = false;  // whether the cut is likely to leave a list
    const uint32_t groups = parts * kGroups;
    const bool by_rank = wishes.k != 0 && wishes.k <= groups, by_weight = wishes.has_least && !wishes.has_p && top < __builtin_inff();
    if (by_rank || by_weight) {
        constexpr uint32_t kOwn = kMostParts * kGroups / kThreads;
        uint32_t keys[kOwn];
#pragma unroll
        for (uint32_t j = 0; j < kOwn; ++j) keys[j] = tid + j * kThreads < groups ? key_of(scratch.groups[static_cast<size_t>(r) * groups + tid + j * kThreads]) : 0u;
        uint32_t turn = 0;
        // the groups whose largest is at least as much as each of three keys
        const auto reach = [&](const uint32_t (&with)[3], uint32_t (&all)[3]) {
            uint32_t own[3] = {0, 0, 0};
#pragma unroll
            for (uint32_t j = 0; j < kOwn; ++j) {
                if (j * kThreads >= groups) break;
#pragma unroll
                for (int i = 0; i < 3; ++i) own[i] += __popcll(__ballot(keys[j] >= with[i]));
            }
            uint32_t* counts = s.counts + (turn++ & 1) * (4 * kWaves);  // (two in turn: one barrier each)
            if ((tid & 63) == 0) {
#pragma unroll
                for (int i = 0; i < 3; ++i) counts[(tid >> 6) * 4 + i] = own[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 3; ++i) all[i] = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
#pragma unroll
                for (int i = 0; i < 3; ++i) all[i] += counts[w * 4 + i];
            }
        };
        if (by_rank) {
            // the k-th largest of the groups' largest, two bits at a time: with the lowest 14 of them left zero it is a bound as well
            uint32_t found = 0;
            for (int bit = 30; bit >= 14; bit -= 2) {
                const uint32_t with[3] = {found | 1u << bit, found | 2u << bit, found | 3u << bit};
                uint32_t all[3];
                reach(with, all);
                found = all[2] >= wishes.k ? with[2] : all[1] >= wishes.k ? with[1] : all[0] >= wishes.k ? with[0] : found;
            }
            cut = fmaxf(cut, value_of(found));
        }
        if (by_weight) cut = fmaxf(cut, cut_at(wishes.least >= 1.0f ? 0.0 : static_cast<double>(__builtin_log2f(wishes.least)) - 1e-4));
        // Of tokens that lie above the cut at random, a group of many has one with 1 - exp(-their share): no more than a list holds, with room
        // for chance.  Lists of up to 1000 tokens or so are the shorter way, longer ones than these 0.7 let pass are not, and some of what lies
        // between would do better without: 24 rows of 100003 with a min-p that 800 tokens pass take 31 us, that 1600 pass 44 by lists and 33 by
        // histograms, 2200 70 and 33; 64 rows of 64000 33, 48 and 35, 80 and 36.
        const uint32_t at_cut = key_of(fmaxf(cut, -3.402823466e38f)), with[3] = {at_cut, at_cut, at_cut};
        uint32_t over_cut[3];
        reach(with, over_cut);
        const float share = static_cast<float>(over_cut[0]) / static_cast<float>(groups);
        few = share < 1.0f && -__builtin_log2f(1.0f - share) * static_cast<float>(groups) < 0.7f * static_cast<float>(kListed);
    }
    cut = fminf(fmaxf(cut, -3.402823466e38f), top);  // (minus infinity counts for nothing)
    Row* const state = scratch.rows + r;

    if (few) {
        uint32_t n;
        if (!list_row<kType>(a, scratch, r, part, &state->spread_arrived, s, cut, top, [](float) { return true; }, &n)) return;
        if (n > kListed) {
            if (tid == 0) {
                state->state = kWide;
                state->top = top;
                state->cut = cut;
            }
            return;
        }
        sort_list(n, s);
        draw_listed(a, r, wishes, weights, n, best, s);
        return;
    }

    // Lanes take turns among four copies of the sums, in the list's place: neighbouring tokens' bins are often the same, and additions
    // to one place of LDS follow one another.  Counts are made where top-k asks for them.
    const Histogram histogram = histogram_of(top, cut);
    const u64 least_sum = wishes.least_sum(one);
    const bool counted = wishes.k != 0;
    constexpr uint32_t kCopies = kListed / kBins;
    __syncthreads();
    clear_bins(s);
    for (uint32_t b = tid; b < kListed; b += kThreads) s.list[b] = 0;
    __syncthreads();
    u64 over = 0;
    each_logit<kType>(row_of(a, r, kType == 0 ? 4 : 2), begin, end, [&](float v, uint32_t) {
        if (histogram.holds(v)) {
            const uint32_t b = histogram.bin(v);
            const u64 w = weights.of(v);
            if (counted) atomicAdd(&s.counts[b], 1u);
            atomicAdd(&s.list[b * kCopies + (tid & (kCopies - 1))], w);
            if (w >= least_sum) over += w;
        }
    });
    __syncthreads();
    for (uint32_t b = tid; b < kBins; b += kThreads) {
        u64 sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < kCopies; ++i) sum += s.list[b * kCopies + i];
        s.sums[b] = sum;
    }
    __syncthreads();
    over = block_sum(over, s);
    u64* const sums = scratch.sums + static_cast<size_t>(r) * parts * (kBins + 1);
    uint32_t* const counts = scratch.counts + static_cast<size_t>(r) * parts * kBins;
    if (parts > 1) {
        for (uint32_t b = tid; b < kBins; b += kThreads) {
            tell(sums + part * (kBins + 1) + b, s.sums[b]);
            if (counted) tell(counts + part * kBins + b, s.counts[b]);
        }
        if (tid == 0) tell(sums + part * (kBins + 1) + kBins, over);
        if (!last_of(&state->spread_arrived, parts, s)) return;
        constexpr uint32_t kAtOnce = 8;  // parts whose numbers are asked for together
        for (uint32_t b = tid; b < kBins; b += kThreads) {
            u64 sum = 0;
            uint32_t count = 0;
            for (uint32_t i0 = 0; i0 < parts; i0 += kAtOnce) {
                u64 held[kAtOnce];
                uint32_t held_counts[kAtOnce];
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce; ++i) {
                    held[i] = i0 + i < parts ? told(sums + (i0 + i) * (kBins + 1) + b) : 0;
                    held_counts[i] = counted && i0 + i < parts ? told(counts + (i0 + i) * kBins + b) : 0;
                }
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce; ++i) {
                    sum += held[i];
                    count += held_counts[i];
                }
            }
            s.sums[b] = sum;
            s.counts[b] = count;
        }
        over = block_sum(tid < parts ? told(sums + tid * (kBins + 1) + kBins) : 0, s);
    }

    // ---- the bins that the filters' and the draw's targets can fall into: what the earlier ones leave is known to a bin
    uint32_t all_count;
    u64 all;
    scan_bins(s, &all_count, &all);
    const auto before = [&](uint32_t bin) { return bin < kBins ? s.sums[bin] : all; };
    const auto bin_of = [&](const Target& target) { return min(find_bin(target, 0, 0, all_count, all, s), kBins - 1); };
    const auto wanted = [&](uint32_t first, uint32_t last) { return Wanted{first, last, s.counts[first], s.sums[first]}; };
    const Wanted none{1, 0, 0, 0};
    Wanted of_k = none, of_p = none;
    u64 low = all, high = all;  // between which the sum of what is kept so far lies
    if (wishes.k != 0 && wishes.k < all_count) {
        const uint32_t b = bin_of(Target{wishes.k, 0});
        of_k = wanted(b, b);
        low = before(b);
        high = before(b + 1);
    }
    if (wishes.has_p) {
        const uint32_t first = bin_of(wishes.nucleus(low));
        const uint32_t last = low == high ? first : bin_of(wishes.nucleus(high));
        of_p = wanted(first, last);
        low = before(first);
        high = before(last + 1);
    }
    if (wishes.has_least) {
        low = min(low, over);
        high = min(high, over);
    }
    low = max(low, one);
    high = max(high, one);
    const uint32_t first = bin_of(wishes.draw(low));
    const uint32_t last = low == high ? first : bin_of(wishes.draw(high));
    if (tid == 0) {
        state->of_k = of_k;
        state->of_p = of_p;
        state->of_u = wanted(first, max(first, last));
        state->all = all;
        state->weighty = over;
        state->all_count = all_count;
        state->top = top;
        state->cut = cut;
        state->state = kNarrow;
    }
}

// A row by one workgroup, whatever it holds.
template <int kType>
__device__ __forceinline__ void draw_wide(const SampleArgs& a, uint32_t r, float top, float cut, u64 best, Shared& s) {
    const Wishes wishes(a, r);
    const void* row = row_of(a, r, kType == 0 ? 4 : 2);
    const Weights weights = weights_of(top, wishes.temperature, a.vocab);
    const Histogram histogram = histogram_of(top, cut);
    const u64 one = 1ull << weights.bits;
    const u64 least_sum = wishes.least_sum(one);
    uint32_t all_count = 0;
    u64 all = 0, weighty = 0, kept = 0;
    bool fresh = false, found = false;
    for (int step = 0; step < 3; ++step) {  // the first k, the nucleus, the draw
        if (!fresh) {
            __syncthreads();
            clear_bins(s);
            u64 over = 0;
            each_logit<kType>(row, 0, a.vocab, [&](float v, uint32_t) {
                if (histogram.holds(v)) {
                    const uint32_t b = histogram.bin(v);
                    const u64 w = weights.of(v);
                    atomicAdd(&s.counts[b], 1u);
                    atomicAdd(&s.sums[b], w);
                    if (w >= least_sum) over += w;
                }
            });
            __syncthreads();
            weighty = block_sum(over, s);
            scan_bins(s, &all_count, &all);
            fresh = true;
        }
        if (step == 0) kept = all;
        if (step == 2) kept = max(wishes.has_least ? min(kept, weighty) : kept, one);
        if ((step == 0 && (wishes.k == 0 || wishes.k >= all_count)) || (step == 1 && !wishes.has_p)) continue;
        const Target target = step == 0 ? Target{wishes.k, 0} : step == 1 ? wishes.nucleus(kept) : wishes.draw(kept);
        found = locate<kType>(row, a.vocab, histogram, all_count, all, target, weights, s, &fresh);
        if (found && step < 2) kept = s.found_sum;
        __syncthreads();
    }
    if (threadIdx.x == 0) put_drawn(a, r, found ? s.found_rank : best, weights, kept);
}

template <int kType>
__global__ __launch_bounds__(kThreads, 4) void settle_kernel(SampleArgs a, Scratch scratch) {
    __shared__ Shared s;
    const uint32_t r = blockIdx.y, part = blockIdx.x, tid = threadIdx.x;
    Row* const state = scratch.rows + r;
    const uint32_t todo = state->state;
    if (todo == kDone || (todo == kWide && part != 0)) return;
    const float top = state->top, cut = state->cut;
    const u64 best = best_of(scratch, r);
    bool wide = todo == kWide;
    const Wishes wishes(a, r);
    const Weights weights = weights_of(top, wishes.temperature, a.vocab);
    const Histogram histogram = histogram_of(top, cut);
    const Wanted of_k = state->of_k, of_p = state->of_p, of_u = state->of_u;
    const auto in = [](const Wanted& w, uint32_t b) { return b >= w.first && b <= w.last; };
    const auto wants = [&](float v) {
        const uint32_t b = histogram.bin(v);
        return in(of_u, b) || in(of_p, b) || in(of_k, b);
    };
    // (a target that is not there has bins 1 to 0)
    const float low = histogram.below(max(of_u.last, max(of_p.last, of_k.last)));
    const float high = histogram.above(min(of_u.first, min(of_p.first <= of_p.last ? of_p.first : of_u.first, of_k.first <= of_k.last ? of_k.first : of_u.first)));
    uint32_t n = 0;
    if (!wide) {
        if (!list_row<kType>(a, scratch, r, part, &state->settle_arrived, s, low, high, wants, &n)) return;
        wide = n > kListed;
    }
    if (wide) {
        draw_wide<kType>(a, r, top, cut, best, s);
        return;
    }
    sort_list(n, s);
    const Listed listed(n, weights, s);
    // the run of the list that is of these bins
    const auto find = [&](const Wanted& w, const Target& target) {
        uint32_t mine = 0, within = 0;
        for (uint32_t i = tid; i < n; i += kThreads) {
            const uint32_t b = histogram.bin(value_at(s.list[i]));
            mine += b < w.first;
            within += in(w, b);
        }
        const u64 both = block_sum(static_cast<u64>(mine) << 32 | within, s);
        const uint32_t from = static_cast<uint32_t>(both >> 32);
        return listed.find(from, from + static_cast<uint32_t>(both), w.count, w.sum, target, s);
    };
    u64 kept = state->all;
    if (of_k.first <= of_k.last) {
        if (find(of_k, Target{wishes.k, 0})) kept = s.found_sum;
        __syncthreads();
    }
    if (wishes.has_p) {
        if (find(of_p, wishes.nucleus(kept))) kept = s.found_sum;
        __syncthreads();
    }
    if (wishes.has_least) kept = min(kept, state->weighty);
    kept = max(kept, 1ull << weights.bits);
    const bool found = find(of_u, wishes.draw(kept));
    if (tid == 0) put_drawn(a, r, found ? s.found_rank : best, weights, kept);
}

struct Layout {
    uint32_t parts, part_len;
    size_t best, groups, lists, sums, counts, bytes;  // where they begin, behind the rows' states
};

// A row's parts: as many as give every unit two workgroups, of 8192 tokens at least: what a workgroup does besides reading its
// tokens takes 10 us (256 rows of 128000 with top-k 50: 61 us in two parts, 72 in four, 102 in eight).
Layout layout_of(const SampleArgs& a, int compute_units) {
    Layout l{};
    const uint64_t wanted = (2 * static_cast<uint64_t>(compute_units) + a.rows - 1) / a.rows, most = (a.vocab + 8191) / 8192;
    l.parts = static_cast<uint32_t>(wanted < most ? wanted : most);
    if (l.parts > kMostParts) l.parts = kMostParts;
    l.part_len = ((a.vocab + l.parts - 1) / l.parts + 7) / 8 * 8;
    l.parts = (a.vocab + l.part_len - 1) / l.part_len;
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t rows = a.rows, all = rows * l.parts;
    l.best = up(rows * sizeof(Row));
    l.groups = l.best + up(all * sizeof(u64));
    l.lists = l.groups + up(all * kGroups * sizeof(float));
    l.sums = l.lists + (l.parts > 1 ? rows * kListed * sizeof(u64) : 0);
    l.counts = l.sums + (l.parts > 1 ? up(all * (kBins + 1) * sizeof(u64)) : 0);
    l.bytes = l.counts + (l.parts > 1 ? up(all * kBins * sizeof(uint32_t)) : 0);
    return l;
}

template <int kType>
hipError_t sample(hipStream_t stream, const SampleArgs& a, void* workspace, const Layout& l) {
    char* const at = static_cast<char*>(workspace);
    const Scratch scratch{reinterpret_cast<Row*>(at), reinterpret_cast<u64*>(at + l.best), reinterpret_cast<float*>(at + l.groups), reinterpret_cast<u64*>(at + l.lists),
                          reinterpret_cast<u64*>(at + l.sums), reinterpret_cast<uint32_t*>(at + l.counts), l.parts, l.part_len};
    const dim3 grid(l.parts, a.rows);
    most_kernel<kType><<<grid, kThreads, 0, stream>>>(a, scratch);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    spread_kernel<kType><<<grid, kThreads, 0, stream>>>(a, scratch);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    settle_kernel<kType><<<grid, kThreads, 0, stream>>>(a, scratch);
    return hipGetLastError();
}

}  // namespace

size_t sample_workspace_bytes(const SampleArgs& args, int compute_units) { return layout_of(args, compute_units).bytes; }

hipError_t launch_sample(hipStream_t stream, const SampleArgs& a, void* workspace, int compute_units) {
    const Layout l = layout_of(a, compute_units);
    if (a.type == 0) return sample<0>(stream, a, workspace, l);
    if (a.type == 1) return sample<1>(stream, a, workspace, l);
    return sample<30>(stream, a, workspace, l);
}

}  // namespace afhip
