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
// A workgroup has a row.  It reads the row once for its largest logit, and once more for the candidates, where a cut is known that
// leaves few: every thread's own largest logit is at hand after the first pass, and the k-th largest of these is below the k-th
// largest of all; min-p's cut follows from the largest.  Otherwise the second pass makes a histogram of counts and sums over the
// logits' range, a third (a fourth) reads the tokens of the bin that a target falls into.
#include "quantized_launch.h"

#include <hip/hip_runtime.h>

namespace afhip {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr uint32_t kBins = 2048, kListed = 4096;
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
    __device__ __forceinline__ double power(float v) const {  // of two
        return v == top ? 0.0 : (static_cast<double>(v) - largest) * per_logit;
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
        if (!(y > -1.0 - bits)) return 0;  // (minus infinity, and no number, among them)
        // added to 2^52 it is rounded to a whole number, which the sum's lower bits are
        return __builtin_bit_cast(u64, exp2_scaled(y, bits) + 0x1p52) & ((1ull << 52) - 1);
    }
    __device__ __forceinline__ double fraction(float v) const {
        const double y = power(v);
        return y > -1000.0 ? exp2_scaled(y, 0) : 0.0;
    }
};

struct Shared {
    u64 list[kListed];
    u64 sums[kBins];
    uint32_t counts[kBins];
    u64 wave_sums[kWaves];
    uint32_t wave_counts[kWaves];
    u64 wave_ranks[kWaves];
    u64 found_sum, found_before, found_rank;
    uint32_t found_count, found_bin, listed, key_low, key_high;
};

template <typename T>
__device__ __forceinline__ T shuffled_up(T v, int d) { return __shfl_up(v, d); }

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

// Sums of counts and sums over the threads before this one.
__device__ __forceinline__ void block_before(uint32_t count, u64 sum, Shared& s, uint32_t* count_before, u64* sum_before) {
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
    for (int w = 0; w < wave; ++w) {
        c += s.wave_counts[w];
        m += s.wave_sums[w];
    }
    __syncthreads();
    *count_before = c;
    *sum_before = m;
}

// What passes: the count, or the sum in 64-bit floating point, up to and with a token.
struct Target {
    uint32_t count;   // at least so many tokens, where not zero
    double sum;       // otherwise: at least, or more than, this sum
    bool more;
    __device__ __forceinline__ bool passed(uint32_t c, u64 m) const {
        if (count != 0) return c >= count;
        return more ? static_cast<double>(m) > sum : static_cast<double>(m) >= sum;
    }
};

// Every logit of the row by f(v, i), a thread's own in rising order; no numbers are minus infinity.
template <int kType, typename F>
__device__ __forceinline__ void each_logit(const void* row, uint32_t vocab, F f) {
    constexpr int kPer = kType == 0 ? 4 : 8;
    struct __attribute__((packed, aligned(kType == 0 ? 4 : 2))) Run { uint32_t words[4]; };  // (rows start at any element)
    const uint32_t runs = vocab / kPer;
    const auto value = [](uint32_t word, int part) {
        float v;
        if (kType == 0) v = __builtin_bit_cast(float, word);
        else if (kType == 30) v = __builtin_bit_cast(float, part == 0 ? word << 16 : word & 0xFFFF0000u);
        else v = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(word >> (16 * part))));
        return v == v ? v : -__builtin_inff();
    };
    const auto visit = [&](const Run& r, uint32_t run) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) f(value(r.words[kType == 0 ? j : j / 2], kType == 0 ? 0 : j % 2), run * kPer + j);
    };
    const Run* from = static_cast<const Run*>(row);
    constexpr uint32_t kAhead = 4;
    uint32_t run = threadIdx.x;
    for (; run + (kAhead - 1) * kThreads < runs; run += kAhead * kThreads) {
        Run held[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) held[j] = from[run + j * kThreads];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) visit(held[j], run + j * kThreads);
    }
    for (; run < runs; run += kThreads) visit(from[run], run);
    for (uint32_t i = runs * kPer + threadIdx.x; i < vocab; i += kThreads) {
        const uint32_t word = kType == 0 ? static_cast<const uint32_t*>(row)[i] : static_cast<const uint16_t*>(row)[i];
        f(value(word, 0), i);
    }
}

// The tokens that `wanted` says, into the list as far as it has room; how many there are.
template <int kType, typename Wanted>
__device__ __forceinline__ uint32_t gather(const void* row, uint32_t vocab, Shared& s, Wanted wanted) {
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    each_logit<kType>(row, vocab, [&](float v, uint32_t i) {
        if (wanted(v)) {
            const uint32_t at = atomicAdd(&s.listed, 1u);
            if (at < kListed) s.list[at] = rank_of(v, i);
        }
    });
    __syncthreads();
    return s.listed;
}

// The list's first n entries in rising order.
__device__ __forceinline__ void sort_list(uint32_t n, Shared& s) {
    uint32_t size = 2;
    while (size < n) size *= 2;
    for (uint32_t i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = ~0ull;
    for (uint32_t k = 2; k <= size; k *= 2) {
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (uint32_t at = threadIdx.x; at < size / 2; at += kThreads) {
                const uint32_t i = 2 * at - (at & (j - 1)), other = i + j;
                const u64 a = s.list[i], b = s.list[other];
                if ((a > b) == ((i & k) == 0)) {
                    s.list[i] = b;
                    s.list[other] = a;
                }
            }
        }
    }
    __syncthreads();
}

// The first of the sorted list's n tokens at which the target is passed, counts and sums before the list being given: into
// found_rank, found_sum (with it), found_before and found_count (with it).  False: none.
__device__ __forceinline__ bool find_listed(uint32_t n, uint32_t count0, u64 sum0, const Target& target, const Weights& weights, Shared& s) {
    constexpr uint32_t kEach = kListed / kThreads;
    const uint32_t first = threadIdx.x * kEach;
    u64 own[kEach], sum = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        own[j] = first + j < n ? weights.of(value_at(s.list[first + j])) : 0;
        sum += own[j];
    }
    uint32_t count;
    u64 before;
    block_before(0, sum, s, &count, &before);
    if (threadIdx.x == 0) s.found_count = 0;
    __syncthreads();
    before += sum0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        const uint32_t c = count0 + first + j;
        // (the one at which it passes: not before it, but with it)
        if (first + j < n && target.passed(c + 1, before + own[j]) && (first + j == 0 || !target.passed(c, before))) {
            s.found_rank = s.list[first + j];
            s.found_before = before;
            s.found_sum = before + own[j];
            s.found_count = c + 1;
        }
        before += own[j];
    }
    __syncthreads();
    return s.found_count != 0;
}

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
    uint32_t count = 0, before;
    u64 unused;
    for (uint32_t i = first; i < last; ++i) count += at(i) == value;
    block_before(count, 0, s, &before, &unused);
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
    block_before(count, sum, s, &count_before, &sum_before);
    if (threadIdx.x == kThreads - 1) {
        s.found_count = count_before + count;
        s.found_sum = sum_before + sum;
    }
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        s.counts[threadIdx.x * kEach + j] = count_before;
        s.sums[threadIdx.x * kEach + j] = sum_before;
        count_before += counts[j];
        sum_before += sums[j];
    }
    __syncthreads();
    *all_count = s.found_count;
    *all_sum = s.found_sum;
    __syncthreads();
}

// The bin in which the target is passed (kBins: none), behind the counts and sums of those before it.
__device__ __forceinline__ uint32_t find_bin(const Target& target, uint32_t count0, u64 sum0, uint32_t all_count, u64 all_sum, Shared& s) {
    if (threadIdx.x == 0) s.found_bin = kBins;
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) {
        const uint32_t c = s.counts[b], next_c = b + 1 < kBins ? s.counts[b + 1] : all_count;
        const u64 m = s.sums[b], next_m = b + 1 < kBins ? s.sums[b + 1] : all_sum;
        if (next_c > c && target.passed(count0 + next_c, sum0 + next_m) && (c == 0 || !target.passed(count0 + c, sum0 + m))) s.found_bin = b;
    }
    __syncthreads();
    return s.found_bin;
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
    uint32_t n = gather<kType>(row, vocab, s, [&](float v) { return histogram.holds(v) && histogram.bin(v) == bin; });
    if (n <= kListed) {
        sort_list(n, s);
        return find_listed(n, count0, sum0, target, weights, s);
    }
    *fresh = false;
    // the bin's range of keys, halved by as many bins as there are until it holds few tokens, or one logit
    if (threadIdx.x == 0) {
        s.key_low = ~0u;
        s.key_high = 0;
    }
    __syncthreads();
    uint32_t low = ~0u, high = 0;
    each_logit<kType>(row, vocab, [&](float v, uint32_t) {
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
        const int shift = max(0, 32 - __builtin_clz(high - low) - 11);
        __syncthreads();
        clear_bins(s);
        each_logit<kType>(row, vocab, [&](float v, uint32_t) {
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
        low = max(low, from - ((1u << shift) - 1));
        high = from;
        n = gather<kType>(row, vocab, s, [&](float v) { const uint32_t key = key_of(v); return key >= low && key <= high && v > -__builtin_inff(); });
        if (n <= kListed) {
            sort_list(n, s);
            return find_listed(n, count0, sum0, target, weights, s);
        }
    }
}

template <int kType>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const uint32_t r = blockIdx.x, tid = threadIdx.x;
    const void* row = static_cast<const char*>(a.logits) + r * a.row_stride * (kType == 0 ? 4 : 2);
    const float temperature = a.temperatures != nullptr ? a.temperatures[r] : 1.0f, p = a.top_p != nullptr ? a.top_p[r] : 1.0f;
    const float least = a.min_p != nullptr ? a.min_p[r] : 0.0f;
    float u = a.uniforms[r];
    uint32_t k = a.top_k != nullptr && a.top_k[r] > 0 ? static_cast<uint32_t>(a.top_k[r]) : 0u;
    if (k >= a.vocab) k = 0;
    const bool has_p = p < 1.0f, has_least = least > 0.0f;
    if (!(u > 0.0f)) u = 0.0f;

    // ---- the largest
    float most = -__builtin_inff();
    uint32_t most_at = 0xFFFFFFFFu;
    each_logit<kType>(row, a.vocab, [&](float v, uint32_t i) {
        if (v > most) {
            most = v;
            most_at = i;
        }
    });
    u64 best = rank_of(most, most_at);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u64 other = __shfl_xor(best, d);
        best = other < best ? other : best;
    }
    if ((tid & 63) == 0) s.wave_ranks[tid >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) best = s.wave_ranks[w] < best ? s.wave_ranks[w] : best;
    const float top = value_at(best);
    if (top == -__builtin_inff() || !(temperature > 0.0f)) {
        if (tid == 0) {
            a.tokens[r] = top == -__builtin_inff() ? -1 : static_cast<int>(static_cast<uint32_t>(best));
            if (a.probabilities != nullptr) a.probabilities[r] = top == -__builtin_inff() ? 0.0f : 1.0f;
        }
        return;
    }

    Weights weights;
    weights.largest = static_cast<double>(top);
    weights.per_logit = kLog2e / static_cast<double>(temperature);
    weights.top = top;
    weights.bits = min(50, 62 - (32 - __builtin_clz(a.vocab - 1 | 1)));  // (the sum of all stays below 2^62)
    const u64 one = 1ull << weights.bits;

    // ---- below which logit no token can be kept, or count in a sum: the logits' own roundings and the division's leave a margin
    const auto cut_at = [&](double power) {
        const double v = weights.largest + power / weights.per_logit * 1.000001;
        return static_cast<float>(v - __builtin_fabs(v) * 0x1p-22);
    };
    float cut = top == __builtin_inff() ? top : cut_at(-1.5 - weights.bits);
    bool few = false;  // whether the cut is likely to leave a list
    constexpr uint32_t kMostRanked = kThreads;
    if (k != 0 && k <= kMostRanked) {
        // the k-th largest of the threads' largest, bit by bit
        const uint32_t mine = key_of(most);
        uint32_t found = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t with = found | 1u << bit;
            if (static_cast<uint32_t>(__syncthreads_count(mine >= with)) >= k) found = with;
        }
        const float kth = value_of(found);
        if (kth > cut) cut = kth;
        few = true;
    }
    if (has_least && !has_p && top < __builtin_inff()) {
        const float at = cut_at(least >= 1.0f ? 0.0 : static_cast<double>(__builtin_log2f(least)) - 1e-4);
        if (at > cut) cut = at;
        few = true;
    }
    cut = fminf(fmaxf(cut, -3.402823466e38f), top);  // (minus infinity counts for nothing)
    const double least_sum = static_cast<double>(least) * static_cast<double>(one);

    u64 kept = 0;
    bool found = false;
    if (few) {
        const uint32_t n = gather<kType>(row, a.vocab, s, [&](float v) { return v >= cut; });
        if (n <= kListed) {
            sort_list(n, s);
            constexpr uint32_t kEach = kListed / kThreads;
            const uint32_t ranked = k != 0 && k < n ? k : n;
            u64 upto = 0, over = 0;
#pragma unroll
            for (uint32_t j = 0; j < kEach; ++j) {
                const uint32_t i = tid * kEach + j;
                if (i < ranked) {
                    const u64 w = weights.of(value_at(s.list[i]));
                    upto += w;
                    if (!has_least || static_cast<double>(w) >= least_sum) over += w;
                }
            }
            kept = block_sum(upto, s);
            if (has_p) {
                find_listed(ranked, 0, 0, Target{0, static_cast<double>(p) * static_cast<double>(kept), false}, weights, s);
                kept = s.found_sum;
                __syncthreads();
            }
            const u64 weighty = block_sum(over, s);
            kept = min(kept, weighty);
            kept = max(kept, one);
            const double target = static_cast<double>(u) * static_cast<double>(kept);
            const bool last = u >= 1.0f;
            found = find_listed(ranked, 0, 0, Target{0, last ? static_cast<double>(kept) : target, !last}, weights, s);
        }
    }
    if (!found) {
        Histogram histogram{top, cut, 0.0f};
        histogram.scale = top > cut && top < __builtin_inff() ? static_cast<float>(kBins - 1) / (top - cut) : 0.0f;
        uint32_t all_count = 0;
        u64 all = 0, weighty = 0;
        bool fresh = false;
        const auto fill = [&] {
            if (fresh) return;
            __syncthreads();
            clear_bins(s);
            u64 over = 0;
            each_logit<kType>(row, a.vocab, [&](float v, uint32_t) {
                if (histogram.holds(v)) {
                    const uint32_t b = histogram.bin(v);
                    const u64 w = weights.of(v);
                    atomicAdd(&s.counts[b], 1u);
                    atomicAdd(&s.sums[b], w);
                    if (static_cast<double>(w) >= least_sum) over += w;
                }
            });
            __syncthreads();
            weighty = block_sum(over, s);
            scan_bins(s, &all_count, &all);
            fresh = true;
        };
        fill();
        kept = all;
        if (k != 0 && k < all_count) {
            if (locate<kType>(row, a.vocab, histogram, all_count, all, Target{k, 0.0, false}, weights, s, &fresh)) kept = s.found_sum;
            __syncthreads();
        }
        if (has_p) {
            fill();
            if (locate<kType>(row, a.vocab, histogram, all_count, all, Target{0, static_cast<double>(p) * static_cast<double>(kept), false}, weights, s, &fresh)) kept = s.found_sum;
            __syncthreads();
        }
        if (has_least) kept = min(kept, weighty);
        kept = max(kept, one);
        fill();
        const bool last = u >= 1.0f;
        found = locate<kType>(row, a.vocab, histogram, all_count, all, Target{0, last ? static_cast<double>(kept) : static_cast<double>(u) * static_cast<double>(kept), !last}, weights, s, &fresh);
    }
    if (tid == 0) {
        const u64 rank = found ? s.found_rank : best;
        a.tokens[r] = static_cast<int>(static_cast<uint32_t>(rank));
        if (a.probabilities != nullptr) a.probabilities[r] = static_cast<float>(weights.fraction(value_at(rank)) * static_cast<double>(one) / static_cast<double>(kept));
    }
}

}  // namespace

size_t sample_workspace_bytes(const SampleArgs&, int) { return 0; }

hipError_t launch_sample(hipStream_t stream, const SampleArgs& a, void*, int) {
    if (a.type == 0) sample_kernel<0><<<a.rows, kThreads, 0, stream>>>(a);
    else if (a.type == 1) sample_kernel<1><<<a.rows, kThreads, 0, stream>>>(a);
    else sample_kernel<30><<<a.rows, kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace afhip
