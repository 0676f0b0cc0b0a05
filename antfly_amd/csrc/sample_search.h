// Where the histogram of a row of logits passes a target.  Of the device this needs threadIdx and __syncthreads alone, so that a host
// that defines them can run it thread by thread.
#pragma once

#include <stdint.h>

namespace afhip {

constexpr int kSampleThreads = 512;
constexpr uint32_t kSampleBins = 1024;

// What passes: the count, or the sum, up to and with a token.  Sums are compared as the whole numbers that they are: the last token of a
// long one can weigh less than its 53rd bit.
struct Target {
    uint32_t count;          // at least so many tokens, where not zero
    unsigned long long sum;  // otherwise at least this sum
    __device__ __forceinline__ bool passed(uint32_t c, unsigned long long m) const { return count != 0 ? c >= count : m >= sum; }
};

// The bin in which the target is passed (kSampleBins: none), behind the counts and sums of those before it.
template <typename Shared>
__device__ __forceinline__ uint32_t find_bin(const Target& target, uint32_t count0, unsigned long long sum0, uint32_t all_count, unsigned long long all_sum, Shared& s) {
    if (threadIdx.x == 0) s.found_bin = kSampleBins;
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < kSampleBins; b += kSampleThreads) {
        const uint32_t c = s.counts[b], next_c = b + 1 < kSampleBins ? s.counts[b + 1] : all_count;
        const unsigned long long m = s.sums[b], next_m = b + 1 < kSampleBins ? s.sums[b + 1] : all_sum;
        const bool holds = target.count != 0 ? next_c > c : next_m > m, is_first = target.count != 0 ? c == 0 : m == 0;  // (counts may be left out)
        if (holds && target.passed(count0 + next_c, sum0 + next_m) && (is_first || !target.passed(count0 + c, sum0 + m))) s.found_bin = b;
    }
    __syncthreads();
    const uint32_t bin = s.found_bin;
    __syncthreads();  // every thread has it before a next search clears the place
    return bin;
}

}  // namespace afhip
