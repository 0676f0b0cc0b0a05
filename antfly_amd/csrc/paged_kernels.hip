// The paged key / value cache: the plan of a batch from its requests' lengths, the store of new tokens, the move of an
// accepted path.  Whole numbers and copies: nothing here is bound by arithmetic.
#include "paged_launch.h"

#include <hip/hip_runtime.h>

namespace afhip {

namespace {

constexpr int kThreads = kCacheThreads;

__device__ __forceinline__ int at_least_zero(int v) { return v > 0 ? v : 0; }

// ---- plan -------------------------------------------------------------------------------------------------------------
//
// With q[r] new tokens and n[r] = ceil((c[r] + q[r]) / B) - ceil(c[r] / B) new blocks of request r, everything follows from
// the two prefix sums  start[r] = sum of q before r,  fresh[r] = sum of n before r:  token i belongs to the last r with
// start[r] <= i, sits at position c[r] + i - start[r], and block b of its row is the table's entry while b < ceil(c[r] / B)
// and free_blocks[fresh[r] + b - ceil(c[r] / B)] beyond.  Both sums are 12 bytes a request with the lengths beside them, so
// every workgroup makes them again in its own LDS instead of a second launch reading them; a token finds its request by
// bisection there.  The token that opens a new block writes the table's entry, and no other token reads it.
// Ancestors: a token follows its parents to the root, in LDS, setting a bit for each (a parent has the smaller index, so the
// words are finished from high to low and the walk ends).
// A few bytes a token: bound by the round trips to memory, one after the other (lengths, then table or free list).  8 requests with
// trees of up to 24 drafts 4 us; 512 requests and 260000 tokens 6 us.
__global__ __launch_bounds__(kThreads) void batch_plan_kernel(BatchPlanArgs a) {
    extern __shared__ int lds[];
    const int requests = static_cast<int>(a.requests);
    int* start = lds;                       // [requests + 1]
    int* fresh = start + requests + 1;      // [requests + 1]
    int* context = fresh + requests + 1;    // [requests]
    int* sums = context + requests;         // [2][4]: the wavefronts' totals
    int* parent = sums + 8;                 // [kPlanWalk + group_tokens], with parents

    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const unsigned base = blockIdx.x * a.group_tokens;
    const unsigned window = base > kPlanWalk ? base - kPlanWalk : 0;
    if (a.parents != nullptr) {
        for (unsigned i = window + tid; i < base + a.group_tokens && i < a.tokens; i += kThreads) parent[i - window] = a.parents[i];
    }
    for (int r = tid; r < requests; r += kThreads) {
        context[r] = at_least_zero(a.context_lens[r]);
        start[r] = at_least_zero(a.query_lens[r]);
    }
    __syncthreads();
    // a run of requests a thread, an odd number: the threads' runs fall on different banks
    const int run = ((requests + kThreads - 1) / kThreads) | 1, first = tid * run;
    int queries = 0, blocks = 0;
    for (int r = first; r < first + run && r < requests; ++r) {
        const int c = context[r], q = start[r];
        const unsigned owned = (static_cast<unsigned>(c) + a.block_size - 1) / a.block_size;
        const unsigned needed = (static_cast<unsigned>(c) + static_cast<unsigned>(q) + a.block_size - 1) / a.block_size;
        start[r] = queries;
        fresh[r] = blocks;
        queries += q;
        blocks += static_cast<int>(needed - owned);
    }
    int q_before = queries, b_before = blocks;  // inclusive sums over the wavefront's lanes
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int q = __shfl_up(q_before, d), b = __shfl_up(b_before, d);
        if (lane >= d) {
            q_before += q;
            b_before += b;
        }
    }
    if (lane == 63) {
        sums[wave] = q_before;
        sums[4 + wave] = b_before;
    }
    __syncthreads();
    q_before -= queries;
    b_before -= blocks;
    for (int w = 0; w < wave; ++w) {
        q_before += sums[w];
        b_before += sums[4 + w];
    }
    for (int r = first; r < first + run && r < requests; ++r) {
        start[r] += q_before;
        fresh[r] += b_before;
    }
    if (tid == 0) {
        start[requests] = sums[0] + sums[1] + sums[2] + sums[3];
        fresh[requests] = sums[4] + sums[5] + sums[6] + sums[7];
    }
    __syncthreads();
    const int total = start[requests];
    if (blockIdx.x == 0) {
        for (int r = tid; r <= requests; r += kThreads) a.query_starts[r] = start[r];
        if (tid == 0) a.blocks_taken[0] = fresh[requests];
    }
    const int words = static_cast<int>(a.mask_words);
    const int walked = a.masks != nullptr ? words * 64 : kPlanWalk;
    for (unsigned i = base + tid; i < base + a.group_tokens && i < a.tokens; i += kThreads) {
        unsigned long long* mask = a.masks != nullptr ? a.masks + static_cast<size_t>(i) * words : nullptr;
        if (static_cast<int>(i) >= total) {
            a.slots[i] = -1;
            a.positions[i] = -1;
            for (int w = 0; mask != nullptr && w < words; ++w) mask[w] = 0;
            continue;
        }
        int low = 0, high = requests - 1;  // the last request that starts at or before i
        while (low < high) {
            const int mid = (low + high + 1) >> 1;
            if (start[mid] <= static_cast<int>(i)) low = mid;
            else high = mid - 1;
        }
        const int t = static_cast<int>(i) - start[low], c = context[low];
        const unsigned position = static_cast<unsigned>(c) + static_cast<unsigned>(t);
        const unsigned column = position / a.block_size, owned = (static_cast<unsigned>(c) + a.block_size - 1) / a.block_size;
        int block = -1;
        if (column < a.table_columns) {
            int* entry = a.block_tables + static_cast<size_t>(low) * a.table_columns + column;
            if (column < owned) {
                block = *entry;
            } else {
                const unsigned from = static_cast<unsigned>(fresh[low]) + (column - owned);
                if (from < a.free_count) block = a.free_blocks[from];
                if (position % a.block_size == 0) *entry = block;
            }
        }
        const unsigned long long slot = static_cast<unsigned long long>(static_cast<unsigned>(block)) * a.block_size + position % a.block_size;
        a.slots[i] = static_cast<unsigned>(block) < a.blocks && slot < 0x80000000ull ? static_cast<int>(slot) : -1;

        int depth = t;
        if (a.parents != nullptr) {
            depth = 0;
            if (t < walked) {
                int at = t, word = t >> 6;
                unsigned long long bits = 1ull << (t & 63);
                for (int w = word + 1; mask != nullptr && w < words; ++w) mask[w] = 0;
                const int* tree = parent + (static_cast<int>(i - window) - t);  // token 0 of the request
                for (;;) {
                    const int up = tree[at];
                    if (up < 0 || up >= at) break;
                    ++depth;
                    if ((up >> 6) != word) {
                        if (mask != nullptr) {
                            mask[word] = bits;
                            for (int w = word - 1; w > (up >> 6); --w) mask[w] = 0;
                        }
                        word = up >> 6;
                        bits = 0;
                    }
                    bits |= 1ull << (up & 63);
                    at = up;
                }
                if (mask != nullptr) {
                    mask[word] = bits;
                    for (int w = word - 1; w >= 0; --w) mask[w] = 0;
                }
            } else if (mask != nullptr) {
                for (int w = 0; w < words; ++w) mask[w] = 0;
            }
        } else if (mask != nullptr) {
            for (int w = 0; w < words; ++w) {
                const int left = t + 1 - w * 64;  // bits of this word
                mask[w] = t >= walked || left <= 0 ? 0ull : left >= 64 ? ~0ull : (1ull << left) - 1;
            }
        }
        a.positions[i] = c + depth;
    }
}

// ---- store ------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const _Float16 x = static_cast<_Float16>(a), y = static_cast<_Float16>(b);  // v_cvt_f16_f32 rounds to nearest even
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, x)) | (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, y)) << 16);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __bf16 x = static_cast<__bf16>(a), y = static_cast<__bf16>(b);
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, x)) | (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, y)) << 16);
}

template <bool kToBf16>
__device__ __forceinline__ uint4 pack8(const float* v) {
    uint4 r;
    r.x = kToBf16 ? pack_bf16(v[0], v[1]) : pack_f16(v[0], v[1]);
    r.y = kToBf16 ? pack_bf16(v[2], v[3]) : pack_f16(v[2], v[3]);
    r.z = kToBf16 ? pack_bf16(v[4], v[5]) : pack_f16(v[4], v[5]);
    r.w = kToBf16 ? pack_bf16(v[6], v[7]) : pack_f16(v[6], v[7]);
    return r;
}

// Eight values of the source's type kType (0 f32, 1 f16, 30 bf16) in the cache's.
template <int kType, bool kToBf16>
__device__ __forceinline__ uint4 load8(const void* base, size_t element) {
    if (kType == 0) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + element);
        const float4 x = p[0], y = p[1];
        const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        return pack8<kToBf16>(v);
    }
    const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + element);
    if ((kType == 30) == kToBf16) return raw;
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint16_t h = static_cast<uint16_t>(words[i / 2] >> (16 * (i & 1)));
        v[i] = kType == 30 ? __builtin_bit_cast(float, static_cast<uint32_t>(h) << 16) : static_cast<float>(__builtin_bit_cast(_Float16, h));
    }
    return pack8<kToBf16>(v);
}

// A thread moves eight values of a key and of a value: 32 + 32 bytes of f32 in, 16 + 16 out.  Bound by those bytes: 7500 tokens of
// 8 heads of 128 (92 MB) 16.5 us, 5.6 TB/s, what a copy reaches.
template <int kType, bool kToBf16>
__global__ __launch_bounds__(kThreads) void cache_store_kernel(CacheView cache, const void* keys, const void* values, size_t token_stride,
                                                              size_t head_stride, const int* slots, uint32_t tokens,
                                                              uint32_t chunks_a_head, uint32_t chunks, uint32_t tokens_a_group,
                                                              uint32_t groups_a_token) {
    uint32_t token, chunk;
    if (groups_a_token > 1) {
        token = blockIdx.x / groups_a_token;
        chunk = (blockIdx.x % groups_a_token) * kThreads + threadIdx.x;
    } else {
        token = blockIdx.x * tokens_a_group + threadIdx.x / chunks;
        chunk = threadIdx.x % chunks;
        if (threadIdx.x >= tokens_a_group * chunks) return;
    }
    if (token >= tokens || chunk >= chunks) return;
    const uint32_t slot = static_cast<uint32_t>(slots[token]);
    const uint32_t block = slot / cache.block_size;
    if (block >= cache.blocks) return;
    const uint32_t head = chunk / chunks_a_head, part = chunk % chunks_a_head;
    const size_t from = static_cast<size_t>(token) * token_stride + static_cast<size_t>(head) * head_stride + part * 8;
    const size_t to = static_cast<size_t>(block) * cache.block_stride + static_cast<size_t>(slot % cache.block_size) * cache.slot_stride +
                      static_cast<size_t>(head) * cache.head_stride + part;
    const uint4 k = load8<kType, kToBf16>(keys, from), v = load8<kType, kToBf16>(values, from);
    cache.keys[to] = k;
    cache.values[to] = v;
}

// ---- move -------------------------------------------------------------------------------------------------------------
//
// A thread owns 16 bytes of every token (a part of one head's key or value), so the order of a path's steps is its own
// program order.  Step i reads place path[i] >= i and the steps before it wrote places below i: no step reads what an
// earlier one wrote, and kSteps of them are loaded before the first is stored.  Bound by three round trips to memory (path,
// table, token): 8 requests with paths of up to 5 tokens 5.5 us.
constexpr int kSteps = 8;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__global__ __launch_bounds__(kThreads) void cache_move_kernel(CacheView cache, const int* block_tables, uint32_t table_columns,
                                                             const int* context_lens, const int* paths, const int* path_lens,
                                                             uint32_t path_columns, uint32_t chunks_a_head, uint32_t chunks) {
    const uint32_t r = blockIdx.x, at = blockIdx.y * kThreads + threadIdx.x;
    if (at >= 2 * chunks) return;
    uint4* store = at < chunks ? cache.keys : cache.values;
    const uint32_t chunk = at < chunks ? at : at - chunks;
    const size_t inside = static_cast<size_t>(chunk / chunks_a_head) * cache.head_stride + chunk % chunks_a_head;
    const int* path = paths + static_cast<size_t>(r) * path_columns;
    const int* table = block_tables + static_cast<size_t>(r) * table_columns;
    const uint32_t count = min(static_cast<uint32_t>(at_least_zero(path_lens[r])), path_columns);
    const uint32_t context = static_cast<uint32_t>(at_least_zero(context_lens[r]));
    constexpr size_t kNone = ~size_t{0};
    auto place = [&](uint32_t position) -> size_t {
        const uint32_t column = position / cache.block_size;
        const uint32_t block = column < table_columns ? static_cast<uint32_t>(table[column]) : ~0u;
        if (block >= cache.blocks) return kNone;
        return static_cast<size_t>(block) * cache.block_stride + static_cast<size_t>(position % cache.block_size) * cache.slot_stride + inside;
    };
    for (uint32_t i0 = 0; i0 < count; i0 += kSteps) {
        int step[kSteps];
        size_t from[kSteps], to[kSteps];
        u32x4 held[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) step[s] = i0 + s < count ? path[i0 + s] : -1;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            from[s] = step[s] >= 0 ? place(context + static_cast<uint32_t>(step[s])) : kNone;
            to[s] = step[s] >= 0 ? place(context + i0 + s) : kNone;
            if (to[s] == kNone) from[s] = kNone;
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (from[s] != kNone) held[s] = *reinterpret_cast<const u32x4*>(store + from[s]);
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (from[s] != kNone) *reinterpret_cast<u32x4*>(store + to[s]) = held[s];
        }
    }
}

template <int kType, bool kToBf16>
hipError_t store(hipStream_t stream, const CacheView& cache, const void* keys, const void* values, size_t token_stride,
                 size_t head_stride, const int* slots, uint32_t tokens) {
    const uint32_t chunks_a_head = cache.head_dim / 8, chunks = cache.kv_heads * chunks_a_head;
    const StoreGrid grid(chunks);
    cache_store_kernel<kType, kToBf16><<<static_cast<uint32_t>(grid.groups(tokens)), kThreads, 0, stream>>>(
        cache, keys, values, token_stride, head_stride, slots, tokens, chunks_a_head, chunks, grid.tokens_a_group, grid.groups_a_token);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_batch_plan(hipStream_t stream, const BatchPlanArgs& args) {
    static LdsLimit limit;
    // A thread has one token, whose round trips follow one another; four where the lengths' sums, made by every workgroup, would take
    // longer: 512 requests of 512 tokens 6.5 us with one and 7.9 with four, 2048 of 100 8.4 and 10.1, 8192 of one 13.8 and 17.4; 8192
    // of 16 25.8 and 18.0, 4096 of 100 24.4 and 13.9.
    BatchPlanArgs a = args;
    a.group_tokens = static_cast<uint64_t>(args.requests) * args.tokens > (1u << 29) ? kPlanTokens : kThreads;
    size_t lds = (3 * static_cast<size_t>(args.requests) + 2 + 8) * sizeof(int);
    if (args.parents != nullptr) lds += (kPlanWalk + a.group_tokens) * sizeof(int);
    const hipError_t e = allow_lds(batch_plan_kernel, lds, &limit);
    if (e != hipSuccess) return e;
    const uint32_t grid = args.tokens == 0 ? 1 : (args.tokens + a.group_tokens - 1) / a.group_tokens;
    batch_plan_kernel<<<grid, kThreads, lds, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_cache_store(hipStream_t stream, const CacheView& cache, bool to_bf16, int type, const void* keys,
                              const void* values, size_t token_stride, size_t head_stride, const int* slots, uint32_t tokens) {
    if (type == 0) {
        return to_bf16 ? store<0, true>(stream, cache, keys, values, token_stride, head_stride, slots, tokens)
                       : store<0, false>(stream, cache, keys, values, token_stride, head_stride, slots, tokens);
    }
    if (type == 1) {
        return to_bf16 ? store<1, true>(stream, cache, keys, values, token_stride, head_stride, slots, tokens)
                       : store<1, false>(stream, cache, keys, values, token_stride, head_stride, slots, tokens);
    }
    return to_bf16 ? store<30, true>(stream, cache, keys, values, token_stride, head_stride, slots, tokens)
                   : store<30, false>(stream, cache, keys, values, token_stride, head_stride, slots, tokens);
}

hipError_t launch_cache_move(hipStream_t stream, const CacheView& cache, const int* block_tables, uint32_t table_columns,
                             const int* context_lens, const int* paths, const int* path_lens, uint32_t requests,
                             uint32_t path_columns) {
    const uint32_t chunks_a_head = cache.head_dim / 8, chunks = cache.kv_heads * chunks_a_head;
    const dim3 grid(requests, (2 * chunks + kThreads - 1) / kThreads);
    cache_move_kernel<<<grid, kThreads, 0, stream>>>(cache, block_tables, table_columns, context_lens, paths, path_lens, path_columns,
                                                    chunks_a_head, chunks);
    return hipGetLastError();
}

}  // namespace afhip
