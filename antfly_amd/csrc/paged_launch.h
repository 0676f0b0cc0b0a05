// Internal C++ interface between the paged-cache and attention kernels and the C ABI.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "lds_limit.h"
#include "qmatmul_launch.h"

namespace afhip {

// Strides in 16-byte units (8 values), which is what the kernels address in: 32 bits reach 64 GiB.
struct CacheView {
    uint4* keys;
    uint4* values;
    uint32_t blocks, block_size, kv_heads, head_dim;
    uint32_t block_stride, slot_stride, head_stride;
};

// n / d for a fixed d: n * ceil(2^32 / d) >> 32, exact while n * d < 2^32 (the product's error, n * (d - 1) at most, stays
// below 2^32).
struct Divisor {
    uint32_t by, multiplier, whole;  // whole: all bits where the divisor is 1, whose multiplier 2^32 does not fit
    Divisor() : Divisor(1) {}
    explicit Divisor(uint32_t d) : by(d), multiplier(d == 1 ? 0 : static_cast<uint32_t>(((uint64_t{1} << 32) + d - 1) / d)), whole(d == 1 ? ~0u : 0) {}
};

constexpr int kPlanTokens = 1024;       // most token places of one workgroup
constexpr int kPlanWalk = 1024;         // most tokens of a request that are walked to the tree's root
constexpr size_t kPlanRequests = 8192;  // their prefix sums are in every workgroup's LDS

struct BatchPlanArgs {
    uint32_t requests, table_columns, block_size, blocks, tokens, mask_words, free_count;
    const int *context_lens, *query_lens, *free_blocks, *parents;
    int *block_tables, *query_starts, *slots, *positions;
    unsigned long long* masks;
    int* blocks_taken;
    uint32_t group_tokens;  // token places of a workgroup (the launch sets it)
};
hipError_t launch_batch_plan(hipStream_t stream, const BatchPlanArgs& args);

constexpr uint32_t kCacheThreads = 256;  // of a workgroup of the store and the move
// A workgroup of the store takes eight values a thread: whole tokens while they fit it, a part of one token otherwise.
struct StoreGrid {
    uint32_t tokens_a_group, groups_a_token;
    StoreGrid(uint32_t chunks) : tokens_a_group(chunks < kCacheThreads ? kCacheThreads / chunks : 1), groups_a_token((chunks - 1) / kCacheThreads + 1) {}
    uint64_t groups(uint32_t tokens) const {
        return groups_a_token > 1 ? static_cast<uint64_t>(tokens) * groups_a_token : (static_cast<uint64_t>(tokens) + tokens_a_group - 1) / tokens_a_group;
    }
};

// type: 0 f32, 1 f16, 30 bf16 (the source's); to_bf16: the cache's.  Strides in elements.
hipError_t launch_cache_store(hipStream_t stream, const CacheView& cache, bool to_bf16, int type, const void* keys,
                              const void* values, size_t token_stride, size_t head_stride, const int* slots, uint32_t tokens);
hipError_t launch_cache_move(hipStream_t stream, const CacheView& cache, const int* block_tables, uint32_t table_columns,
                             const int* context_lens, const int* paths, const int* path_lens, uint32_t requests,
                             uint32_t path_columns);

struct TreeAttentionArgs {
    CacheView cache;
    Divisor block_size;
    const void* query;
    void* out;
    const int *query_starts, *context_lens, *block_tables;
    const unsigned long long* masks;
    size_t query_token_stride, query_head_stride, out_token_stride, out_head_stride;  // elements
    uint32_t requests, tokens, heads, group, max_query_len, max_key_len, table_columns, mask_words;
    float scale;
    bool cache_bf16, f32;  // f32: query and out; otherwise they are of the cache's type
};
size_t tree_attention_workspace_bytes(const TreeAttentionArgs& args, int compute_units);
bool tree_attention_fits_a_launch(const TreeAttentionArgs& args, int compute_units);
hipError_t launch_tree_attention(hipStream_t stream, const TreeAttentionArgs& args, void* workspace, int compute_units);

}  // namespace afhip
