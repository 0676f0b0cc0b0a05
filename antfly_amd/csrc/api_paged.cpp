// C ABI of the paged key / value cache and the attention over it: argument checks, then one or two launches.
#include <hip/hip_runtime_api.h>

#include "api_checks.h"
#include "api_internal.h"
#include "paged_launch.h"

using namespace afhip;

namespace {

// Checks everything but the workspace; *empty: there is nothing to compute.
afhip_status attention_args(const afhip_tree_attention* t, TreeAttentionArgs* out, bool* empty) {
    if (t == nullptr) return AFHIP_ERR_INVALID_ARGUMENT;
    CacheView cache;
    const afhip_status s = view_of(t->cache, &cache);
    if (s != AFHIP_OK) return s;
    const bool f32 = t->type == AFHIP_TYPE_F32;
    if (!f32 && t->type != t->cache.type) return AFHIP_ERR_UNSUPPORTED_TENSOR_TYPE;
    if (t->heads == 0 || t->heads % t->cache.kv_heads != 0 || t->heads > kInt32Max || t->requests > kInt32Max || t->tokens > kInt32Max ||
        t->max_query_len > kInt32Max || t->max_key_len > kInt32Max || t->table_columns > kInt32Max)
        return AFHIP_ERR_INVALID_STATE;
    size_t most, rows;
    if (t->cache.head_dim > 256 || t->mask_words > 16 || t->requests > 65535 ||
        !checked_mul(t->max_key_len, t->cache.block_size, &most) || most >= (size_t{1} << 32) ||
        !checked_mul(t->max_query_len, t->heads, &rows) || rows > kInt32Max)
        return AFHIP_ERR_OP_UNSUPPORTED;
    *empty = t->requests == 0 || t->tokens == 0 || t->max_query_len == 0;
    if (!*empty) {
        const size_t unit = f32 ? 4 : 8, size = f32 ? 4 : 2;
        size_t q, o, entries;
        if (t->query_token_stride % unit != 0 || t->query_head_stride % unit != 0 || t->out_token_stride % unit != 0 ||
            t->out_head_stride % unit != 0 ||
            !span(t->tokens, t->query_token_stride, t->heads, t->query_head_stride, t->cache.head_dim, &q) ||
            !span(t->tokens, t->out_token_stride, t->heads, t->out_head_stride, t->cache.head_dim, &o) ||
            !checked_mul(t->requests, t->table_columns, &entries))
            return AFHIP_ERR_INVALID_STATE;
        size_t masks = 0;
        if (!checked_mul(q, size, &q) || !checked_mul(o, size, &o) || q > t->query.len || o > t->out.len || !aligned(t->query, 16) ||
            !aligned(t->out, 16) || !holds(t->query_starts, t->requests + 1, 4) || !holds(t->context_lens, t->requests, 4) ||
            !holds(t->block_tables, entries, 4) || !checked_mul(t->tokens, t->mask_words, &masks) ||
            (t->masks.ptr != 0 && !holds(t->masks, masks, 8)))
            return AFHIP_ERR_INVALID_STATE;
    }
    *out = TreeAttentionArgs{cache,
                             Divisor(cache.block_size),
                             reinterpret_cast<const void*>(t->query.ptr),
                             reinterpret_cast<void*>(t->out.ptr),
                             reinterpret_cast<const int*>(t->query_starts.ptr),
                             reinterpret_cast<const int*>(t->context_lens.ptr),
                             reinterpret_cast<const int*>(t->block_tables.ptr),
                             reinterpret_cast<const unsigned long long*>(t->masks.ptr),
                             t->query_token_stride,
                             t->query_head_stride,
                             t->out_token_stride,
                             t->out_head_stride,
                             static_cast<uint32_t>(t->requests),
                             static_cast<uint32_t>(t->tokens),
                             static_cast<uint32_t>(t->heads),
                             static_cast<uint32_t>(t->heads / t->cache.kv_heads),
                             static_cast<uint32_t>(t->max_query_len),
                             static_cast<uint32_t>(t->max_key_len),
                             static_cast<uint32_t>(t->table_columns),
                             static_cast<uint32_t>(t->mask_words),
                             t->scale,
                             t->cache.type == AFHIP_TYPE_BF16,
                             f32};
    return AFHIP_OK;
}

}  // namespace

extern "C" {

afhip_status afhip_launch_batch_plan(void* stream, const afhip_batch_plan* p) {
    if (p == nullptr) return AFHIP_ERR_INVALID_ARGUMENT;
    if (p->block_size == 0 || p->block_size > kInt32Max || p->table_columns > kInt32Max || p->tokens > kInt32Max - kPlanTokens ||
        p->blocks > kInt32Max)
        return AFHIP_ERR_INVALID_STATE;
    if (p->requests > kPlanRequests || p->mask_words > 16) return AFHIP_ERR_OP_UNSUPPORTED;
    size_t entries, masks;
    if (!checked_mul(p->requests, p->table_columns, &entries) || !checked_mul(p->tokens, p->mask_words, &masks) ||
        !holds(p->context_lens, p->requests, 4) || !holds(p->query_lens, p->requests, 4) || !holds(p->block_tables, entries, 4) ||
        !holds(p->query_starts, p->requests + 1, 4) || !holds(p->slots, p->tokens, 4) || !holds(p->positions, p->tokens, 4) ||
        !holds(p->blocks_taken, 1, 4) || (p->parents.ptr != 0 && !holds(p->parents, p->tokens, 4)) ||
        (p->masks.ptr != 0 && !holds(p->masks, masks, 8)) || (p->free_blocks.len >= 4 && !aligned(p->free_blocks, 4)))
        return AFHIP_ERR_INVALID_STATE;
    const size_t free_count = p->free_blocks.len / 4;
    BatchPlanArgs a{};
    a.requests = static_cast<uint32_t>(p->requests);
    a.table_columns = static_cast<uint32_t>(p->table_columns);
    a.block_size = static_cast<uint32_t>(p->block_size);
    a.blocks = static_cast<uint32_t>(p->blocks);
    a.tokens = static_cast<uint32_t>(p->tokens);
    a.mask_words = static_cast<uint32_t>(p->mask_words);
    a.free_count = static_cast<uint32_t>(free_count < kInt32Max ? free_count : kInt32Max);
    a.context_lens = reinterpret_cast<const int*>(p->context_lens.ptr);
    a.query_lens = reinterpret_cast<const int*>(p->query_lens.ptr);
    a.free_blocks = reinterpret_cast<const int*>(p->free_blocks.ptr);
    a.parents = p->tokens != 0 ? reinterpret_cast<const int*>(p->parents.ptr) : nullptr;
    a.block_tables = reinterpret_cast<int*>(p->block_tables.ptr);
    a.query_starts = reinterpret_cast<int*>(p->query_starts.ptr);
    a.slots = reinterpret_cast<int*>(p->slots.ptr);
    a.positions = reinterpret_cast<int*>(p->positions.ptr);
    a.masks = masks != 0 ? reinterpret_cast<unsigned long long*>(p->masks.ptr) : nullptr;
    a.blocks_taken = reinterpret_cast<int*>(p->blocks_taken.ptr);
    return status_of(launch_batch_plan(static_cast<hipStream_t>(stream), a));
}

afhip_status afhip_launch_cache_store(void* stream, const afhip_paged_cache* cache, int type, afhip_buffer keys, afhip_buffer values,
                                      size_t token_stride, size_t head_stride, afhip_buffer slots, size_t tokens) {
    if (cache == nullptr) return AFHIP_ERR_INVALID_ARGUMENT;
    CacheView view;
    const afhip_status s = view_of(*cache, &view);
    if (s != AFHIP_OK) return s;
    if (type != AFHIP_TYPE_F32 && type != AFHIP_TYPE_F16 && type != AFHIP_TYPE_BF16) return AFHIP_ERR_UNSUPPORTED_TENSOR_TYPE;
    if (tokens == 0) return AFHIP_OK;
    const size_t unit = type == AFHIP_TYPE_F32 ? 4 : 8, size = type == AFHIP_TYPE_F32 ? 4 : 2;
    size_t elements, bytes, chunks;
    if (tokens > kInt32Max || token_stride % unit != 0 || head_stride % unit != 0 ||
        !span(tokens, token_stride, cache->kv_heads, head_stride, cache->head_dim, &elements) || !checked_mul(elements, size, &bytes) ||
        bytes > keys.len || bytes > values.len || !aligned(keys, 16) || !aligned(values, 16) || !holds(slots, tokens, 4))
        return AFHIP_ERR_INVALID_STATE;
    if (!checked_mul(cache->kv_heads, cache->head_dim / 8, &chunks) || chunks > kInt32Max ||
        !fits_a_launch(StoreGrid(static_cast<uint32_t>(chunks)).groups(static_cast<uint32_t>(tokens)), kCacheThreads))
        return AFHIP_ERR_OP_UNSUPPORTED;
    return status_of(launch_cache_store(static_cast<hipStream_t>(stream), view, cache->type == AFHIP_TYPE_BF16, type,
                                        reinterpret_cast<const void*>(keys.ptr), reinterpret_cast<const void*>(values.ptr), token_stride,
                                        head_stride, reinterpret_cast<const int*>(slots.ptr), static_cast<uint32_t>(tokens)));
}

afhip_status afhip_launch_cache_move(void* stream, const afhip_paged_cache* cache, afhip_buffer block_tables, size_t table_columns,
                                     afhip_buffer context_lens, afhip_buffer paths, afhip_buffer path_lens, size_t requests,
                                     size_t path_columns) {
    if (cache == nullptr) return AFHIP_ERR_INVALID_ARGUMENT;
    CacheView view;
    const afhip_status s = view_of(*cache, &view);
    if (s != AFHIP_OK) return s;
    if (requests == 0 || path_columns == 0) return AFHIP_OK;
    size_t entries, steps, chunks;
    if (requests > kInt32Max || table_columns > kInt32Max || path_columns > kInt32Max || !checked_mul(requests, table_columns, &entries) ||
        !checked_mul(requests, path_columns, &steps) || !holds(block_tables, entries, 4) || !holds(context_lens, requests, 4) ||
        !holds(paths, steps, 4) || !holds(path_lens, requests, 4))
        return AFHIP_ERR_INVALID_STATE;
    if (!checked_mul(cache->kv_heads, cache->head_dim / 8, &chunks) || chunks > 65535 * 128 || !fits_a_launch(requests, kCacheThreads))
        return AFHIP_ERR_OP_UNSUPPORTED;
    return status_of(launch_cache_move(static_cast<hipStream_t>(stream), view, reinterpret_cast<const int*>(block_tables.ptr),
                                       static_cast<uint32_t>(table_columns), reinterpret_cast<const int*>(context_lens.ptr),
                                       reinterpret_cast<const int*>(paths.ptr), reinterpret_cast<const int*>(path_lens.ptr),
                                       static_cast<uint32_t>(requests), static_cast<uint32_t>(path_columns)));
}

size_t afhip_tree_attention_workspace_bytes(const afhip_tree_attention* attention) {
    TreeAttentionArgs args{};
    bool empty = true;
    if (attention_args(attention, &args, &empty) != AFHIP_OK || empty) return 0;
    return tree_attention_workspace_bytes(args, gemv_compute_units());
}

afhip_status afhip_launch_tree_attention(void* stream, const afhip_tree_attention* attention, afhip_buffer workspace) {
    TreeAttentionArgs args{};
    bool empty = true;
    const afhip_status s = attention_args(attention, &args, &empty);
    if (s != AFHIP_OK || empty) return s;
    const int units = gemv_compute_units();
    if (!tree_attention_fits_a_launch(args, units)) return AFHIP_ERR_OP_UNSUPPORTED;
    const size_t needed = tree_attention_workspace_bytes(args, units);
    if (needed > workspace.len || (needed != 0 && !aligned(workspace, 256))) return AFHIP_ERR_INVALID_STATE;
    return status_of(launch_tree_attention(static_cast<hipStream_t>(stream), args, reinterpret_cast<void*>(workspace.ptr), units));
}

}  // extern "C"
