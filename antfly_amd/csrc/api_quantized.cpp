// C ABI of a sampled serving step on an 8-bit paged cache: argument checks, then one to three launches.
#include <hip/hip_runtime_api.h>
#include <math.h>

#include "api_checks.h"
#include "api_internal.h"
#include "quantized_launch.h"

using namespace afhip;

namespace {

bool array_type(int type) { return type == AFHIP_TYPE_F32 || type == AFHIP_TYPE_F16 || type == AFHIP_TYPE_BF16; }
size_t size_of(int type) { return type == AFHIP_TYPE_F32 ? 4 : 2; }

afhip_status view_of(const afhip_quantized_cache& c, QuantizedView* view) {
    if (c.type != AFHIP_TYPE_I8 && c.type != AFHIP_TYPE_E4M3) return AFHIP_ERR_UNSUPPORTED_TENSOR_TYPE;
    size_t slots, codes, scales, scale_bytes;
    if (c.blocks == 0 || c.block_size == 0 || c.kv_heads == 0 || c.head_dim == 0 || !checked_mul(c.blocks, c.block_size, &slots) ||
        slots > kInt32Max || c.kv_heads > kInt32Max || c.head_dim > kInt32Max || c.head_dim % 16 != 0 || c.block_stride % 16 != 0 ||
        c.slot_stride % 16 != 0 || c.head_stride % 16 != 0)
        return AFHIP_ERR_INVALID_STATE;
    if (!span(c.blocks, c.block_stride, c.block_size, c.slot_stride, c.head_dim, &codes) || !add(&codes, c.kv_heads - 1, c.head_stride) ||
        codes >= (size_t{1} << 36) || c.block_stride / 16 > 0xffffffffu || c.slot_stride / 16 > 0xffffffffu || c.head_stride / 16 > 0xffffffffu)
        return AFHIP_ERR_INVALID_STATE;
    if (!span(c.blocks, c.scale_block_stride, c.block_size, c.scale_slot_stride, 1, &scales) || !add(&scales, c.kv_heads - 1, c.scale_head_stride) ||
        scales >= (size_t{1} << 32) || c.scale_block_stride > 0xffffffffu || c.scale_slot_stride > 0xffffffffu || c.scale_head_stride > 0xffffffffu)
        return AFHIP_ERR_INVALID_STATE;
    scale_bytes = scales * 4;
    if (codes > c.keys.len || codes > c.values.len || !aligned(c.keys, 16) || !aligned(c.values, 16) || scale_bytes > c.key_scales.len ||
        scale_bytes > c.value_scales.len || !aligned(c.key_scales, 4) || !aligned(c.value_scales, 4))
        return AFHIP_ERR_INVALID_STATE;
    if (c.head_dim > 256) return AFHIP_ERR_OP_UNSUPPORTED;
    *view = QuantizedView{reinterpret_cast<uint4*>(c.keys.ptr),
                          reinterpret_cast<uint4*>(c.values.ptr),
                          reinterpret_cast<float*>(c.key_scales.ptr),
                          reinterpret_cast<float*>(c.value_scales.ptr),
                          static_cast<uint32_t>(c.blocks),
                          static_cast<uint32_t>(c.block_size),
                          static_cast<uint32_t>(c.kv_heads),
                          static_cast<uint32_t>(c.head_dim),
                          static_cast<uint32_t>(c.block_stride / 16),
                          static_cast<uint32_t>(c.slot_stride / 16),
                          static_cast<uint32_t>(c.head_stride / 16),
                          static_cast<uint32_t>(c.scale_block_stride),
                          static_cast<uint32_t>(c.scale_slot_stride),
                          static_cast<uint32_t>(c.scale_head_stride),
                          c.type == AFHIP_TYPE_E4M3};
    return AFHIP_OK;
}

// Rows of heads of `type` that are read or written: strides in multiples of `unit` elements, the address of `alignment` bytes.
bool rows_fit(afhip_buffer b, int type, size_t tokens, size_t token_stride, size_t heads, size_t head_stride, size_t head_dim, size_t unit, size_t alignment) {
    size_t elements, bytes;
    return token_stride % unit == 0 && head_stride % unit == 0 && span(tokens, token_stride, heads, head_stride, head_dim, &elements) &&
           checked_mul(elements, size_of(type), &bytes) && bytes <= b.len && aligned(b, alignment);
}
HeadRows rows_of(afhip_buffer b, size_t token_stride, size_t head_stride) { return HeadRows{reinterpret_cast<void*>(b.ptr), token_stride, head_stride}; }

// The tokens of a store or a load against a cache's heads; AFHIP_OK with tokens == 0: nothing to do.
afhip_status token_rows(int type, afhip_buffer keys, afhip_buffer values, size_t token_stride, size_t head_stride, afhip_buffer slots, size_t tokens,
                        size_t kv_heads, size_t head_dim) {
    if (!array_type(type)) return AFHIP_ERR_UNSUPPORTED_TENSOR_TYPE;
    if (tokens == 0) return AFHIP_OK;
    const size_t unit = type == AFHIP_TYPE_F32 ? 4 : 8;
    if (tokens > kInt32Max || !rows_fit(keys, type, tokens, token_stride, kv_heads, head_stride, head_dim, unit, 16) ||
        !rows_fit(values, type, tokens, token_stride, kv_heads, head_stride, head_dim, unit, 16) || !holds(slots, tokens, 4))
        return AFHIP_ERR_INVALID_STATE;
    return AFHIP_OK;
}

// Checks a rotation and fills everything but the keys' target; *empty: there is nothing to do.
afhip_status rotation_args(const afhip_head_rotation* r, bool writes_keys, HeadsArgs* out, bool* empty) {
    if (r == nullptr) return AFHIP_ERR_INVALID_ARGUMENT;
    if (!array_type(r->type) || !array_type(r->out_type)) return AFHIP_ERR_UNSUPPORTED_TENSOR_TYPE;
    size_t places;
    if (r->tokens > kInt32Max || r->heads > kInt32Max || r->kv_heads == 0 || r->kv_heads > kInt32Max || r->head_dim == 0 || r->head_dim % 8 != 0 ||
        r->rotary_dim % 8 != 0 || r->rotary_dim > r->head_dim || r->axes == 0 || r->axes > 16 || !checked_mul(r->axes, r->tokens, &places) ||
        isnan(r->epsilon) || r->epsilon < 0.0f)
        return AFHIP_ERR_INVALID_STATE;
    if (r->head_dim > 256) return AFHIP_ERR_OP_UNSUPPORTED;
    for (size_t p = 0; p < r->rotary_dim / 2; ++p) {
        if (r->pair_axes[p] >= r->axes) return AFHIP_ERR_INVALID_STATE;
    }
    *empty = r->tokens == 0;
    if (*empty) return AFHIP_OK;
    const size_t in = r->type == AFHIP_TYPE_F32 ? 16 : 8, to = r->out_type == AFHIP_TYPE_F32 ? 16 : 8;
    if ((r->heads != 0 && (!rows_fit(r->query, r->type, r->tokens, r->query_token_stride, r->heads, r->query_head_stride, r->head_dim, 4, in) ||
                           !rows_fit(r->out_query, r->out_type, r->tokens, r->out_query_token_stride, r->heads, r->out_query_head_stride, r->head_dim, 4, to))) ||
        !rows_fit(r->key, r->type, r->tokens, r->key_token_stride, r->kv_heads, r->key_head_stride, r->head_dim, 4, in) ||
        (writes_keys && !rows_fit(r->out_key, r->out_type, r->tokens, r->out_key_token_stride, r->kv_heads, r->out_key_head_stride, r->head_dim, 4, to)) ||
        (r->rotary_dim != 0 && (!holds(r->positions, places, 4) || !holds(r->frequencies, r->rotary_dim / 2, 4))) ||
        (r->query_weight.ptr != 0 && !holds(r->query_weight, r->head_dim, 4)) || (r->key_weight.ptr != 0 && !holds(r->key_weight, r->head_dim, 4)))
        return AFHIP_ERR_INVALID_STATE;
    *out = HeadsArgs{};
    out->query = rows_of(r->query, r->query_token_stride, r->query_head_stride);
    out->key = rows_of(r->key, r->key_token_stride, r->key_head_stride);
    out->out_query = rows_of(r->out_query, r->out_query_token_stride, r->out_query_head_stride);
    out->out_key = rows_of(r->out_key, r->out_key_token_stride, r->out_key_head_stride);
    out->positions = r->rotary_dim != 0 ? reinterpret_cast<const int*>(r->positions.ptr) : nullptr;
    out->frequencies = reinterpret_cast<const float*>(r->frequencies.ptr);
    out->query_weight = reinterpret_cast<const float*>(r->query_weight.ptr);
    out->key_weight = reinterpret_cast<const float*>(r->key_weight.ptr);
    out->target = HeadTarget::arrays;
    out->out_type = r->out_type;
    out->tokens = static_cast<uint32_t>(r->tokens);
    out->heads = static_cast<uint32_t>(r->heads);
    out->kv_heads = static_cast<uint32_t>(r->kv_heads);
    out->head_dim = static_cast<uint32_t>(r->head_dim);
    out->rotary_dim = static_cast<uint32_t>(r->rotary_dim);
    out->epsilon = r->epsilon;
    out->interleaved = r->interleaved != 0;
    out->one_axis = true;
    for (size_t p = 0; p < 128; ++p) {
        out->pair_axes[p] = p < r->rotary_dim / 2 ? r->pair_axes[p] : 0;
        out->one_axis = out->one_axis && out->pair_axes[p] == 0;
    }
    return AFHIP_OK;
}

afhip_status run_heads(void* stream, int type, const HeadsArgs& args) {
    const uint64_t items = static_cast<uint64_t>(args.heads) + args.kv_heads + args.value_heads;
    if (items > kInt32Max || !heads_fit_a_launch(args.tokens, static_cast<uint32_t>(items), args.head_dim)) return AFHIP_ERR_OP_UNSUPPORTED;
    return status_of(launch_heads(static_cast<hipStream_t>(stream), type, args, gemv_compute_units()));
}

// Checks everything but the workspace; *empty: there is nothing to compute.
afhip_status attention_args(const afhip_quantized_attention* t, QuantizedAttentionArgs* out, bool* empty) {
    if (t == nullptr) return AFHIP_ERR_INVALID_ARGUMENT;
    QuantizedView cache;
    const afhip_status s = view_of(t->cache, &cache);
    if (s != AFHIP_OK) return s;
    if (!array_type(t->type)) return AFHIP_ERR_UNSUPPORTED_TENSOR_TYPE;
    if (t->heads == 0 || t->heads % t->cache.kv_heads != 0 || t->heads > kInt32Max || t->requests > kInt32Max || t->tokens > kInt32Max ||
        t->max_query_len > kInt32Max || t->max_key_len > kInt32Max || t->table_columns > kInt32Max || t->window > kInt32Max || isnan(t->softcap) ||
        t->softcap < 0.0f || isinf(t->softcap))
        return AFHIP_ERR_INVALID_STATE;
    size_t most, rows;
    // (a tile's keys are divided by the block size as far as 31 behind the last one)
    if (t->requests > 65535 || !checked_mul(t->max_key_len + 32, t->cache.block_size, &most) || most >= (size_t{1} << 32) ||
        !checked_mul(t->max_query_len, t->heads, &rows) || rows > kInt32Max)
        return AFHIP_ERR_OP_UNSUPPORTED;
    *empty = t->requests == 0 || t->tokens == 0 || t->max_query_len == 0;
    if (!*empty) {
        const size_t unit = t->type == AFHIP_TYPE_F32 ? 4 : 8;
        size_t entries;
        if (!rows_fit(t->query, t->type, t->tokens, t->query_token_stride, t->heads, t->query_head_stride, t->cache.head_dim, unit, 16) ||
            !rows_fit(t->out, t->type, t->tokens, t->out_token_stride, t->heads, t->out_head_stride, t->cache.head_dim, unit, 16) ||
            !checked_mul(t->requests, t->table_columns, &entries) || !holds(t->query_starts, t->requests + 1, 4) ||
            !holds(t->context_lens, t->requests, 4) || !holds(t->block_tables, entries, 4) || (t->slopes.ptr != 0 && !holds(t->slopes, t->heads, 4)))
            return AFHIP_ERR_INVALID_STATE;
    }
    *out = QuantizedAttentionArgs{cache,
                                  Divisor(cache.block_size),
                                  reinterpret_cast<const void*>(t->query.ptr),
                                  reinterpret_cast<void*>(t->out.ptr),
                                  reinterpret_cast<const int*>(t->query_starts.ptr),
                                  reinterpret_cast<const int*>(t->context_lens.ptr),
                                  reinterpret_cast<const int*>(t->block_tables.ptr),
                                  reinterpret_cast<const float*>(t->slopes.ptr),
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
                                  static_cast<uint32_t>(t->window),
                                  t->scale,
                                  t->softcap,
                                  t->type};
    return AFHIP_OK;
}

afhip_status sample_args(const afhip_sample* t, SampleArgs* out, bool* empty) {
    if (t == nullptr) return AFHIP_ERR_INVALID_ARGUMENT;
    if (!array_type(t->type)) return AFHIP_ERR_UNSUPPORTED_TENSOR_TYPE;
    if (t->vocab == 0) return AFHIP_ERR_INVALID_STATE;
    if (t->vocab > (size_t{1} << 24) || t->rows > 65535) return AFHIP_ERR_OP_UNSUPPORTED;
    *empty = t->rows == 0;
    if (!*empty) {
        size_t elements, bytes;
        if (!span(t->rows, t->row_stride, 1, 0, t->vocab, &elements) || !checked_mul(elements, size_of(t->type), &bytes) || bytes > t->logits.len ||
            !aligned(t->logits, size_of(t->type)) || !holds(t->uniforms, t->rows, 4) || !holds(t->tokens, t->rows, 4))
            return AFHIP_ERR_INVALID_STATE;
        for (const afhip_buffer b : {t->temperatures, t->top_k, t->top_p, t->min_p, t->probabilities}) {
            if (b.ptr != 0 && !holds(b, t->rows, 4)) return AFHIP_ERR_INVALID_STATE;
        }
    }
    *out = SampleArgs{reinterpret_cast<const void*>(t->logits.ptr),
                      t->row_stride,
                      reinterpret_cast<const float*>(t->temperatures.ptr),
                      reinterpret_cast<const float*>(t->top_p.ptr),
                      reinterpret_cast<const float*>(t->min_p.ptr),
                      reinterpret_cast<const float*>(t->uniforms.ptr),
                      reinterpret_cast<const int*>(t->top_k.ptr),
                      reinterpret_cast<int*>(t->tokens.ptr),
                      reinterpret_cast<float*>(t->probabilities.ptr),
                      static_cast<uint32_t>(t->rows),
                      static_cast<uint32_t>(t->vocab),
                      t->type};
    return AFHIP_OK;
}

}  // namespace

extern "C" {

afhip_status afhip_launch_quantized_store(void* stream, const afhip_quantized_cache* cache, int type, afhip_buffer keys, afhip_buffer values,
                                          size_t token_stride, size_t head_stride, afhip_buffer slots, size_t tokens) {
    if (cache == nullptr) return AFHIP_ERR_INVALID_ARGUMENT;
    HeadsArgs args{};
    afhip_status s = view_of(*cache, &args.quantized);
    if (s == AFHIP_OK) s = token_rows(type, keys, values, token_stride, head_stride, slots, tokens, cache->kv_heads, cache->head_dim);
    if (s != AFHIP_OK || tokens == 0) return s;
    args.key = rows_of(keys, token_stride, head_stride);
    args.value = rows_of(values, token_stride, head_stride);
    args.slots = reinterpret_cast<const int*>(slots.ptr);
    args.target = args.quantized.e4m3 ? HeadTarget::e4m3_cache : HeadTarget::i8_cache;
    args.tokens = static_cast<uint32_t>(tokens);
    args.kv_heads = args.value_heads = args.quantized.kv_heads;
    args.head_dim = args.quantized.head_dim;
    return run_heads(stream, type, args);
}

afhip_status afhip_launch_quantized_load(void* stream, const afhip_quantized_cache* cache, int type, afhip_buffer keys, afhip_buffer values,
                                         size_t token_stride, size_t head_stride, afhip_buffer slots, size_t tokens) {
    if (cache == nullptr) return AFHIP_ERR_INVALID_ARGUMENT;
    QuantizedView view;
    afhip_status s = view_of(*cache, &view);
    if (s == AFHIP_OK) s = token_rows(type, keys, values, token_stride, head_stride, slots, tokens, cache->kv_heads, cache->head_dim);
    if (s != AFHIP_OK || tokens == 0) return s;
    size_t groups;
    const size_t lanes = view.head_dim <= 64 ? 8 : view.head_dim <= 128 ? 16 : 32, each = 256 / lanes;
    if (!checked_mul(tokens, 2 * cache->kv_heads, &groups) || groups > 0xffffffffu || !fits_a_launch((groups + each - 1) / each, 256)) return AFHIP_ERR_OP_UNSUPPORTED;
    return status_of(launch_quantized_load(static_cast<hipStream_t>(stream), view, type, rows_of(keys, token_stride, head_stride),
                                           rows_of(values, token_stride, head_stride), reinterpret_cast<const int*>(slots.ptr), static_cast<uint32_t>(tokens), gemv_compute_units()));
}

afhip_status afhip_launch_head_rotation(void* stream, const afhip_head_rotation* rotation) {
    HeadsArgs args;
    bool empty = true;
    const afhip_status s = rotation_args(rotation, true, &args, &empty);
    if (s != AFHIP_OK || empty) return s;
    return run_heads(stream, rotation->type, args);
}

afhip_status afhip_launch_rotated_store(void* stream, const afhip_head_rotation* rotation, const afhip_paged_cache* cache,
                                        const afhip_quantized_cache* quantized, afhip_buffer values, size_t token_stride, size_t head_stride,
                                        afhip_buffer slots) {
    if ((cache == nullptr) == (quantized == nullptr)) return AFHIP_ERR_INVALID_ARGUMENT;
    CacheView view{};
    QuantizedView codes{};
    afhip_status s = cache != nullptr ? view_of(*cache, &view) : view_of(*quantized, &codes);
    if (s != AFHIP_OK) return s;
    HeadsArgs args;
    bool empty = true;
    s = rotation_args(rotation, false, &args, &empty);
    if (s != AFHIP_OK) return s;
    if (rotation->kv_heads != (cache != nullptr ? view.kv_heads : codes.kv_heads) || rotation->head_dim != (cache != nullptr ? view.head_dim : codes.head_dim))
        return AFHIP_ERR_INVALID_STATE;
    if (empty) return AFHIP_OK;
    if (!rows_fit(values, rotation->type, rotation->tokens, token_stride, rotation->kv_heads, head_stride, rotation->head_dim, 4,
                  rotation->type == AFHIP_TYPE_F32 ? 16 : 8) ||
        !holds(slots, rotation->tokens, 4))
        return AFHIP_ERR_INVALID_STATE;
    args.value = rows_of(values, token_stride, head_stride);
    args.value_heads = args.kv_heads;
    args.slots = reinterpret_cast<const int*>(slots.ptr);
    args.cache = view;
    args.quantized = codes;
    args.target = cache != nullptr ? (cache->type == AFHIP_TYPE_BF16 ? HeadTarget::bf16_cache : HeadTarget::f16_cache)
                                   : (codes.e4m3 ? HeadTarget::e4m3_cache : HeadTarget::i8_cache);
    return run_heads(stream, rotation->type, args);
}

size_t afhip_quantized_attention_workspace_bytes(const afhip_quantized_attention* attention) {
    QuantizedAttentionArgs args{};
    bool empty = true;
    if (attention_args(attention, &args, &empty) != AFHIP_OK || empty) return 0;
    return quantized_attention_workspace_bytes(args, gemv_compute_units());
}

afhip_status afhip_launch_quantized_attention(void* stream, const afhip_quantized_attention* attention, afhip_buffer workspace) {
    QuantizedAttentionArgs args{};
    bool empty = true;
    const afhip_status s = attention_args(attention, &args, &empty);
    if (s != AFHIP_OK || empty) return s;
    const int units = gemv_compute_units();
    if (!quantized_attention_fits_a_launch(args, units)) return AFHIP_ERR_OP_UNSUPPORTED;
    const size_t needed = quantized_attention_workspace_bytes(args, units);
    if (needed > workspace.len || (needed != 0 && !aligned(workspace, 256))) return AFHIP_ERR_INVALID_STATE;
    return status_of(launch_quantized_attention(static_cast<hipStream_t>(stream), args, reinterpret_cast<void*>(workspace.ptr), units));
}

size_t afhip_sample_workspace_bytes(const afhip_sample* sample) {
    SampleArgs args{};
    bool empty = true;
    if (sample_args(sample, &args, &empty) != AFHIP_OK || empty) return 0;
    return sample_workspace_bytes(args, gemv_compute_units());
}

afhip_status afhip_launch_sample(void* stream, const afhip_sample* sample, afhip_buffer workspace) {
    SampleArgs args{};
    bool empty = true;
    const afhip_status s = sample_args(sample, &args, &empty);
    if (s != AFHIP_OK || empty) return s;
    const int units = gemv_compute_units();
    const size_t needed = sample_workspace_bytes(args, units);
    if (needed > workspace.len || (needed != 0 && !aligned(workspace, 256))) return AFHIP_ERR_INVALID_STATE;
    return status_of(launch_sample(static_cast<hipStream_t>(stream), args, reinterpret_cast<void*>(workspace.ptr), units));
}

}  // extern "C"
