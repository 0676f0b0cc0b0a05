// Internal C++ interface between the kernels of a sampled serving step on an 8-bit paged cache and the C ABI.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "paged_launch.h"

namespace afhip {

// Codes are addressed in 16-byte units (32 bits reach 64 GiB), scales in elements.
struct QuantizedView {
    uint4 *keys, *values;
    float *key_scales, *value_scales;
    uint32_t blocks, block_size, kv_heads, head_dim;
    uint32_t block_stride, slot_stride, head_stride;
    uint32_t scale_block_stride, scale_slot_stride, scale_head_stride;
    bool e4m3;
};

// [tokens][heads][head_dim], strides in elements
struct HeadRows {
    void* data;
    size_t token_stride, head_stride;
};

enum class HeadTarget : int { arrays, f16_cache, bf16_cache, i8_cache, e4m3_cache };

// What one launch does to the heads of a projection: queries and keys normed and rotated, keys and values written.
struct HeadsArgs {
    HeadRows query, key, value, out_query, out_key;
    CacheView cache;          // of the 16-bit targets
    QuantizedView quantized;  // of the 8-bit ones
    const int *slots, *positions;
    const float *frequencies, *query_weight, *key_weight;
    HeadTarget target;  // of the keys, and of the values with them
    int out_type;       // of the arrays
    uint32_t tokens, heads, kv_heads, value_heads, head_dim, rotary_dim;  // value_heads: 0 or kv_heads
    float epsilon;
    bool interleaved, one_axis;  // one_axis: all pairs turn with the first positions
    uint32_t groups_a_token, tokens_a_group, chunk;  // the launch sets these
    uint8_t pair_axes[128];
};
bool heads_fit_a_launch(uint32_t tokens, uint32_t heads, uint32_t head_dim);
// type: 0 f32, 1 f16, 30 bf16, of everything that is read
hipError_t launch_heads(hipStream_t stream, int type, const HeadsArgs& args, int compute_units);

hipError_t launch_quantized_load(hipStream_t stream, const QuantizedView& cache, int type, const HeadRows& keys, const HeadRows& values,
                                 const int* slots, uint32_t tokens, int compute_units);

struct QuantizedAttentionArgs {
    QuantizedView cache;
    Divisor block_size;
    const void* query;
    void* out;
    const int *query_starts, *context_lens, *block_tables;
    const float* slopes;
    size_t query_token_stride, query_head_stride, out_token_stride, out_head_stride;  // elements
    uint32_t requests, tokens, heads, group, max_query_len, max_key_len, table_columns, window;
    float scale, softcap;
    int type;
};
size_t quantized_attention_workspace_bytes(const QuantizedAttentionArgs& args, int compute_units);
bool quantized_attention_fits_a_launch(const QuantizedAttentionArgs& args, int compute_units);
hipError_t launch_quantized_attention(hipStream_t stream, const QuantizedAttentionArgs& args, void* workspace, int compute_units);

struct SampleArgs {
    const void* logits;
    size_t row_stride;
    const float *temperatures, *top_p, *min_p, *uniforms;
    const int* top_k;
    int* tokens;
    float* probabilities;
    uint32_t rows, vocab;
    int type;
};
size_t sample_workspace_bytes(const SampleArgs& args, int compute_units);
hipError_t launch_sample(hipStream_t stream, const SampleArgs& args, void* workspace, int compute_units);

}  // namespace afhip
