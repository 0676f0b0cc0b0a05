// Attention of a batch's new tokens (drafted trees, chains, single tokens) over a paged key / value cache.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j - m),   over the keys j that t sees
//
// One pass over the keys with the running maximum m and sum of the softmax.  The rows of one key head are its query heads'
// tokens packed together (row = token * group + head in group), so a key is read once for all of them.
//
// The products are on the 16 x 16 x 32 matrix instructions with the keys as the first operand: the result of K Q^T has one
// row of the packed queries to a lane (column = lane % 16) and four consecutive keys in its registers, so maximum, sum and
// rescaling are a lane's own, but for one exchange between the four lanes of a row.  Its registers are the second operand of
// V^T P^T as they stand: the order of the 32 keys inside the instruction is free as long as V follows it (lane group g holds
// keys 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3).  V comes row-major and is needed column-major: it goes through LDS and
// is read with the transposing ds_read_b64_tr_b16.  K goes from memory into the operand registers, no LDS.
//
// A wavefront works alone on tiles of 32 keys (its own part of LDS, no barrier in the loop); the four wavefronts of a
// workgroup take tiles in turn and add up at the end.  Few rows on long contexts are split over workgroups as well, and a
// second kernel joins the parts.
#include "paged_launch.h"

#include <hip/hip_runtime.h>

namespace afhip {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kTile = 32;             // keys of one wavefront's step
constexpr uint32_t kNowhere = ~0u;    // of a key that has no place in the cache
constexpr float kLog2e = 1.4426950408889634f;
// A row's maximum follows its scores only when they pass it by more than 2^kSlack: the weights stay below 2^kSlack, far
// inside every type here, and most tiles leave the sums as they are.
constexpr float kSlack = 8.0f;

template <bool kBf16>
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    if (kBf16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool kBf16>
__device__ __forceinline__ short narrow(float v) {
    if (kBf16) return __builtin_bit_cast(short, static_cast<__bf16>(v));
    return __builtin_bit_cast(short, static_cast<_Float16>(v));
}
template <bool kBf16>
__device__ __forceinline__ float widen(short v) {
    if (kBf16) return static_cast<float>(__builtin_bit_cast(__bf16, v));
    return static_cast<float>(__builtin_bit_cast(_Float16, v));
}

// Largest of, or sum over, the four lanes that hold a row (lane % 16), in all of them: the value of the other half (32 lanes)
// and then of the other 16 lanes of a half, by the swapping register moves.
__device__ __forceinline__ void swap_halves(float* a, float* b) {
    const unsigned x = __builtin_bit_cast(unsigned, *a);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const unsigned first = r[0], second = r[1];  // (a bit_cast of r[1] itself reads r[0])
    *a = __builtin_bit_cast(float, first);
    *b = __builtin_bit_cast(float, second);
}
__device__ __forceinline__ void swap_rows(float* a, float* b) {
    const unsigned x = __builtin_bit_cast(unsigned, *a);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const unsigned first = r[0], second = r[1];
    *a = __builtin_bit_cast(float, first);
    *b = __builtin_bit_cast(float, second);
}
__device__ __forceinline__ float row_max(float v) {
    float other;
    swap_halves(&v, &other);
    v = fmaxf(v, other);
    swap_rows(&v, &other);
    return fmaxf(v, other);
}
__device__ __forceinline__ float row_sum(float v) {
    float other;
    swap_halves(&v, &other);
    v += other;
    swap_rows(&v, &other);
    return v + other;
}

__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& d) { return d.multiplier == 0 ? n : __umulhi(n, d.multiplier); }

// What a split of a request's keys holds for one row: the row's maximum (in units of log2) and the sum of its weights.
struct Part {
    float most, sum;
};

// exp2(a - b) where both may be minus infinity (nothing seen yet): then 1, of sums that are zero.
__device__ __forceinline__ float exp2_between(float a, float b) { return a == b ? 1.0f : __builtin_amdgcn_exp2f(a - b); }

// Which of the 32 keys from `first` on a row sees: bit j for key first + j.
__device__ __forceinline__ uint32_t seen_bits(int first, int context, int token, const unsigned long long* words, int count) {
    const int draft = first - context;  // the first key as a new token of the request
    if (words == nullptr) {
        const int left = token + 1 - draft;
        return left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
    }
    if (draft <= -32) return ~0u;
    if (draft < 0) {
        const uint32_t tree = count > 0 ? static_cast<uint32_t>(words[0] << -draft) : 0u;
        return tree | ((1u << -draft) - 1);
    }
    const int word = draft >> 6, shift = draft & 63;
    unsigned long long bits = word < count ? words[word] >> shift : 0ull;
    if (shift > 32 && word + 1 < count) bits |= words[word + 1] << (64 - shift);
    return static_cast<uint32_t>(bits);
}

// kDim: the head's values, rounded up to a size that is here (the rest are zeros that are not read).  kF32: query and out
// are f32.  kQ: sixteens of rows.
template <int kDim, bool kBf16, bool kF32, int kQ>
__global__ __launch_bounds__(kThreads) void tree_attention_kernel(TreeAttentionArgs a, uint32_t row_tiles, uint32_t splits,
                                                                 uint32_t split_keys, float* part_out, Part* parts) {
    constexpr int kSteps = kDim / 32;                            // products of K Q^T along the head
    constexpr int kTerms = kF32 ? (kBf16 ? 3 : 2) : 1;           // of a query value: 24 bits of three bf16, 22 of two f16
    constexpr int kParts = kTerms;                               // of a weight
    constexpr int kRows = 16 * kQ;
    constexpr int kRowBytes = kDim * 2 + 32;  // of V in LDS: four rows of a lane group and the four groups fall on other banks
    constexpr int kLoads = kTile * kDim / 8 / 64;                // 16-byte loads of V a lane
    constexpr int kChunks = kDim / 8;                            // 16-byte parts of a row
    extern __shared__ __attribute__((aligned(16))) char lds[];

    // the row tiles of a key head's split lie on one XCD (workgroups go round them in turn): they share its L2
    const uint32_t item = (blockIdx.x >> 3) / row_tiles * 8 + (blockIdx.x & 7), row_tile = (blockIdx.x >> 3) % row_tiles;
    if (item >= a.requests * a.cache.kv_heads * splits) return;
    const uint32_t request = item / (a.cache.kv_heads * splits), kv_head = item % a.cache.kv_heads;
    const uint32_t split = item / a.cache.kv_heads % splits;

    const int begin = min(max(a.query_starts[request], 0), static_cast<int>(a.tokens));
    const int end = min(max(a.query_starts[request + 1], begin), static_cast<int>(a.tokens));
    const int tokens = min(end - begin, static_cast<int>(a.max_query_len));
    const int group = static_cast<int>(a.group), rows = tokens * group, first_row = static_cast<int>(row_tile) * kRows;
    if (first_row >= rows) return;
    const int context = max(a.context_lens[request], 0);
    const unsigned long long most_keys = min(static_cast<unsigned long long>(a.table_columns) * a.block_size.by,
                                             static_cast<unsigned long long>(a.max_key_len));
    int keys = static_cast<int>(min(static_cast<unsigned long long>(context) + tokens, most_keys));
    const int last_token = min(first_row + kRows - 1, rows - 1) / group;
    if (a.masks == nullptr) keys = static_cast<int>(min(static_cast<unsigned long long>(keys), static_cast<unsigned long long>(context) + last_token + 1));
    const int key_begin = static_cast<int>(min(static_cast<unsigned long long>(split) * split_keys, static_cast<unsigned long long>(keys)));
    const int key_end = static_cast<int>(min(static_cast<unsigned long long>(key_begin) + split_keys, static_cast<unsigned long long>(keys)));

    const int tid = static_cast<int>(threadIdx.x), wave = tid >> 6, lane = tid & 63, column = lane & 15, quarter = lane >> 4;
    char* v_lds = lds + wave * (kTile * kRowBytes);
    const int* table = a.block_tables + static_cast<size_t>(request) * a.table_columns;
    const uint32_t head_at = kv_head * a.cache.head_stride;
    const int chunks = static_cast<int>(a.cache.head_dim / 8);  // that hold something

    // where a key's values lie, in 16-byte units
    auto place = [&](int key) -> uint32_t {
        if (key >= key_end) return kNowhere;
        const uint32_t col = divide(static_cast<uint32_t>(key), a.block_size);
        const uint32_t block = static_cast<uint32_t>(table[col]);
        if (block >= a.cache.blocks) return kNowhere;
        return block * a.cache.block_stride + (static_cast<uint32_t>(key) - col * a.block_size.by) * a.cache.slot_stride + head_at;
    };

    // ---- the rows
    s16x8 query[kQ][kSteps][kTerms];
    float unit[kQ];  // what a product of the row is multiplied by: scale, log2(e), and for f32 on f16 the row's power of two
    const unsigned long long* words[kQ];
    int row_token[kQ];
    bool real[kQ];
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        const int row = first_row + qt * 16 + column;
        real[qt] = row < rows;
        row_token[qt] = real[qt] ? row / group : 0;
        const int head = static_cast<int>(kv_head) * group + (real[qt] ? row % group : 0);
        const size_t token = static_cast<size_t>(begin + row_token[qt]);
        words[qt] = a.masks != nullptr ? a.masks + token * a.mask_words : nullptr;
        unit[qt] = a.scale * kLog2e;
        const size_t at = token * a.query_token_stride + static_cast<size_t>(head) * a.query_head_stride;
        if (kF32) {
            float v[kSteps][8];
            float most = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int chunk = s * 4 + quarter;
                const bool held = real[qt] && chunk < chunks;
                const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.query) + at) + 2 * chunk;
                const float4 x = held ? p[0] : float4{0, 0, 0, 0}, y = held ? p[1] : float4{0, 0, 0, 0};
                v[s][0] = x.x; v[s][1] = x.y; v[s][2] = x.z; v[s][3] = x.w;
                v[s][4] = y.x; v[s][5] = y.y; v[s][6] = y.z; v[s][7] = y.w;
#pragma unroll
                for (int j = 0; j < 8; ++j) most = fmaxf(most, __builtin_fabsf(v[s][j]));
            }
            if (!kBf16) {  // f16 has 5 exponent bits: the row's largest value goes to [0.5, 1)
                most = row_max(most);
                const bool moves = most > 0.0f && most < __builtin_inff();
                const int exponent = moves ? __builtin_amdgcn_frexp_expf(most) : 0;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[s][j] = __builtin_amdgcn_ldexpf(v[s][j], -exponent);
                }
                unit[qt] = __builtin_amdgcn_ldexpf(unit[qt], exponent);
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float rest = v[s][j];
#pragma unroll
                    for (int term = 0; term < kTerms; ++term) {
                        query[qt][s][term][j] = narrow<kBf16>(rest);
                        rest -= widen<kBf16>(query[qt][s][term][j]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int chunk = s * 4 + quarter;
                const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.query) + at) + chunk;
                const uint4 raw = real[qt] && chunk < chunks ? *p : uint4{0, 0, 0, 0};
                query[qt][s][0] = __builtin_bit_cast(s16x8, raw);
            }
        }
    }

    f32x4 out[kQ][kDim / 16];
    float most[kQ], sum[kQ];
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        most[qt] = -__builtin_inff();
        sum[qt] = 0.0f;
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) out[qt][d] = f32x4{0, 0, 0, 0};
    }

    // ---- the keys
    uint4 key_regs[2][kSteps], value_regs[kLoads];
    auto load = [&](uint32_t at) {  // `at`: lane l % 32 has the place of key l % 32
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t from = static_cast<uint32_t>(__shfl(static_cast<int>(at), half * 16 + column));
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int chunk = s * 4 + quarter;
                const uint4 zero{0, 0, 0, 0};
                key_regs[half][s] = from != kNowhere && chunk < chunks ? a.cache.keys[static_cast<size_t>(from) + chunk] : zero;
            }
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int slot = i * 64 + lane, chunk = slot % kChunks;
            const uint32_t from = static_cast<uint32_t>(__shfl(static_cast<int>(at), slot / kChunks));
            const uint4 zero{0, 0, 0, 0};
            value_regs[i] = from != kNowhere && chunk < chunks ? a.cache.values[static_cast<size_t>(from) + chunk] : zero;
        }
    };
    int tile = key_begin + wave * kTile;
    uint32_t at = place(tile + (lane & 31));
    load(at);
    uint32_t at_next = place(tile + kWaves * kTile + (lane & 31));
    for (; tile < key_end; tile += kWaves * kTile) {
        const uint32_t held = static_cast<uint32_t>(__ballot(at != kNowhere));  // keys of the tile that have a place
        const bool clean = tile + kTile <= context && held == ~0u;               // every row sees every key
        uint32_t odd = 0;  // keys with a value that is no finite number (looked for only where some row may not see them)
        if (!clean) {
            constexpr uint32_t kExponent = kBf16 ? 0x7F80u : 0x7C00u;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint32_t* w = reinterpret_cast<uint32_t*>(&value_regs[i]);
                bool found = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if ((w[j] & kExponent) == kExponent) {
                        found = true;
                        w[j] &= 0xFFFF0000u;
                    }
                    if ((w[j] >> 16 & kExponent) == kExponent) {
                        found = true;
                        w[j] &= 0x0000FFFFu;
                    }
                }
                unsigned long long which = __ballot(found);
                while (which != 0) {
                    const int l = __builtin_ctzll(which);
                    which &= which - 1;
                    odd |= 1u << ((i * 64 + l) / kChunks);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int slot = i * 64 + lane;
            *reinterpret_cast<uint4*>(v_lds + slot / kChunks * kRowBytes + slot % kChunks * 16) = value_regs[i];
        }
        f32x4 score[kQ][2];
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                score[qt][half] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; --term)  // the small terms first
                        score[qt][half] = mfma<kBf16>(__builtin_bit_cast(s16x8, key_regs[half][s]), query[qt][s][term], score[qt][half]);
                }
            }
        }
        const uint32_t at_now = at;
        at = at_next;
        if (tile + kWaves * kTile < key_end) {
            load(at);
            at_next = place(tile + 2 * kWaves * kTile + (lane & 31));
        }

        float peak[kQ];
        bool passes = false;
        uint32_t seen[kQ];
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
            seen[qt] = ~0u;
            if (!clean) seen[qt] = real[qt] ? seen_bits(tile, context, row_token[qt], words[qt], static_cast<int>(a.mask_words)) & held : 0u;
            peak[qt] = -__builtin_inff();
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x = score[qt][half][j] * unit[qt];
                    if (!clean && (seen[qt] >> (half * 16 + quarter * 4 + j) & 1) == 0) x = -__builtin_inff();
                    score[qt][half][j] = x;
                    peak[qt] = fmaxf(peak[qt], x);
                }
            }
            peak[qt] = row_max(peak[qt]);
            passes |= peak[qt] > most[qt] + kSlack;
        }
        if (__any(passes)) {
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
                const float next = peak[qt] > most[qt] + kSlack ? peak[qt] : most[qt];  // each row by itself: no other row's keys move its bits
                const float by = exp2_between(most[qt], next);
                most[qt] = next;
                sum[qt] *= by;
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) out[qt][d][j] *= by;
                }
            }
        }
        s16x8 weight[kQ][kParts];
        float weights[kQ][8];
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
            const float from = most[qt] == -__builtin_inff() ? 0.0f : most[qt];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = __builtin_amdgcn_exp2f(score[qt][j >> 2][j & 3] - from);
                weights[qt][j] = p;
                sum[qt] += p;
                float rest = p;
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                    weight[qt][part][j] = narrow<kBf16>(rest);
                    rest -= widen<kBf16>(weight[qt][part][j]);
                }
            }
        }
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) {
            s16x8 v;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = half * 16 + quarter * 4 + (column >> 2);
                const char* from = v_lds + row * kRowBytes + d * 32 + (column & 3) * 8;
                const s16x4 four = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)from);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[half * 4 + j] = four[j];
            }
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                for (int part = kParts - 1; part >= 0; --part) out[qt][d] = mfma<kBf16>(v, weight[qt][part], out[qt][d]);
            }
        }
        // A row that does not see a key must not get 0 * inf from it: the products above took such values as zeros, and the
        // rows that see them add them here, one by one.
        while (odd != 0) {
            const int key = __builtin_ctz(odd);
            odd &= odd - 1;
            const uint32_t from = static_cast<uint32_t>(__shfl(static_cast<int>(at_now), key));
            const int holder = key % 16 / 4, index = key / 16 * 4 + key % 4;
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
                float p = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float other = __shfl(weights[qt][j], holder * 16 + column);
                    if (j == index) p = other;
                }
                if ((seen[qt] >> key & 1) == 0) continue;
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int dim = d * 16 + quarter * 4 + j;
                        if (dim >= chunks * 8) continue;
                        const float v = widen<kBf16>(reinterpret_cast<const short*>(a.cache.values)[static_cast<size_t>(from) * 8 + dim]);
                        if (!(__builtin_fabsf(v) < __builtin_inff())) out[qt][d][j] = __builtin_fmaf(p, v, out[qt][d][j]);
                    }
                }
            }
        }
    }

    // ---- the four wavefronts' sums
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) sum[qt] = row_sum(sum[qt]);
    constexpr int kPitch = kDim + 4;                       // floats of a row in LDS
    float* sums = reinterpret_cast<float*>(lds);           // [2][kRows][kPitch]
    Part* wave_parts = reinterpret_cast<Part*>(sums + 2 * kRows * kPitch);  // [kWaves][kRows]
    __syncthreads();  // V is done with
    if (quarter == 0) {
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) wave_parts[wave * kRows + qt * 16 + column] = Part{most[qt], sum[qt]};
    }
    __syncthreads();
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        float all = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) all = fmaxf(all, wave_parts[w * kRows + qt * 16 + column].most);
        const float by = exp2_between(most[qt], all);
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
            for (int j = 0; j < 4; ++j) out[qt][d][j] *= by;
        }
    }
    auto cell = [&](int region, int qt, int d) {
        return reinterpret_cast<f32x4*>(sums + (region * kRows + qt * 16 + column) * kPitch + d * 16 + quarter * 4);
    };
#pragma unroll
    for (int round = 0; round < 2; ++round) {  // wavefronts 2 and 3 to 0 and 1, then 0 and 1 side by side
        if (round == 0 ? wave >= 2 : wave < 2) {
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) *cell(wave & 1, qt, d) = out[qt][d];
            }
        }
        __syncthreads();
        if (round == 0 && wave < 2) {
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) out[qt][d] += *cell(wave, qt, d);
            }
        }
        // (a wavefront writes only the region it alone has read: no barrier between)
    }

    // ---- out: four values a thread
    constexpr int kFours = kDim / 4;
    for (int i = tid; i < kRows * kFours; i += kThreads) {
        const int r = i / kFours, d = i % kFours * 4, row = first_row + r;
        if (row >= rows || d >= chunks * 8) continue;
        const f32x4 x = *reinterpret_cast<const f32x4*>(sums + r * kPitch + d) + *reinterpret_cast<const f32x4*>(sums + (kRows + r) * kPitch + d);
        float all = -__builtin_inff(), total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) all = fmaxf(all, wave_parts[w * kRows + r].most);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) total += wave_parts[w * kRows + r].sum * exp2_between(wave_parts[w * kRows + r].most, all);
        const size_t token = static_cast<size_t>(begin + row / group);
        const int head = static_cast<int>(kv_head) * group + row % group;
        if (splits > 1) {
            const size_t index = (static_cast<size_t>(split) * a.tokens + token) * a.heads + head;
            *reinterpret_cast<f32x4*>(part_out + index * a.cache.head_dim + d) = x;
            if (d == 0) parts[index] = Part{all, total};
        } else {
            const size_t to = token * a.out_token_stride + static_cast<size_t>(head) * a.out_head_stride + d;
            const float by = total == 0.0f ? 0.0f : 1.0f / total;
            if (kF32) {
                *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + to) = x * by;
            } else {
                s16x4 y;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = narrow<kBf16>(x[j] * by);
                *reinterpret_cast<s16x4*>(static_cast<uint16_t*>(a.out) + to) = y;
            }
        }
    }
}

// The parts of a row from `splits` workgroups, one wavefront a row: each part is brought to the common maximum.
template <bool kBf16, bool kF32>
__global__ __launch_bounds__(kThreads) void join_parts_kernel(TreeAttentionArgs a, uint32_t splits, const float* part_out, const Part* parts) {
    const uint32_t request = blockIdx.y, row = blockIdx.x * kWaves + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int begin = min(max(a.query_starts[request], 0), static_cast<int>(a.tokens));
    const int end = min(max(a.query_starts[request + 1], begin), static_cast<int>(a.tokens));
    const uint32_t tokens = min(static_cast<uint32_t>(end - begin), a.max_query_len);
    if (row >= tokens * a.heads) return;
    const size_t token = static_cast<size_t>(begin) + row / a.heads;
    const uint32_t head = row % a.heads;
    const size_t stride = static_cast<size_t>(a.tokens) * a.heads, index = token * a.heads + head;
    const Part mine = lane < static_cast<int>(splits) ? parts[index + lane * stride] : Part{-__builtin_inff(), 0.0f};
    float most = mine.most;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
    const float by = exp2_between(mine.most, most);
    float total = mine.sum * by;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
    const float over = total == 0.0f ? 0.0f : 1.0f / total;
    for (uint32_t d = lane * 4; d < a.cache.head_dim; d += 256) {
        f32x4 x{0, 0, 0, 0};
        for (uint32_t s = 0; s < splits; ++s) {
            // (by readlane: lanes past the head's end are not in this loop, and a shuffle would not read them)
            const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, by), s));
            const f32x4 y = *reinterpret_cast<const f32x4*>(part_out + (index + s * stride) * a.cache.head_dim + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(y[j], f, x[j]);
        }
        const size_t to = token * a.out_token_stride + static_cast<size_t>(head) * a.out_head_stride + d;
        if (kF32) {
            *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + to) = x * over;
        } else {
            s16x4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = narrow<kBf16>(x[j] * over);
            *reinterpret_cast<s16x4*>(static_cast<uint16_t*>(a.out) + to) = y;
        }
    }
}

struct Shape {
    int dim, sixteens;  // kDim, kQ
    uint32_t row_tiles, splits, split_keys;
};

constexpr uint32_t kMostSplits = 64;  // a lane of the joining wavefront each

Shape shape_of(const TreeAttentionArgs& a, int compute_units) {
    Shape s;
    s.dim = a.cache.head_dim <= 64 ? 64 : a.cache.head_dim <= 128 ? 128 : 256;
    const uint64_t rows = static_cast<uint64_t>(a.max_query_len) * a.group;
    // sixteens of rows as the queries' registers allow: three terms of f32 queries, or heads of 256, take two
    const int most = a.f32 || s.dim == 256 ? 2 : 4;
    s.sixteens = rows <= 16 ? 1 : rows <= 32 || most == 2 ? 2 : 4;
    s.row_tiles = static_cast<uint32_t>((rows + 16 * s.sixteens - 1) / (16 * s.sixteens));
    const uint64_t base = static_cast<uint64_t>(a.requests) * a.cache.kv_heads * s.row_tiles;
    const uint64_t wanted = base == 0 ? 1 : (4 * static_cast<uint64_t>(compute_units) + base - 1) / base;
    uint64_t splits = wanted < kMostSplits ? wanted : kMostSplits;
    const uint64_t least = 256;  // keys that are worth a workgroup
    if (splits > (a.max_key_len + least - 1) / least) splits = (a.max_key_len + least - 1) / least;
    if (splits == 0) splits = 1;
    const uint64_t step = kWaves * kTile;
    const uint64_t keys = ((a.max_key_len + splits - 1) / splits + step - 1) / step * step;
    s.split_keys = static_cast<uint32_t>(keys == 0 ? step : keys);
    s.splits = static_cast<uint32_t>((a.max_key_len + s.split_keys - 1) / s.split_keys);
    if (s.splits == 0) s.splits = 1;
    return s;
}

size_t part_out_bytes(const TreeAttentionArgs& a, const Shape& s) {
    return (static_cast<size_t>(s.splits) * a.tokens * a.heads * a.cache.head_dim * sizeof(float) + 255) / 256 * 256;
}

template <int kDim, bool kBf16, bool kF32, int kQ>
hipError_t attend(hipStream_t stream, const TreeAttentionArgs& a, const Shape& s, void* workspace) {
    static LdsLimit limit;
    const size_t v_bytes = static_cast<size_t>(kWaves) * kTile * (kDim * 2 + 32);
    const size_t sum_bytes = 2 * 16 * kQ * (kDim + 4) * sizeof(float) + kWaves * 16 * kQ * sizeof(Part);
    const size_t lds = v_bytes > sum_bytes ? v_bytes : sum_bytes;
    const auto kernel = tree_attention_kernel<kDim, kBf16, kF32, kQ>;
    hipError_t e = allow_lds(kernel, lds, &limit);
    if (e != hipSuccess) return e;
    float* part_out = static_cast<float*>(workspace);
    Part* parts = s.splits > 1 ? reinterpret_cast<Part*>(static_cast<char*>(workspace) + part_out_bytes(a, s)) : nullptr;
    const uint32_t items = a.requests * a.cache.kv_heads * s.splits;
    kernel<<<(items + 7) / 8 * 8 * s.row_tiles, kThreads, lds, stream>>>(a, s.row_tiles, s.splits, s.split_keys, part_out, parts);
    e = hipGetLastError();
    if (e != hipSuccess || s.splits == 1) return e;
    const dim3 grid(static_cast<uint32_t>((static_cast<uint64_t>(a.max_query_len) * a.heads + kWaves - 1) / kWaves), a.requests);
    join_parts_kernel<kBf16, kF32><<<grid, kThreads, 0, stream>>>(a, s.splits, part_out, parts);
    return hipGetLastError();
}

template <int kDim, bool kBf16, bool kF32>
hipError_t attend_rows(hipStream_t stream, const TreeAttentionArgs& a, const Shape& s, void* workspace) {
    if (s.sixteens == 1) return attend<kDim, kBf16, kF32, 1>(stream, a, s, workspace);
    if constexpr (!kF32 && kDim < 256) {
        if (s.sixteens == 4) return attend<kDim, kBf16, kF32, 4>(stream, a, s, workspace);
    }
    return attend<kDim, kBf16, kF32, 2>(stream, a, s, workspace);
}

template <int kDim>
hipError_t attend_types(hipStream_t stream, const TreeAttentionArgs& a, const Shape& s, void* workspace) {
    if (a.cache_bf16) return a.f32 ? attend_rows<kDim, true, true>(stream, a, s, workspace) : attend_rows<kDim, true, false>(stream, a, s, workspace);
    return a.f32 ? attend_rows<kDim, false, true>(stream, a, s, workspace) : attend_rows<kDim, false, false>(stream, a, s, workspace);
}

}  // namespace

size_t tree_attention_workspace_bytes(const TreeAttentionArgs& args, int compute_units) {
    const Shape s = shape_of(args, compute_units);
    return s.splits == 1 ? 0 : part_out_bytes(args, s) + static_cast<size_t>(s.splits) * args.tokens * args.heads * sizeof(Part);
}

hipError_t launch_tree_attention(hipStream_t stream, const TreeAttentionArgs& args, void* workspace, int compute_units) {
    const Shape s = shape_of(args, compute_units);
    if (s.dim == 64) return attend_types<64>(stream, args, s, workspace);
    if (s.dim == 128) return attend_types<128>(stream, args, s, workspace);
    return attend_types<256>(stream, args, s, workspace);
}

}  // namespace afhip
