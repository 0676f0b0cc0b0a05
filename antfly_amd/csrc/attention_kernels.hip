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
// Keys and values of a tile of 32 keys come from memory straight into LDS (no registers in between), the next tile's while
// this one is worked on.  A workgroup's four wavefronts are kKeyGroups groups that take tiles in turn; the wavefronts of one
// group share its tiles and have 16 kQ rows each.  Few rows: four groups that need no barrier in the loop and add up at the
// end; many rows: one group, every key read once for 128 rows.  Few rows on long contexts are split over workgroups as well,
// and a second kernel joins the parts.
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

// Whether one of the two values of a register is no finite number.
template <bool kBf16>
__device__ __forceinline__ bool is_odd(uint32_t w) {
    constexpr uint32_t kExponent = kBf16 ? 0x7F80u : 0x7C00u;
    return (w & kExponent) == kExponent || (w >> 16 & kExponent) == kExponent;
}
template <bool kBf16>
__device__ __forceinline__ bool is_odd(short v) {
    constexpr short kExponent = kBf16 ? 0x7F80 : 0x7C00;
    return (v & kExponent) == kExponent;
}

__device__ const uint4 kNothing{0, 0, 0, 0};  // what keys without a place and values past a head's end are loaded from

// 16 bytes a lane from memory to 1 KiB of LDS from `to` on (a uniform address).
__device__ __forceinline__ void load_to_lds(uint32_t to, const uint4* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}

// Where 16-byte piece `piece` of row `row` of a tile lies in LDS, in pieces.  The pieces of a row are in an order of its own,
// so that the same piece of 16 rows (what the lanes of an operand read) falls on all banks: 256 bytes of them.
template <int kDim>
__device__ __forceinline__ int lds_piece(int row, int piece) {
    constexpr int kPieces = kDim / 8;
    return row * kPieces + (kPieces == 8 ? piece ^ (row >> 1 & 7) : piece ^ (row & 15));
}

template <int kDim, int kQ, int kKeyGroups>
constexpr size_t attention_lds_bytes() {
    constexpr int kRows = 16 * kQ * (kWaves / kKeyGroups);
    constexpr size_t tiles = static_cast<size_t>(kKeyGroups) * 2 * 2 * kTile * kDim * 2;
    constexpr size_t sums = kKeyGroups == 1 ? 0 : static_cast<size_t>(kKeyGroups) * kRows * ((kDim + 4) * sizeof(float) + sizeof(Part));
    return tiles > sums ? tiles : sums;
}

// kDim: the head's values, rounded up to a size that is here (the rest are zeros).  kF32: query and out are f32.
template <int kDim, bool kBf16, bool kF32, int kQ, int kKeyGroups>
__global__ __launch_bounds__(kThreads, kF32 ? 1 : 2) void tree_attention_kernel(TreeAttentionArgs a, uint32_t row_tiles, uint32_t splits,
                                                                 uint32_t split_keys, float* part_out, Part* parts) {
    constexpr int kSteps = kDim / 32;                            // products of K Q^T along the head
    constexpr int kTerms = kF32 ? (kBf16 ? 3 : 2) : 1;           // of a query value or a weight: 24 bits of three bf16, 22 of two f16
    constexpr int kRowGroups = kWaves / kKeyGroups, kRows = 16 * kQ * kRowGroups;
    constexpr int kPieces = kDim / 8;                            // 16-byte pieces of a row
    constexpr int kTileBytes = kTile * kDim * 2;                 // of K, and of V behind it
    constexpr int kLoads = kTile * kPieces / 64 / kRowGroups;    // of a wavefront, 1 KiB each, for K and for V
    extern __shared__ __attribute__((aligned(1024))) char lds[];

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

    const int tid = static_cast<int>(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int column = lane & 15, quarter = lane >> 4;
    const int key_group = wave / kRowGroups, row_group = wave % kRowGroups;
    char* const tiles = lds + key_group * (4 * kTileBytes);
    const uint32_t tiles_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)tiles));
    const int* table = a.block_tables + static_cast<size_t>(request) * a.table_columns;
    const uint32_t head_at = kv_head * a.cache.head_stride;
    const int pieces = static_cast<int>(a.cache.head_dim / 8);  // that hold something

    // where a key's values lie, in 16-byte units
    auto place = [&](int key) -> uint32_t {
        if (key >= key_end) return kNowhere;
        const uint32_t col = divide(static_cast<uint32_t>(key), a.block_size);
        const uint32_t block = static_cast<uint32_t>(table[col]);
        if (block >= a.cache.blocks) return kNowhere;
        return block * a.cache.block_stride + (static_cast<uint32_t>(key) - col * a.block_size.by) * a.cache.slot_stride + head_at;
    };
    // this wavefront's part of a tile's K and V; `at`: lane l % 32 has the place of key l % 32
    auto request_tile = [&](uint32_t at, int stage) {
        const uint32_t to = tiles_at + stage * (2 * kTileBytes) + row_group * (kLoads * 1024);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int slot = (row_group * kLoads + i) * 64 + lane, row = slot / kPieces, piece = lds_piece<kDim>(row, slot % kPieces) % kPieces;
            const uint32_t from = static_cast<uint32_t>(__shfl(static_cast<int>(at), row));
            const bool there = from != kNowhere && piece < pieces;
            load_to_lds(to + i * 1024, there ? a.cache.keys + from + piece : &kNothing);
            load_to_lds(to + kTileBytes + i * 1024, there ? a.cache.values + from + piece : &kNothing);
        }
    };
    const int step = kKeyGroups * kTile, first_tile = key_begin + key_group * kTile;
    uint32_t at = place(first_tile + (lane & 31));
    request_tile(at, 0);
    uint32_t at_next = place(first_tile + step + (lane & 31));

    // ---- the rows
    s16x8 query[kQ][kSteps][kTerms];
    float unit[kQ];  // what a product of the row is multiplied by: |scale|, log2(e), and for f32 on f16 the row's power of two
    const unsigned long long* words[kQ];
    int row_token[kQ];
    bool real[kQ];
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;  // a negative scale turns the queries round
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        const int row = first_row + (row_group * kQ + qt) * 16 + column;
        real[qt] = row < rows;
        row_token[qt] = real[qt] ? row / group : 0;
        const int head = static_cast<int>(kv_head) * group + (real[qt] ? row % group : 0);
        const size_t token = static_cast<size_t>(begin + row_token[qt]);
        words[qt] = a.masks != nullptr ? a.masks + token * a.mask_words : nullptr;
        unit[qt] = fmaxf(__builtin_fabsf(a.scale) * kLog2e, 1e-30f);  // (never 0, which would make minus infinity no number)
        const size_t from = token * a.query_token_stride + static_cast<size_t>(head) * a.query_head_stride;
        if (kF32) {
            float v[kSteps][8];
            float most = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int piece = s * 4 + quarter;
                const bool held = real[qt] && piece < pieces;
                const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.query) + from) + 2 * piece;
                const float4 x = held ? p[0] : float4{0, 0, 0, 0}, y = held ? p[1] : float4{0, 0, 0, 0};
                v[s][0] = x.x; v[s][1] = x.y; v[s][2] = x.z; v[s][3] = x.w;
                v[s][4] = y.x; v[s][5] = y.y; v[s][6] = y.z; v[s][7] = y.w;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (flip != 0) v[s][j] = -v[s][j];
                    most = fmaxf(most, __builtin_fabsf(v[s][j]));
                }
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
                const int piece = s * 4 + quarter;
                const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.query) + from) + piece;
                uint4 raw = real[qt] && piece < pieces ? *p : uint4{0, 0, 0, 0};
                raw = uint4{raw.x ^ flip, raw.y ^ flip, raw.z ^ flip, raw.w ^ flip};
                query[qt][s][0] = __builtin_bit_cast(s16x8, raw);
            }
        }
    }

    f32x4 out[kQ][kDim / 16];
    float most[kQ], sum[kQ];  // the largest product so far (before `unit`), and this lane's part of the weights' sum
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        most[qt] = -__builtin_inff();
        sum[qt] = 0.0f;
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) out[qt][d] = f32x4{0, 0, 0, 0};
    }

    // ---- the keys
    int stage = 0;
    for (int first = key_begin; first < key_end; first += step, stage ^= 1) {
        const int tile = first + key_group * kTile;
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // this wavefront's part of the tile is there
        if (kRowGroups > 1) __syncthreads();                // everyone's is, and the other stage has been read
        const uint32_t at_now = at;
        at = at_next;
        if (tile + step < key_end) {
            request_tile(at, stage ^ 1);
            at_next = place(tile + 2 * step + (lane & 31));
        }
        if (tile >= key_end) continue;
        const char* k_lds = tiles + stage * (2 * kTileBytes);
        char* v_lds = tiles + stage * (2 * kTileBytes) + kTileBytes;

        const uint32_t held = static_cast<uint32_t>(__ballot(at_now != kNowhere));  // keys of the tile that have a place
        const bool clean = tile + kTile <= context && held == ~0u;                   // every row sees every key

        f32x4 score[kQ][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const s16x8 k = *reinterpret_cast<const s16x8*>(k_lds + lds_piece<kDim>(half * 16 + column, s * 4 + quarter) * 16);
#pragma unroll
                for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; --term)  // the small terms first
                        score[qt][half] = mfma<kBf16>(k, query[qt][s][term], s == 0 && term == kTerms - 1 ? f32x4{0, 0, 0, 0} : score[qt][half]);
                }
            }
        }
        uint32_t odd = 0;  // keys with a value that is no finite number (looked for only where some row may not see them)
        uint32_t seen[kQ];
        if (!clean) {
            for (int slot = lane; slot < kTile * kPieces; slot += 64) {
                const uint4 v = *reinterpret_cast<const uint4*>(v_lds + slot * 16);
                unsigned long long which = __ballot(is_odd<kBf16>(v.x) || is_odd<kBf16>(v.y) || is_odd<kBf16>(v.z) || is_odd<kBf16>(v.w));
                while (which != 0) {
                    const int l = __builtin_ctzll(which);
                    which &= which - 1;
                    odd |= 1u << __builtin_amdgcn_readlane(slot / kPieces, l);
                }
            }
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
                seen[qt] = real[qt] ? seen_bits(tile, context, row_token[qt], words[qt], static_cast<int>(a.mask_words)) & held : 0u;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if ((seen[qt] >> (half * 16 + quarter * 4 + j) & 1) == 0) score[qt][half][j] = -__builtin_inff();
                    }
                }
            }
        }
        float peak[kQ];
        bool passes = false;
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
            const f32x4 x = score[qt][0], y = score[qt][1];
            peak[qt] = row_max(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]))));
            passes |= (peak[qt] - most[qt]) * unit[qt] > kSlack;
        }
        if (__any(passes)) {
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
                // each row by itself: no other row's keys move its bits
                const float next = (peak[qt] - most[qt]) * unit[qt] > kSlack ? peak[qt] : most[qt];
                const float by = most[qt] == next ? 1.0f : __builtin_amdgcn_exp2f((most[qt] - next) * unit[qt]);
                most[qt] = next;
                sum[qt] *= by;
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) out[qt][d][j] *= by;
                }
            }
        }
        s16x8 weight[kQ][kTerms];
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
            const float from = most[qt] == -__builtin_inff() ? 0.0f : -most[qt] * unit[qt];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(score[qt][j >> 2][j & 3], unit[qt], from));
                sum[qt] += p;
                float rest = p;
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    weight[qt][term][j] = narrow<kBf16>(rest);
                    if (term + 1 < kTerms) rest -= widen<kBf16>(weight[qt][term][j]);
                }
            }
        }
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) {
            s16x8 v;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = half * 16 + quarter * 4 + (column >> 2);
                const char* from = v_lds + lds_piece<kDim>(row, d * 2 + (column >> 1 & 1)) * 16 + (column & 1) * 8;
                const s16x4 four = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)from);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[half * 4 + j] = four[j];
            }
            if (odd != 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = is_odd<kBf16>(static_cast<short>(v[j])) ? static_cast<short>(0) : v[j];
            }
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                for (int term = kTerms - 1; term >= 0; --term) out[qt][d] = mfma<kBf16>(v, weight[qt][term], out[qt][d]);
            }
        }
        // A row that does not see a key must not get 0 * inf from it: the products above took such values as zeros, and the
        // rows that see them add them here, key by key.
        while (odd != 0) {
            const int key = __builtin_ctz(odd);
            odd &= odd - 1;
            const int holder = key % 16 / 4, index = key / 16 * 4 + key % 4;
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
                float p = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float other = __shfl(widen<kBf16>(weight[qt][0][j]), holder * 16 + column);
                    if (j == index) p = other;
                }
                if ((seen[qt] >> key & 1) == 0) continue;
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
                    const char* from = v_lds + lds_piece<kDim>(key, d * 2 + (quarter >> 1)) * 16 + (quarter & 1) * 8;
                    const s16x4 four = *reinterpret_cast<const s16x4*>(from);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (is_odd<kBf16>(static_cast<short>(four[j]))) out[qt][d][j] = __builtin_fmaf(p, widen<kBf16>(four[j]), out[qt][d][j]);
                    }
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // (of a workgroup without keys: its first request)

    // ---- the key groups' sums, and out: four values a lane
    float all[kQ];  // the row's maximum in units of log2
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        sum[qt] = row_sum(sum[qt]);
        all[qt] = most[qt] == -__builtin_inff() ? most[qt] : most[qt] * unit[qt];
    }
    auto put = [&](int row, int d, f32x4 x, float highest, float total) {
        if (row >= rows || d >= pieces * 8) return;
        const size_t token = static_cast<size_t>(begin + row / group);
        const int head = static_cast<int>(kv_head) * group + row % group;
        if (splits > 1) {
            const size_t index = (static_cast<size_t>(split) * a.tokens + token) * a.heads + head;
            *reinterpret_cast<f32x4*>(part_out + index * a.cache.head_dim + d) = x;
            if (d == 0) parts[index] = Part{highest, total};
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
    };
    if (kKeyGroups == 1) {
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d)
                put(first_row + (row_group * kQ + qt) * 16 + column, d * 16 + quarter * 4, out[qt][d], all[qt], sum[qt]);
        }
        return;
    }
    constexpr int kPitch = kDim + 4;                                                   // floats of a row in LDS
    float* sums = reinterpret_cast<float*>(lds);                                       // [kKeyGroups][kRows][kPitch]
    Part* group_parts = reinterpret_cast<Part*>(sums + kKeyGroups * kRows * kPitch);   // [kKeyGroups][kRows]
    __syncthreads();  // the tiles are done with
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        const int r = key_group * kRows + (row_group * kQ + qt) * 16 + column;
        if (quarter == 0) group_parts[r] = Part{all[qt], sum[qt]};
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) *reinterpret_cast<f32x4*>(sums + r * kPitch + d * 16 + quarter * 4) = out[qt][d];
    }
    __syncthreads();
    constexpr int kFours = kDim / 4;
    for (int i = tid; i < kRows * kFours; i += kThreads) {
        const int r = i / kFours, d = i % kFours * 4;
        float highest = -__builtin_inff(), total = 0.0f;
#pragma unroll
        for (int g = 0; g < kKeyGroups; ++g) highest = fmaxf(highest, group_parts[g * kRows + r].most);
        f32x4 x{0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < kKeyGroups; ++g) {
            const float by = exp2_between(group_parts[g * kRows + r].most, highest);
            total = __builtin_fmaf(group_parts[g * kRows + r].sum, by, total);
            const f32x4 y = *reinterpret_cast<const f32x4*>(sums + (g * kRows + r) * kPitch + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(y[j], by, x[j]);
        }
        put(first_row + r, d, x, highest, total);
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
    int dim, sixteens, key_groups;  // kDim, kQ, kKeyGroups
    uint32_t row_tiles, splits, split_keys;
};

constexpr uint32_t kMostSplits = 64;  // a lane of the joining wavefront each

Shape shape_of(const TreeAttentionArgs& a, int compute_units) {
    Shape s;
    s.dim = a.cache.head_dim <= 64 ? 64 : a.cache.head_dim <= 128 ? 128 : 256;
    const uint64_t rows = static_cast<uint64_t>(a.max_query_len) * a.group;
    if (s.dim == 256) {  // two stages of four groups' tiles would not fit LDS, and two sixteens of rows not the registers
        s.sixteens = 1;
        s.key_groups = rows <= 32 ? 2 : 1;
    } else {
        s.sixteens = rows <= 16 ? 1 : 2;
        s.key_groups = rows <= 32 ? 4 : rows <= 64 ? 2 : 1;
    }
    const uint64_t tile_rows = 16 * s.sixteens * (kWaves / s.key_groups);
    s.row_tiles = static_cast<uint32_t>((rows + tile_rows - 1) / tile_rows);
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

template <int kDim, bool kBf16, bool kF32, int kQ, int kKeyGroups>
hipError_t attend(hipStream_t stream, const TreeAttentionArgs& a, const Shape& s, void* workspace) {
    static LdsLimit limit;
    constexpr size_t lds = attention_lds_bytes<kDim, kQ, kKeyGroups>();
    const auto kernel = tree_attention_kernel<kDim, kBf16, kF32, kQ, kKeyGroups>;
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
    if constexpr (kDim == 256) {
        if (s.key_groups == 2) return attend<kDim, kBf16, kF32, 1, 2>(stream, a, s, workspace);
        return attend<kDim, kBf16, kF32, 1, 1>(stream, a, s, workspace);
    } else {
        if (s.sixteens == 1) return attend<kDim, kBf16, kF32, 1, 4>(stream, a, s, workspace);
        if (s.key_groups == 4) return attend<kDim, kBf16, kF32, 2, 4>(stream, a, s, workspace);
        if (s.key_groups == 2) return attend<kDim, kBf16, kF32, 2, 2>(stream, a, s, workspace);
        return attend<kDim, kBf16, kF32, 2, 1>(stream, a, s, workspace);
    }
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
