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
// keys 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3).  V comes row-major and is needed column-major: it is read from LDS with the
// transposing ds_read_b64_tr_b16.  F32 queries and the weights beside them are two terms of f16 or three of bf16, each a product
// of its own: 22 and 24 bits.  A weight's first term has sums of its own.  f16 ends at 2^-24: its weights are kept high in the type
// (kLift), and the second term is 2^12 times itself.
//
// Keys and values come in tiles of 32 keys from memory straight into a ring of tiles in LDS (no registers in between),
// requested kStages - 1 tiles ahead, their places found a tile before that.  The wavefronts of a workgroup share its tiles and
// have 16 kQ rows each: a lone wavefront (no barrier anywhere) up to 16 rows, four of them, and every key read once, for 64 or 128.
// Long contexts are shared out over workgroups by the lengths that the device holds, so that ragged requests keep all of them
// busy to the end, and a second kernel joins the parts.  Short ones stay with one workgroup a key head: it has kKeyGroups such
// groups of wavefronts that take tiles in turn, and adds them up itself.
//
// What bounds it, on heads of 128, 32 of them on 8 key heads, 5.15 TB/s being what a copy reaches.  Few rows: the cache's bytes.
// 64 requests of 1 token on 4000 keys 185 us (5.7 TB/s), on 1000 keys 53 us (4.9); 2 requests of 7 to 13 tokens x 28 heads on 107000
// and 119000 keys 110 us (4.2 TB/s).  Many rows: the issue of a tile, 32 matrix instructions and 142 others (16 exponentials among
// them) a wavefront with 32 rows, of which two fit a SIMD: 8 requests of 64 tokens on 8000 keys 107 us, 630 TFLOP/s.  Short
// contexts: the round trips to memory before the first tile (lengths, block table, keys), and a tile's own latency, 0.85 us: 8
// requests of 64 tokens on 20 keys (3 tiles) 11.9 us, on 190 keys (8 tiles) 16.3.
#include "paged_launch.h"

#include <hip/hip_runtime.h>
#include <math.h>

#include <type_traits>

namespace afhip {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int kTile = 32;             // keys of one wavefront's step
constexpr uint32_t kNowhere = ~0u;    // of a key that has no place in the cache
constexpr float kLog2e = 1.4426950408889634f;
// The number that is taken off a row's scores follows their maximum only when that passes it by more than kSlack: the weights
// stay below 2^kSlack, far inside every type here, most tiles leave the sums as they are, and no lane has to know the others'
// scores to see that.
constexpr float kSlack = 8.0f;
constexpr float kUnset = 3e38f;
constexpr float kLowest = -3e38f;        // the maximum of a row whose seen scores are all minus infinity, or no numbers
constexpr float kLeastUnit = 0x1p-126f;  // of what a product is multiplied by
// Where a row's largest weight is put (a power of two): as high as f16 allows, whose steps below 2^-14 are 2^-24 whatever the
// weight.  Half a step is 2^-32 of the largest weight then, 2^-44 where there is a second term of 2^12 times the rest.  bf16 has
// f32's exponents.
template <bool kBf16>
constexpr float kLift = kBf16 ? 0.0f : 7.0f;
constexpr float kRestScale = 4096.0f;  // (the rest of a weight of 2^15 is 2^3 at most)

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

__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& d) { return __umulhi(n, d.multiplier) + (n & d.whole); }

// What a split of a request's keys holds for one row: the row's maximum (in units of log2, minus infinity where it saw no key) and
// the sum of its weights.
struct Part {
    float most, sum;
};
__device__ __forceinline__ Part part_of(bool saw, float shift, float sum) { return Part{!saw ? -__builtin_inff() : shift == kUnset ? kLowest : -shift, sum}; }

// exp2(a - b) where both may be minus infinity (nothing seen yet): then 1, of sums that are zero.
__device__ __forceinline__ float exp2_between(float a, float b) { return a == b ? 1.0f : __builtin_amdgcn_exp2f(a - b); }

// Which of the 32 keys from `first` on a row sees: bit j for key first + j.  `word0`: the row's first mask word; `words` null:
// no masks.
__device__ __forceinline__ uint32_t seen_bits(int first, int context, int token, unsigned long long word0, const unsigned long long* words, int count) {
    const int draft = first - context;  // the first key as a new token of the request
    if (words == nullptr) {
        const int left = token + 1 - draft;
        return left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
    }
    if (draft <= -32) return ~0u;
    if (draft < 0) return static_cast<uint32_t>(word0 << -draft) | ((1u << -draft) - 1);
    const int word = draft >> 6, shift = draft & 63;
    unsigned long long low = word0, high = 0;
    if (count > 1) {  // (otherwise no memory is read here)
        low = word < count ? words[word] : 0ull;
        if (shift > 32 && word + 1 < count) high = words[word + 1];
    } else if (word > 0) {
        low = 0;
    }
    unsigned long long bits = low >> shift;
    if (shift > 32) bits |= high << (64 - shift);
    return static_cast<uint32_t>(bits);
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// No finite number: all bits of the exponent.
template <bool kBf16>
__device__ __forceinline__ bool is_odd(unsigned short v) {
    constexpr unsigned short kExponent = kBf16 ? 0x7F80 : 0x7C00;
    return (v & kExponent) == kExponent;
}

__device__ const uint4 kNothing{0, 0, 0, 0};  // what values past a head's end are loaded from

// 16 bytes a lane from memory to 1 KiB of LDS from `to` on (a uniform address).
__device__ __forceinline__ void load_to_lds(uint32_t to, const uint4* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}

// Where 16-byte piece `piece` of row `row` of a tile lies in LDS, in pieces.  The pieces of a row are in an order of its own,
// so that what the lanes of an operand read falls on all banks (256 bytes of them): one piece of 16 rows of K, two
// neighbouring pieces of eight rows of V.
template <int kDim>
__device__ __forceinline__ int key_piece(int row, int piece) {
    constexpr int kPieces = kDim / 8;
    return row * kPieces + (kPieces == 8 ? piece ^ (row >> 1 & 7) : piece ^ (row & 15));
}
template <int kDim>
__device__ __forceinline__ int value_piece(int row, int piece) {
    constexpr int kPieces = kDim / 8;
    return row * kPieces + (kPieces == 8 ? piece ^ (row & 6) : piece ^ (row << 1 & 14));
}

// s_waitcnt for "at most kLeft vector memory operations outstanding" (nothing else waited for).
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLeft) : "memory");
}

// Four values of a result from their sums; zero where nothing was seen (a sum of zero of what was seen, weights of minus infinity
// only, makes no numbers).
template <bool kBf16, bool kF32>
__device__ __forceinline__ void store_row(const TreeAttentionArgs& a, size_t token, uint32_t head, int d, f32x4 x, float total, bool saw) {
    const size_t to = token * a.out_token_stride + static_cast<size_t>(head) * a.out_head_stride + d;
    const float by = saw ? 1.0f / total : 0.0f;
    if (kF32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + to) = x * by;
    } else {
        s16x4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = narrow<kBf16>(x[j] * by);
        *reinterpret_cast<s16x4*>(static_cast<uint16_t*>(a.out) + to) = y;
    }
}

// What the launch's shape and the lengths on the device say of one request.
struct Share {
    int begin, tokens, context, keys;   // its first row of query, new tokens, cached tokens, both together
    uint32_t row_tiles, splits, tiles;  // workgroups' rows, parts of its keys, tiles of keys in a part
    uint32_t first, first_slot;         // number of its first workgroup, and of its first part
};

__device__ __forceinline__ Share lengths_of(const TreeAttentionArgs& a, uint32_t request, int rows_a_tile) {
    Share s{};
    s.begin = min(max(a.query_starts[request], 0), static_cast<int>(a.tokens));
    const int end = min(max(a.query_starts[request + 1], s.begin), static_cast<int>(a.tokens));
    s.tokens = min(end - s.begin, static_cast<int>(a.max_query_len));
    s.context = max(a.context_lens[request], 0);
    const unsigned long long most = min(static_cast<unsigned long long>(a.table_columns) * a.block_size.by, static_cast<unsigned long long>(a.max_key_len));
    s.keys = static_cast<int>(min(static_cast<unsigned long long>(s.context) + s.tokens, most));
    s.row_tiles = (static_cast<uint32_t>(s.tokens) * a.group + rows_a_tile - 1) / rows_a_tile;
    return s;
}

// A lane's value of the data-parallel move kControl, zero where the move has none for it or its row of 16 is not in kRows.
template <int kControl, int kRows, typename T>
__device__ __forceinline__ T moved(T v) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kControl, kRows, 0xF, false));
}

// Sum over the wavefront's lanes up to this one: within rows of 16 lanes, then the rows below.
template <typename T>
__device__ __forceinline__ T sum_up_to(T v) {
    v += moved<0x111, 0xF>(v);  // from 1, 2, 4, 8 lanes below
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    v += moved<0x142, 0xA>(v);  // a row's last lane to the next row
    v += moved<0x143, 0xC>(v);  // lane 31 to the upper half
    return v;
}

// How the keys are shared out.  A part has the same number of tiles for all requests (evened out within a request), `least`
// at least: the smallest of a few sizes for which the parts, each request's rounded up, are no more than plan.most
// workgroups.  The sizes lie between what plan.most would hold if nothing had to be rounded and what it surely holds, when
// the rounding adds a part to every row tile and key head.  Workgroups are numbered by request, key head, part, row tile;
// parts of requests that have several are numbered the same way.  Every wavefront works this out for itself from the lengths.
struct SharePlan {
    uint32_t target, most, least;  // workgroups without and with the rounding's
    uint32_t row_tiles;            // of the largest request
    uint32_t slots;                // parts that there is room for
    bool one_round;                // all parts at once: as many as plan.most allows
    bool even;                     // otherwise every request is one part, and has as many workgroups as the largest may need
};

// `of`: a workgroup's number (by_request false) or a request's.  False: there is no such workgroup.
template <bool kByRequest>
__device__ __forceinline__ bool find_share(const TreeAttentionArgs& a, const SharePlan& plan, int rows_a_tile, uint32_t of, uint32_t* request, Share* out) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const uint32_t heads = a.cache.kv_heads;
    if (!plan.even) {
        const uint32_t r = kByRequest ? of : of / (heads * plan.row_tiles);
        if (r >= a.requests) return false;
        *request = r;
        *out = lengths_of(a, r, rows_a_tile);
        out->splits = 1;
        out->tiles = (out->keys + kTile - 1) / kTile;
        out->first = r * heads * plan.row_tiles;
        out->row_tiles = plan.row_tiles;  // (its numbering; rows past its own are empty)
        return true;
    }
    Share mine{};
    float work = 0.0f;  // (a float's error is far below the whole tiles that parts are rounded to: 2^-10 more covers it)
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 64) {
        if (r0 + lane < a.requests) {
            mine = lengths_of(a, r0 + lane, rows_a_tile);
            work += static_cast<float>((mine.keys + kTile - 1) / kTile) * static_cast<float>(mine.row_tiles);
        }
    }
    work = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sum_up_to(work)), 63));
    const auto size = [&](uint32_t workgroups) {
        const float each = work * (static_cast<float>(heads) * 1.001f) / static_cast<float>(workgroups);
        return max(static_cast<uint32_t>(fminf(each, 0x1p30f)) + 1, plan.least);
    };
    // (a quotient in floats, rounded up but for a thousandth of a part, which is more than its error: the same here and below, and
    // a part's tiles follow from it)
    const auto parts_of = [](uint32_t all, float inverse) { return max(static_cast<uint32_t>(static_cast<float>(all) * inverse + 0.999f), 1u); };
    constexpr int kSizes = 4;
    const uint32_t surely = size(plan.target), hardly = plan.one_round ? min(size(plan.most), surely) : surely;
    uint32_t tiles = surely;
    if (hardly < surely) {
        uint32_t sizes[kSizes], counts[kSizes];
        float inverse[kSizes];
#pragma unroll
        for (int i = 0; i < kSizes; ++i) {
            sizes[i] = hardly + (surely - hardly) * i / kSizes;
            inverse[i] = __builtin_amdgcn_rcpf(static_cast<float>(sizes[i]));
            counts[i] = 0;
        }
        for (uint32_t r0 = 0; r0 < a.requests; r0 += 64) {
            if (r0 + lane < a.requests) {
                if (a.requests > 64) mine = lengths_of(a, r0 + lane, rows_a_tile);
                const uint32_t all = (mine.keys + kTile - 1) / kTile;
#pragma unroll
                for (int i = 0; i < kSizes; ++i) counts[i] += mine.row_tiles * parts_of(all, inverse[i]);
            }
        }
#pragma unroll
        for (int i = kSizes - 1; i >= 0; --i) {
            const uint32_t parts = __builtin_amdgcn_readlane(sum_up_to(counts[i]), 63);
            if (parts * heads <= plan.most) tiles = sizes[i];
        }
    }
    const float inverse_tiles = __builtin_amdgcn_rcpf(static_cast<float>(tiles));
    uint32_t before = 0, slots_before = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 64) {
        uint32_t count = 0, slots = 0;
        mine.splits = 0;
        if (r0 + lane < a.requests) {
            if (a.requests > 64) mine = lengths_of(a, r0 + lane, rows_a_tile);
            const uint32_t all = (mine.keys + kTile - 1) / kTile;
            mine.splits = parts_of(all, inverse_tiles);
            mine.tiles = (all + mine.splits - 1) / mine.splits;
            count = mine.row_tiles * mine.splits * heads;
            slots = mine.splits > 1 ? count : 0;
        }
        const uint32_t upto = sum_up_to(count), slots_upto = sum_up_to(slots);
        mine.first = before + upto - count;
        mine.first_slot = slots_before + slots_upto - slots;
        const unsigned long long here = kByRequest ? (of >= r0 && of < r0 + 64 ? 1ull << (of - r0) : 0ull)
                                                   : __ballot(of >= mine.first && of < mine.first + count);
        if (here != 0) {
            const int l = __builtin_ctzll(here);
            *request = r0 + l;
            out->begin = __builtin_amdgcn_readlane(mine.begin, l);
            out->tokens = __builtin_amdgcn_readlane(mine.tokens, l);
            out->context = __builtin_amdgcn_readlane(mine.context, l);
            out->keys = __builtin_amdgcn_readlane(mine.keys, l);
            out->row_tiles = __builtin_amdgcn_readlane(mine.row_tiles, l);
            out->splits = __builtin_amdgcn_readlane(mine.splits, l);
            out->tiles = __builtin_amdgcn_readlane(mine.tiles, l);
            out->first = __builtin_amdgcn_readlane(mine.first, l);
            out->first_slot = __builtin_amdgcn_readlane(mine.first_slot, l);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        slots_before += __builtin_amdgcn_readlane(slots_upto, 63);
    }
    return false;
}

// kDim: the head's values, rounded up to a size that is here (the rest are zeros).  kF32: query and out are f32.
// Two wavefronts a SIMD (256 registers) wherever the sums leave room for them, all but heads of 256 (8 requests of 5 tokens on 3000
// keys, f32 on f16: 28.9 us, with the 260 to 320 registers that the compiler takes when it may 37.7).
template <int kDim, bool kBf16, bool kF32, int kQ, int kRowWaves, int kKeyGroups, int kStages>
__global__ __launch_bounds__(kRowWaves * kKeyGroups * 64, kDim == 256 ? 1 : 2) void tree_attention_kernel(TreeAttentionArgs a, SharePlan plan, float* part_out,
                                                                                                 Part* parts) {
    constexpr int kSteps = kDim / 32;                            // products of K Q^T along the head
    constexpr int kTerms = kF32 ? (kBf16 ? 3 : 2) : 1;           // of a query value or a weight: 24 bits of three bf16, 22 of two f16
    constexpr int kWaves = kRowWaves * kKeyGroups, kRows = 16 * kQ * kRowWaves, kStep = kTile * kKeyGroups;
    constexpr int kPieces = kDim / 8;                            // 16-byte pieces of a row
    constexpr int kTileBytes = kTile * kDim * 2;                 // of K, and of V behind it
    constexpr int kLoads = kTile * kPieces / 64 / kRowWaves;     // of a wavefront, 1 KiB each, for K and for V
    extern __shared__ __attribute__((aligned(1024))) char lds[];

    // workgroups go round the eight XCDs in turn: the row tiles of a part, which share its keys, lie on one and share its L2
    const uint32_t number = ((blockIdx.x >> 3) / plan.row_tiles * 8 + (blockIdx.x & 7)) * plan.row_tiles + (blockIdx.x >> 3) % plan.row_tiles;
    uint32_t request;
    Share share;
    if (!find_share<false>(a, plan, kRows, number, &request, &share)) return;
    const uint32_t inside = number - share.first, row_tile = inside % share.row_tiles, split = inside / share.row_tiles % share.splits;
    const uint32_t kv_head = inside / share.row_tiles / share.splits, slot = share.first_slot + inside;
    const int begin = share.begin, context = share.context, group = static_cast<int>(a.group), rows = share.tokens * group;
    const int first_row = static_cast<int>(row_tile) * kRows;
    if (first_row >= rows || (share.splits > 1 && slot >= plan.slots)) return;
    int keys = share.keys;
    const int last_token = min(first_row + kRows - 1, rows - 1) / group;
    if (a.masks == nullptr) keys = static_cast<int>(min(static_cast<unsigned long long>(keys), static_cast<unsigned long long>(context) + last_token + 1));
    const int split_keys = static_cast<int>(share.tiles) * kTile;  // (splits * split_keys < keys + splits * kTile: far from 2^31)
    const int key_begin = min(static_cast<int>(split) * split_keys, keys), key_end = min(key_begin + split_keys, keys);

    const int tid = static_cast<int>(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int column = lane & 15, quarter = lane >> 4;
    const int row_wave = wave % kRowWaves, key_group = wave / kRowWaves;
    const int my_row = first_row + row_wave * 16 * kQ;  // of this wavefront's first
    const bool works = my_row < rows;               // otherwise it only helps to load
    if (share.splits > 1 && key_begin >= key_end) {  // none of this part's keys is there for these rows: the part says so
        for (int r = tid; r < kRows; r += kWaves * 64) parts[static_cast<size_t>(slot) * kRows + r] = Part{-__builtin_inff(), 0.0f};
        return;
    }
    char* const ring = lds + key_group * (kStages * 2 * kTileBytes);
    const uint32_t ring_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)ring));
    const int pieces = static_cast<int>(a.cache.head_dim / 8);  // that hold something
    const bool whole_heads = pieces == kPieces;

    // where 64 blocks from `window_at` on lie, in 16-byte units, one a lane; which of them there are
    const int* table = a.block_tables + static_cast<size_t>(request) * a.table_columns;
    const uint32_t last_block = key_begin < key_end ? divide(static_cast<uint32_t>(key_end - 1), a.block_size) : 0;
    uint32_t window = 0, window_at = 0, window_end = 0;  // (keys from window_end on are not in it)
    unsigned long long there = 0;
    // Where this lane's row of load i of a tile lies.  (A key without a place is not seen by any row: what is loaded for it may
    // be anything.)
    uint32_t block_at[kLoads], past[kLoads];  // its block's place, and how far into the block
    auto find_rows = [&](int tile) -> uint32_t {  // the tile's keys that have a place
        if (static_cast<uint32_t>(tile) + kTile > window_end) {
            window_at = divide(static_cast<uint32_t>(tile), a.block_size);
            const uint32_t block_column = window_at + lane;
            const uint32_t block = block_column <= last_block ? static_cast<uint32_t>(table[block_column]) : kNowhere;
            there = __ballot(block < a.cache.blocks);
            window = block < a.cache.blocks ? block * a.cache.block_stride + kv_head * a.cache.head_stride : 0;
            window_end = (window_at + 64) * a.block_size.by;  // (below 2^32: a bound of the keys times the block size)
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t key = static_cast<uint32_t>(tile) + (row_wave * kLoads + i) * (64 / kPieces) + lane / kPieces, block = divide(key, a.block_size);
            // (a place past the last key's block is block 0's)
            block_at[i] = static_cast<uint32_t>(__shfl(static_cast<int>(window), static_cast<int>(block - window_at)));
            past[i] = (key - block * a.block_size.by) * a.cache.slot_stride;
        }
        const uint32_t key = static_cast<uint32_t>(tile) + (lane & 31), column_of = divide(key, a.block_size) - window_at;
        return static_cast<uint32_t>(__ballot((there >> column_of & 1) != 0 && static_cast<int>(key) < key_end));
    };
    // Requests this wavefront's part of the K and V that find_rows() has found.
    auto request_tile = [&](int stage) {
        const uint32_t to = ring_at + stage * (2 * kTileBytes) + row_wave * (kLoads * 1024);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int slot = (row_wave * kLoads + i) * 64 + lane, row = slot / kPieces;
            const int kp = key_piece<kDim>(row, slot % kPieces) % kPieces, vp = value_piece<kDim>(row, slot % kPieces) % kPieces;
            const uint32_t from = block_at[i] + past[i];
            const uint4 *k = a.cache.keys + (from + kp), *v = a.cache.values + (from + vp);
            if (!whole_heads) {
                if (kp >= pieces) k = &kNothing;
                if (vp >= pieces) v = &kNothing;
            }
            load_to_lds(to + i * 1024, k);
            load_to_lds(to + kTileBytes + i * 1024, v);
        }
    };
    // ---- the rows
    // (requested before the tiles: what waits for them does not wait for a tile)
    uint4 raw[kQ][kSteps][kF32 ? 2 : 1];
    float unit[kQ];  // what a product of the row is multiplied by: |scale|, log2(e), and for f32 on f16 the row's power of two
    const unsigned long long* words[kQ];
    unsigned long long word0[kQ];
    int row_token[kQ];
    bool real[kQ];
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        const int row = my_row + qt * 16 + column;
        real[qt] = row < rows;
        row_token[qt] = real[qt] ? row / group : 0;
        const int head = static_cast<int>(kv_head) * group + (real[qt] ? row % group : 0);
        const size_t token = static_cast<size_t>(begin + row_token[qt]);
        words[qt] = a.masks != nullptr ? a.masks + token * a.mask_words : nullptr;
        word0[qt] = a.masks != nullptr && a.mask_words > 0 ? words[qt][0] : 0ull;
        unit[qt] = __builtin_fabsf(a.scale) * kLog2e;
        const size_t from = token * a.query_token_stride + static_cast<size_t>(head) * a.query_head_stride;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int piece = s * 4 + quarter;
            const char* p = static_cast<const char*>(a.query) + (from + static_cast<size_t>(piece) * 8) * (kF32 ? 4 : 2);
#pragma unroll
            for (int i = 0; i < (kF32 ? 2 : 1); ++i) raw[qt][s][i] = real[qt] && piece < pieces ? reinterpret_cast<const uint4*>(p)[i] : uint4{0, 0, 0, 0};
        }
    }

    uint32_t held_ahead[kStages];  // of the tiles on their way, the next one's first, and of the one found
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
        const int tile = key_begin + key_group * kTile + i * kStep;
        held_ahead[i] = tile < key_end ? find_rows(tile) : 0u;
        if (i < kStages - 1 && tile < key_end) request_tile(i);
    }

    s16x8 query[kQ][kSteps][kTerms];
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;  // a negative scale turns the queries round
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        if (kF32) {
            float v[kSteps][8];
            float most = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint4 four = raw[qt][s][j / 4 * kF32];
                    const uint32_t words[4] = {four.x, four.y, four.z, four.w};
                    v[s][j] = __builtin_bit_cast(float, words[j % 4]);
                    if (flip != 0) v[s][j] = -v[s][j];
                    most = fmaxf(most, __builtin_fabsf(v[s][j]));
                }
            }
            if (!kBf16) {
                // f16 has 5 exponent bits: the row's largest value goes to [2^14, 2^15), and half of the second term's smallest step
                // is 2^-39 of it
                most = row_max(most);
                const bool moves = most > 0.0f && most < __builtin_inff();
                const int exponent = moves ? __builtin_amdgcn_frexp_expf(most) - 15 : 0;
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
                const uint4 v = raw[qt][s][0];
                query[qt][s][0] = __builtin_bit_cast(s16x8, uint4{v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip});
            }
        }
        // (never 0, which would make the minus infinity of a key that is not seen no number; nor none, which the queries are instead)
        if (!(unit[qt] >= kLeastUnit)) unit[qt] = kLeastUnit;
        if (__builtin_isnan(a.scale)) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int term = 0; term < kTerms; ++term) query[qt][s][term] = static_cast<s16x8>(-1);
            }
        }
    }

    f32x4 out[kQ][kDim / 16];
    // The later terms' sums, with f16 kRestScale times themselves.  An infinite value makes infinities of either sign or no numbers of
    // them; those of the first terms are what the weights would make of it.
    constexpr bool kApart = kF32;
    constexpr float kRestIs = kBf16 ? 1.0f : kRestScale;
    f32x4 low[kApart ? kQ : 1][kApart ? kDim / 16 : 1];
    // A weight is exp2(product * unit + shift): the shift takes off the row's largest score (up to kSlack more than it) and adds
    // kLift, kUnset until the row has seen a key.  And this lane's part of the weights' sum.
    constexpr float kHighest = kLift<kBf16> + kSlack;
    float shift[kQ], sum[kQ];
    uint32_t saw[kQ];       // not zero: the row has seen a key of a tile that not every row sees
    uint32_t all_saw = 0;  // not zero: every row has seen a tile
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        shift[qt] = kUnset;
        sum[qt] = 0.0f;
        saw[qt] = 0;
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) {
            out[qt][d] = f32x4{0, 0, 0, 0};
            if constexpr (kApart) low[qt][d] = f32x4{0, 0, 0, 0};
        }
    }

    // ---- the keys
    int stage = 0, free_stage = kStages - 1;
    for (int first = key_begin; first < key_end; first += kStep) {
        const int tile = first + key_group * kTile;
        // this wavefront's part of the tile is there: all but what was requested behind it, all of it near the end
        if (tile + (kStages - 2) * kStep < key_end) wait_loads<2 * kLoads * (kStages - 2)>();
        else wait_loads<0>();
        if (kRowWaves > 1) __syncthreads();        // everyone's is, and the stage to be filled has been read
        const uint32_t held = held_ahead[0];
#pragma unroll
        for (int i = 0; i + 1 < kStages; ++i) held_ahead[i] = held_ahead[i + 1];
        if (tile + (kStages - 1) * kStep < key_end) request_tile(free_stage);
        if (tile + kStages * kStep < key_end) held_ahead[kStages - 1] = find_rows(tile + kStages * kStep);  // a tile ahead of its request
        const char* k_lds = ring + stage * (2 * kTileBytes);
        const char* v_lds = k_lds + kTileBytes;
        stage = stage + 1 == kStages ? 0 : stage + 1;
        free_stage = free_stage + 1 == kStages ? 0 : free_stage + 1;
        if (!works || tile >= key_end) continue;
        const bool clean = tile + kTile <= context && held == ~0u;  // every row sees every key
        all_saw |= clean;

        // the operands of a product first, all of them: none of them waits for LDS by itself
        s16x8 key[2][kSteps];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s)  // (rows 16 apart have their pieces in the same order)
                key[half][s] = *reinterpret_cast<const s16x8*>(k_lds + key_piece<kDim>(column, s * 4 + quarter) * 16 + half * (16 * kDim * 2));
        }
        __builtin_amdgcn_sched_barrier(0);
        f32x4 score[kQ][2];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; --term)  // the small terms first
                        score[qt][half] = mfma<kBf16>(key[half][s], query[qt][s][term], s == 0 && term == kTerms - 1 ? f32x4{0, 0, 0, 0} : score[qt][half]);
                }
            }
        }
        s16x8 value[kDim / 16];
#pragma unroll
        for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = quarter * 4 + (column >> 2);
                const char* from = v_lds + value_piece<kDim>(row, d * 2 + (column >> 1 & 1)) * 16 + (column & 1) * 8 + half * (16 * kDim * 2);
                const s16x4 four = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)from);
#pragma unroll
                for (int j = 0; j < 4; ++j) value[d][half * 4 + j] = four[j];
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        uint32_t odd = 0;  // keys with a value that is no finite number (looked for only where some row may not see them)
        uint32_t seen[kQ];
        if (!clean) {
            u16x2 most[4];  // largest magnitudes of this lane's keys: two a register, as in `value`
#pragma unroll
            for (int pair = 0; pair < 4; ++pair) {
                most[pair] = u16x2{0, 0};
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
                    const u16x2 two{static_cast<unsigned short>(value[d][2 * pair]), static_cast<unsigned short>(value[d][2 * pair + 1])};
                    most[pair] = __builtin_elementwise_max(most[pair], static_cast<u16x2>(two & static_cast<unsigned short>(0x7FFF)));
                }
            }
            u16x2 all = __builtin_elementwise_max(__builtin_elementwise_max(most[0], most[1]), __builtin_elementwise_max(most[2], most[3]));
            if (__any(is_odd<kBf16>(all[0]) || is_odd<kBf16>(all[1]))) {  // which keys
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const unsigned long long which = __ballot(is_odd<kBf16>(most[j / 2][j % 2]));
#pragma unroll
                    for (int holder = 0; holder < 4; ++holder) {
                        if ((which >> (holder * 16) & 0xFFFF) != 0) odd |= 1u << (j / 4 * 16 + holder * 4 + j % 4);
                    }
                }
            }
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
                seen[qt] = real[qt] ? seen_bits(tile, context, row_token[qt], word0[qt], words[qt], static_cast<int>(a.mask_words)) & held : 0u;
                saw[qt] |= seen[qt];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if ((seen[qt] >> (half * 16 + quarter * 4 + j) & 1) == 0) score[qt][half][j] = -__builtin_inff();
                    }
                }
            }
        }
        float x[kQ][8];
        bool passes = false;
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[qt][j] = __builtin_fmaf(score[qt][j >> 2][j & 3], unit[qt], shift[qt]);
            const auto larger = [](float a, float b) { return kF32 ? __builtin_elementwise_maximum(a, b) : fmaxf(a, b); };  // (f32 queries: no number if one is none)
            const float most = larger(larger(larger(x[qt][0], x[qt][1]), larger(x[qt][2], x[qt][3])), larger(larger(x[qt][4], x[qt][5]), larger(x[qt][6], x[qt][7])));
            passes |= kF32 ? !(most <= kHighest) : most > kHighest;
        }
        if (__any(passes)) {
            if constexpr (kF32) {
                // An infinite key: the terms of a query value may be zero or of either sign, and their infinities then make no number of
                // the score.  The first terms alone give it as the value would.
                bool none = false;
#pragma unroll
                for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) none |= __builtin_isnan(x[qt][j]);
                }
                if (__any(none)) {
                    f32x4 first_terms[kQ][2];
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const s16x8 k = *reinterpret_cast<const s16x8*>(k_lds + key_piece<kDim>(column, s * 4 + quarter) * 16 + half * (16 * kDim * 2));
#pragma unroll
                            for (int qt = 0; qt < kQ; ++qt) first_terms[qt][half] = mfma<kBf16>(k, query[qt][s][0], s == 0 ? f32x4{0, 0, 0, 0} : first_terms[qt][half]);
                        }
                    }
#pragma unroll
                    for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (__builtin_isnan(score[qt][j >> 2][j & 3])) score[qt][j >> 2][j & 3] = first_terms[qt][j >> 2][j & 3];
                            x[qt][j] = __builtin_fmaf(score[qt][j >> 2][j & 3], unit[qt], shift[qt]);
                        }
                    }
                }
            }
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
                const f32x4 lo = score[qt][0], hi = score[qt][1];
                const float peak = row_max(fmaxf(fmaxf(fmaxf(lo[0], lo[1]), fmaxf(lo[2], lo[3])), fmaxf(fmaxf(hi[0], hi[1]), fmaxf(hi[2], hi[3]))));
                // each row by itself: no other row's keys move its bits
                const float next = __builtin_fmaf(peak, unit[qt], shift[qt]) > kHighest ? __builtin_fmaf(-peak, unit[qt], kLift<kBf16>) : shift[qt];
                const float by = next == shift[qt] ? 1.0f : __builtin_amdgcn_exp2f(next - shift[qt]);
                shift[qt] = next;
                sum[qt] *= by;
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        out[qt][d][j] *= by;
                        if constexpr (kApart) low[qt][d][j] *= by;
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) x[qt][j] = __builtin_fmaf(score[qt][j >> 2][j & 3], unit[qt], next);
            }
        }
        // (With 16-bit queries a weight is one term, rounded to the cache's type: 8 trees of 64 drafts on 300 to 4000 keys in bf16 are off by
        // 1.86e-3 of their norm, where the rounding of the result alone makes 1.59e-3; a second term takes that away, and 49.6 us
        // instead of 44.3.)
        s16x8 weight[kQ][kTerms];
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = __builtin_amdgcn_exp2f(x[qt][j]);
                sum[qt] += p;
                float rest = p;
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    weight[qt][term][j] = narrow<kBf16>(rest);
                    if (term + 1 < kTerms) rest = (rest - widen<kBf16>(weight[qt][term][j])) * kRestIs;
                }
            }
        }
        odd = __builtin_amdgcn_readfirstlane(odd);
        if (odd != 0) {
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                for (int j = 0; j < 8; ++j) value[d][j] = is_odd<kBf16>(static_cast<unsigned short>(value[d][j])) ? static_cast<short>(0) : value[d][j];
            }
        }
#pragma unroll
        for (int term = kTerms - 1; term >= 0; --term) {
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                for (int qt = 0; qt < kQ; ++qt) {
                    if constexpr (kApart) {
                        if (term > 0) {
                            low[qt][d] = mfma<kBf16>(value[d], weight[qt][term], low[qt][d]);
                            continue;
                        }
                    }
                    out[qt][d] = mfma<kBf16>(value[d], weight[qt][term], out[qt][d]);
                }
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
                    const char* from = v_lds + value_piece<kDim>(key, d * 2 + (quarter >> 1)) * 16 + (quarter & 1) * 8;
                    const s16x4 four = *reinterpret_cast<const s16x4*>(from);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (is_odd<kBf16>(static_cast<unsigned short>(four[j]))) out[qt][d][j] = __builtin_fmaf(p, widen<kBf16>(four[j]), out[qt][d][j]);
                    }
                }
            }
        }
    }

    if constexpr (kApart) {
        float none = 0.0f;  // no number if one of the results is none
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    low[qt][d][j] = __builtin_fmaf(low[qt][d][j], 1.0f / kRestIs, out[qt][d][j]);
                    none = __builtin_fmaf(low[qt][d][j], 0.0f, none);
                }
            }
        }
        if (__any(__builtin_isnan(none))) {
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (!__builtin_isfinite(out[qt][d][j])) low[qt][d][j] = out[qt][d][j];
                    }
                }
            }
        }
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d) out[qt][d] = low[qt][d];
        }
    }

    // ---- the key groups' sums
    if constexpr (kKeyGroups > 1) {
        constexpr int kPitch = kDim + 4;                                                   // floats of a row in LDS
        float* sums = reinterpret_cast<float*>(lds);                                       // [kKeyGroups][kRows][kPitch]
        Part* group_parts = reinterpret_cast<Part*>(sums + kKeyGroups * kRows * kPitch);   // [kKeyGroups][kRows]
        __syncthreads();                                                                   // the tiles are done with
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
            const int r = key_group * kRows + (row_wave * kQ + qt) * 16 + column;
            const float total = row_sum(sum[qt]);
            if (quarter == 0) group_parts[r] = part_of((saw[qt] | all_saw) != 0, shift[qt], total);
#pragma unroll
            for (int d = 0; d < kDim / 16; ++d) *reinterpret_cast<f32x4*>(sums + r * kPitch + d * 16 + quarter * 4) = out[qt][d];
        }
        __syncthreads();
        for (int i = tid; i < kRows * (kDim / 4); i += kWaves * 64) {
            const int r = i / (kDim / 4), d = i % (kDim / 4) * 4, row = first_row + r;
            if (row >= rows || d >= pieces * 8) continue;
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
            store_row<kBf16, kF32>(a, static_cast<size_t>(begin + row / group), kv_head * a.group + row % group, d, x, total, highest != -__builtin_inff());
        }
        return;
    }

    // ---- out: a lane has four consecutive values of its row in each register group
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        const float total = row_sum(sum[qt]);
        if (!real[qt]) continue;
        const int row = my_row + qt * 16 + column;
        const size_t part = static_cast<size_t>(slot) * kRows + (row - first_row);
        if (share.splits > 1 && quarter == 0) parts[part] = part_of((saw[qt] | all_saw) != 0, shift[qt], total);
#pragma unroll
        for (int dt = 0; dt < kDim / 16; ++dt) {
            const int d = dt * 16 + quarter * 4;
            if (d >= pieces * 8) continue;
            if (share.splits > 1) *reinterpret_cast<f32x4*>(part_out + part * a.cache.head_dim + d) = out[qt][dt];
            else store_row<kBf16, kF32>(a, static_cast<size_t>(begin + row_token[qt]), kv_head * a.group + row % group, d, out[qt][dt], total, (saw[qt] | all_saw) != 0);
        }
    }
}

// The parts of a row, brought to their common maximum: a wavefront takes rows of one request in turn.  kLanes lanes have four
// values of a row each.  Few parts: every group of kLanes has a row of its own; many: the groups share a row's parts.  Up to
// eight parts are requested at a time.  Bound by the parts' bytes, which come from beyond the L2 that wrote them: 4 parts of 16384 rows
// of 128 (33 MB) 10 us, of which a launch and the lengths are 4.
constexpr int kJoinWaves = 4;
template <bool kBf16, bool kF32, int kLanes>
__global__ __launch_bounds__(kJoinWaves * 64) void join_parts_kernel(TreeAttentionArgs a, SharePlan plan, int rows_a_tile, const float* part_out,
                                                                    const Part* parts) {
    constexpr uint32_t kGroups = 64 / kLanes;
    uint32_t request;
    Share share;
    if (!find_share<true>(a, plan, rows_a_tile, blockIdx.y, &request, &share) || share.splits == 1) return;
    if (share.first_slot + share.row_tiles * share.splits * a.cache.kv_heads > plan.slots) return;  // (starts that go back: more rows than tokens)
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const uint32_t group = lane / kLanes, d = lane % kLanes * 4;
    const uint32_t rows = static_cast<uint32_t>(share.tokens) * a.group;  // of one key head
    const size_t stride = static_cast<size_t>(share.row_tiles) * rows_a_tile;
    const bool alone = share.splits <= 8;
    const uint32_t rows_a_wave = alone ? kGroups : 1, step = alone ? 1 : kGroups, first_part = alone ? 0 : group;
    for (uint32_t base = (blockIdx.x * kJoinWaves + (threadIdx.x >> 6)) * rows_a_wave; base < rows * a.cache.kv_heads; base += gridDim.x * kJoinWaves * rows_a_wave) {
        const uint32_t at = min(base + (alone ? group : 0), rows * a.cache.kv_heads - 1);  // (past the last row: it again, not stored)
        const uint32_t kv_head = at / rows, row = at % rows;
        const size_t slot = share.first_slot + static_cast<size_t>(kv_head) * share.splits * share.row_tiles + row / rows_a_tile;
        const size_t first = slot * rows_a_tile + row % rows_a_tile;
        float most = -__builtin_inff(), total = 0.0f;
        f32x4 x{0, 0, 0, 0};
        auto add = [&](auto batch, uint32_t s0) {  // (past the end: the last part again, not counted)
            constexpr int kBatch = decltype(batch)::value;
            f32x4 y[kBatch];
            Part part[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const uint32_t s = s0 + first_part + i * step;
                const size_t from = first + min(s, share.splits - 1) * stride;
                part[i] = parts[from];
                if (s >= share.splits) part[i] = Part{-__builtin_inff(), 0.0f};
                y[i] = *reinterpret_cast<const f32x4*>(part_out + from * a.cache.head_dim + (d < a.cache.head_dim ? d : 0));
            }
            float next = most;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) next = fmaxf(next, part[i].most);
            const float kept = exp2_between(most, next);
            total *= kept;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] *= kept;
            most = next;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const bool counts = part[i].most != -__builtin_inff();  // (a part that saw no key has not been written)
                const float by = counts ? exp2_between(part[i].most, most) : 0.0f;
                total = __builtin_fmaf(part[i].sum, by, total);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(counts ? y[i][j] : 0.0f, by, x[j]);
            }
        };
        uint32_t s0 = 0;
        for (; s0 + 8 * step <= share.splits; s0 += 8 * step) add(std::integral_constant<int, 8>{}, s0);
        for (; s0 + step < share.splits; s0 += 4 * step) add(std::integral_constant<int, 4>{}, s0);
        if (s0 < share.splits) add(std::integral_constant<int, 1>{}, s0);
#pragma unroll
        for (int w = kLanes; w < 64 && !alone; w *= 2) {
            const float other = __shfl_xor(most, w), next = fmaxf(most, other);
            const float mine = exp2_between(most, next), theirs = exp2_between(other, next);
            most = next;
            total = total * mine + __shfl_xor(total, w) * theirs;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = x[j] * mine + __shfl_xor(x[j], w) * theirs;
        }
        if ((alone ? base + group >= rows * a.cache.kv_heads : group != 0) || d >= a.cache.head_dim) continue;
        store_row<kBf16, kF32>(a, static_cast<size_t>(share.begin) + row / a.group, kv_head * a.group + row % a.group, d, x, total, most != -__builtin_inff());
    }
}

struct Shape {
    int dim, sixteens, waves;  // kDim, kQ, kRowWaves
    bool gathered;             // one workgroup for all keys of a key head
    int compute_units;
    SharePlan plan;
    uint64_t groups, slots;  // most workgroups, and parts of requests that have several
    int rows_a_tile() const { return 16 * sixteens * waves; }
};

// Sixteens of rows that a wavefront has where there are many: two where its registers leave room for another wavefront on the SIMD.
// Heads of 128, f32 on f16, one and two: 8 requests of 64 tokens on 300 keys 19.3 and 28.9 us, on 4000 keys 99 and 126, 512 tokens
// on 2000 keys 72 and 100; on bf16 20.6 and 32.5, 114 and 142, 81 and 111.
constexpr int most_sixteens(int dim, bool f32) { return dim == 256 || (dim == 128 && f32) ? 1 : 2; }

constexpr uint32_t kMostEvened = 1024;  // requests: every wavefront reads their lengths, 64 at a time

Shape shape_of(const TreeAttentionArgs& a, int compute_units) {
    Shape s;
    s.compute_units = compute_units;
    s.dim = a.cache.head_dim <= 64 ? 64 : a.cache.head_dim <= 128 ? 128 : 256;
    const uint64_t rows = static_cast<uint64_t>(a.max_query_len) * a.group;
    s.sixteens = rows <= 64 ? 1 : most_sixteens(s.dim, a.f32);
    s.waves = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    // One workgroup for all keys of a key head where a second launch would take longer than its tiles, one after the other: the more
    // such workgroups, the longer (8 key heads of 128, bf16, uniform lengths; in parts / gathered): 1 request of 1 token on 500 keys
    // 10.0 / 8.6 us, on 1000 10.4 / 13.2; 8 requests on 700 keys 13.3 / 12.0, on 1500 16.2 / 19.7; 32 requests on 700 keys 22.1 / 18.4,
    // on 2000 53.6 / 49.8.  Up to 2048 keys: past that ragged requests would keep few units busy.
    const uint64_t together = 512 + 6 * static_cast<uint64_t>(a.requests) * a.cache.kv_heads;
    s.gathered = rows <= 32 && a.max_key_len <= (together < 2048 ? together : 2048);
    const uint64_t tile_rows = s.rows_a_tile(), most_row_tiles = (rows + tile_rows - 1) / tile_rows;
    // row tiles of the whole batch: every request's last one may be part empty
    uint64_t row_tiles = static_cast<uint64_t>(a.tokens) * a.group / tile_rows + a.requests;
    if (row_tiles > a.requests * most_row_tiles) row_tiles = a.requests * most_row_tiles;
    const uint64_t tiles = (static_cast<uint64_t>(a.max_key_len) + kTile - 1) / kTile;
    s.plan.row_tiles = static_cast<uint32_t>(most_row_tiles);
    // A part's sums are written and read again, 8 head_dim bytes a row, where a tile of keys is 128 head_dim: fewer tiles than that, or
    // than two, are not worth a workgroup.
    s.plan.least = static_cast<uint32_t>(tile_rows / 16 > 2 ? tile_rows / 16 : 2);
    const uint64_t heads = a.cache.kv_heads, base = row_tiles * heads;
    // One round of what the compute units hold at once (by LDS and registers; lone wavefronts four, not the five whose LDS would be
    // all there is: 16 requests of 1 token on 8000 keys 107 us with four, 120 with five), the workgroups that rounding adds among
    // them; a batch that fills much of that anyway shares out over half a round more, three quarters for lone wavefronts (64
    // requests of 1 token on 100 to 4000 keys: 112 us with three quarters, 121 with half).  Workgroups of 128 rows, and of 64 f32
    // rows of heads of 128 where there are more, which the units are slow on, fill the round exactly: 8 requests of 64 tokens on 8000 keys
    // 103 us, with what surely fits 116 (f32 on f16 174 and 237).  Fewer rows wait for memory, and parts cost more than idle units
    // do: 24 requests of 16 tokens on 8000 keys 175 us filled, 172 not.
    const uint64_t resident = static_cast<uint64_t>(compute_units) * (s.waves == 1 ? 4 : s.waves == 2 ? 3 : 2);
    const uint64_t fewest = s.waves == 1 ? resident * 3 / 4 : resident / 2;
    s.plan.one_round = (s.sixteens == 2 || (a.f32 && s.dim == 128 && rows > 64)) && base <= resident;
    uint64_t target = resident > base ? resident - base : 0;
    if (target < fewest && !s.plan.one_round) target = fewest;
    s.plan.target = static_cast<uint32_t>(target);
    s.plan.most = static_cast<uint32_t>(base + target);
    s.plan.even = !s.gathered && a.requests <= kMostEvened;
    if (s.plan.even && s.plan.one_round) {
        // Parts are worth it where they save more tiles than the second launch takes (3 us) and their sums, in and out at 6 TB/s; a
        // tile takes 0.75 us, 1.4 times that with two workgroups on a unit.  64 tokens x 32 heads, 8 key heads of 128, bf16: 16
        // requests on 300 keys 20 us in one part and 33 in two, on 4000 keys 129 and 105; 1 request on 300 keys 18 and 16.5.
        const double parts = fmin(base == 0 ? 1.0 : floor(static_cast<double>(s.plan.most) / base), ceil(static_cast<double>(tiles) / s.plan.least));
        const double saved = tiles - tiles / parts * (base * parts > compute_units ? 1.4 : 1.0);
        s.plan.even = parts > 1 && saved > 4 + 0.029 * base * parts;
    }
    if (!s.plan.even) {
        s.groups = a.requests * most_row_tiles * heads;
    } else {
        const uint64_t finest = row_tiles * heads * (tiles <= s.plan.least ? 1 : (tiles + s.plan.least - 1) / s.plan.least);
        s.groups = s.plan.most;
        if (s.groups > finest) s.groups = finest;
    }
    s.groups = (s.groups + 8 * most_row_tiles - 1) / (8 * most_row_tiles) * (8 * most_row_tiles);
    s.slots = !s.plan.even || tiles <= s.plan.least ? 0 : s.groups;
    s.plan.slots = static_cast<uint32_t>(s.slots);
    return s;
}

size_t part_out_bytes(const TreeAttentionArgs& a, const Shape& s) {
    return (s.slots * s.rows_a_tile() * a.cache.head_dim * sizeof(float) + 255) / 256 * 256;
}

template <int kDim, bool kBf16, bool kF32, int kQ, int kRowWaves, int kKeyGroups, int kStages>
hipError_t attend(hipStream_t stream, const TreeAttentionArgs& a, const Shape& s, void* workspace) {
    static LdsLimit limit;
    constexpr size_t ring = static_cast<size_t>(kKeyGroups) * kStages * 2 * kTile * kDim * 2;
    constexpr size_t sums = kKeyGroups == 1 ? 0 : static_cast<size_t>(kKeyGroups) * 16 * kQ * kRowWaves * ((kDim + 4) * sizeof(float) + sizeof(Part));
    constexpr size_t lds = ring > sums ? ring : sums;
    static_assert(lds <= 160 * 1024, "a compute unit's LDS");
    const auto kernel = tree_attention_kernel<kDim, kBf16, kF32, kQ, kRowWaves, kKeyGroups, kStages>;
    hipError_t e = allow_lds(kernel, lds, &limit);
    if (e != hipSuccess) return e;
    float* part_out = static_cast<float*>(workspace);
    Part* parts = s.slots != 0 ? reinterpret_cast<Part*>(static_cast<char*>(workspace) + part_out_bytes(a, s)) : nullptr;
    kernel<<<static_cast<uint32_t>(s.groups), kRowWaves * kKeyGroups * 64, lds, stream>>>(a, s.plan, part_out, parts);
    e = hipGetLastError();
    if (e != hipSuccess || s.slots == 0) return e;
    // eight workgroups a compute unit over all requests, or one wavefront a row
    const uint64_t rows = static_cast<uint64_t>(a.max_query_len) * a.heads, most = (8 * static_cast<uint64_t>(s.compute_units) + a.requests - 1) / a.requests;
    const uint64_t groups = (rows + kJoinWaves - 1) / kJoinWaves;
    const dim3 grid(static_cast<uint32_t>(groups < most ? groups : most), a.requests);
    join_parts_kernel<kBf16, kF32, kDim / 4><<<grid, kJoinWaves * 64, 0, stream>>>(a, s.plan, s.rows_a_tile(), part_out, parts);
    return hipGetLastError();
}

// Groups of wavefronts that a workgroup with all of a head's keys has (by LDS).
constexpr int key_groups(int dim) { return dim == 256 ? 2 : 4; }

// The ring's length: as many stages as let two workgroups of four wavefronts, or four of one, on a unit's 160 KiB of LDS; key
// groups have two.
template <int kDim, bool kBf16, bool kF32>
hipError_t attend_rows(hipStream_t stream, const TreeAttentionArgs& a, const Shape& s, void* workspace) {
    constexpr int kGroups = key_groups(kDim);
    if (s.gathered) {
        if (s.waves == 1) return attend<kDim, kBf16, kF32, 1, 1, kGroups, 2>(stream, a, s, workspace);
        return attend<kDim, kBf16, kF32, 1, 2, kGroups, 2>(stream, a, s, workspace);
    }
    constexpr int kAlone = kDim == 64 ? 3 : 2, kTwo = kDim == 256 ? 2 : 3;
    if (s.waves == 1) return attend<kDim, kBf16, kF32, 1, 1, 1, kAlone>(stream, a, s, workspace);
    if (s.waves == 2) return attend<kDim, kBf16, kF32, 1, 2, 1, kTwo>(stream, a, s, workspace);
    if (s.sixteens == 1) return attend<kDim, kBf16, kF32, 1, 4, 1, kTwo>(stream, a, s, workspace);
    if constexpr (most_sixteens(kDim, kF32) == 2) return attend<kDim, kBf16, kF32, 2, 4, 1, 4>(stream, a, s, workspace);
    else return hipErrorInvalidValue;  // (one sixteen always)
}

template <int kDim>
hipError_t attend_types(hipStream_t stream, const TreeAttentionArgs& a, const Shape& s, void* workspace) {
    if (a.cache_bf16) return a.f32 ? attend_rows<kDim, true, true>(stream, a, s, workspace) : attend_rows<kDim, true, false>(stream, a, s, workspace);
    return a.f32 ? attend_rows<kDim, false, true>(stream, a, s, workspace) : attend_rows<kDim, false, false>(stream, a, s, workspace);
}

}  // namespace

size_t tree_attention_workspace_bytes(const TreeAttentionArgs& args, int compute_units) {
    const Shape s = shape_of(args, compute_units);
    return s.slots == 0 ? 0 : part_out_bytes(args, s) + s.slots * s.rows_a_tile() * sizeof(Part);
}

bool tree_attention_fits_a_launch(const TreeAttentionArgs& args, int compute_units) {
    const Shape s = shape_of(args, compute_units);
    return fits_a_launch(s.groups, static_cast<uint64_t>(s.waves) * (s.gathered ? key_groups(s.dim) : 1) * 64);
}

hipError_t launch_tree_attention(hipStream_t stream, const TreeAttentionArgs& args, void* workspace, int compute_units) {
    const Shape s = shape_of(args, compute_units);
    if (s.dim == 64) return attend_types<64>(stream, args, s, workspace);
    if (s.dim == 128) return attend_types<128>(stream, args, s, workspace);
    return attend_types<256>(stream, args, s, workspace);
}

}  // namespace afhip
