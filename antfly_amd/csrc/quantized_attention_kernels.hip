// Attention of a batch's new tokens over an 8-bit paged key / value cache.
//
//   out[t][h] = sum_j p_j u_j v_j / sum_j p_j,   p_j = exp(s_j - m),   s_j from scale * k_scale_j * (q . k_j),   u_j the value's scale
//
// One pass over the keys with a running reference m and sum of the softmax.  The rows of one key head are its query heads' tokens
// packed together (row = token * group + head in group), sixteen or 32 to a wavefront, so a key is read once for all of them.
//
// The products are on the 16 x 16 x 32 bf16 matrix instructions with the keys as the first operand: K Q^T has one row of the packed
// queries to a lane (column = lane % 16) and four keys in its registers, and these are, after the softmax, the second operand of
// V^T P^T as they stand.  Which key is which row of an instruction, and which of the head's values which row of which product, is
// free: row 4 q + i of half h of a tile is key 16 h + 4 i + q, so that the four quarters of a wavefront read four neighbouring keys,
// and value kVec * column + t is in product t, so that a lane's share of a key is one run of bytes.
//
// Codes come from memory straight into a ring of tiles in LDS that each wavefront has for itself (no barrier anywhere), and go to
// bf16, which holds every one of them exactly, as they are read from there; of values the bytes of two keys are put side by side
// before.  A tile's stage is requested anew as soon as its codes are in registers, so two tiles are on their way while a third is
// worked on.  F32 queries and the weights beside them are three terms of bf16, f16 two, each a product of its own; bf16 queries are
// one, but their weights two (one term of 8 bits would be the largest error of all; the second costs 0.6 us of 61 on 2 requests of
// 131000 keys).  On whole numbers the queries are three digits to the base 256, and K Q^T is on the i8 instructions: the codes as
// they are, sums exact.
//
// Wavefronts of a workgroup have parts of its keys and add up in LDS; long contexts are shared out over workgroups by the lengths
// that the device holds, and a second kernel joins the parts.
//
// Bound by the cache's bytes where keys are many: 64 requests of 100 to 4000 keys, 8 heads of 128 in whole numbers, 68 us, 4.2 TB/s;
// 2 requests of 99001 to 131000 keys, 4 heads of 128 e4m3, 53 us (4.5 TB/s) and 6 for the join.  The rest is the start: lengths, block
// table, then the first tiles, 4 to 7 us one after the other, so that one request of 700 keys takes 13 us, of which a launch is 4.
// Where a wavefront has few tiles (16 requests of 3 to 7 new tokens: 36 us with the join's 6) they are most of the time.  Prompts are bound
// by what is done for every tile of keys again by each 32 rows (4000 tokens, 32 heads on 8 of 128, bf16: 381 us on whole numbers, 332 on
// e4m3; 16 of 200 tokens 80 and 70, mostly starts).
#include "quantized_launch.h"

#include <hip/hip_runtime.h>

#include "xcd_order.h"

namespace afhip {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;
constexpr float kLog2e = 1.4426950408889634f;
// The number that is taken off a row's scores follows their maximum only when that passes it by more than kSlack (in units of log2):
// bf16 and f32 hold 2^kSlack as well as 1, most tiles leave the sums as they are, and no lane has to know the others' scores.
constexpr float kSlack = 12.0f;
constexpr float kLowest = -3e38f;  // the maximum of a row whose seen scores are all minus infinity

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
// Largest of, or sum over, the four lanes that hold a row (lane % 16), in all of them.
__device__ __forceinline__ float row_max(float v) {
    float other;
    swap_halves(&v, &other);
    v = fmaxf(v, other);
    swap_rows(&v, &other);
    return fmaxf(v, other);
}
__device__ __forceinline__ uint32_t row_max_bits(uint32_t v) {
    v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32)));
    return max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
}
__device__ __forceinline__ float row_sum(float v) {
    float other;
    swap_halves(&v, &other);
    v += other;
    swap_rows(&v, &other);
    return v + other;
}

__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& d) { return __umulhi(n, d.multiplier) + (n & d.whole); }

__device__ __forceinline__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(a), static_cast<__bf16>(b)}); }

// Two codes, in the low or the high half of a word, as two bf16.
template <bool kHigh>
__device__ __forceinline__ uint32_t two_e4m3(uint32_t codes) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, kHigh));
}
__device__ __forceinline__ float one_i8(uint32_t codes, int byte) { return static_cast<float>(static_cast<int8_t>(codes >> (8 * byte))); }

// Eight codes of a key as one operand's registers.
__device__ __forceinline__ bf16x8 operand_of(uint32_t low, uint32_t high) {
    return __builtin_bit_cast(bf16x8, u32x4{two_e4m3<false>(low), two_e4m3<true>(low), two_e4m3<false>(high), two_e4m3<true>(high)});
}

__device__ __forceinline__ f32x4 product(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// tanh to f32's last bits: the series up to x^11 where it is small (the next term is below 2e-8 of it), 1 - 2 / (e^2x + 1) else.
__device__ __forceinline__ float hyperbolic(float x) {
    const float z = x * x;
    const float small = x * __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -8.86323553e-3f, 2.18694885e-2f), -5.39682540e-2f), 1.33333333e-1f), -3.33333333e-1f), 1.0f);
    const float large = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(2.0f * kLog2e * __builtin_fabsf(x)) + 1.0f);
    return __builtin_fabsf(x) < 0.35f ? small : __builtin_copysignf(large, x);
}

// What a share of a request's keys holds for one row: the reference of its weights (in units of log2; minus infinity where it saw no
// key) and their sum.
struct Part {
    float most, sum;
};
__device__ __forceinline__ float exp2_between(float a, float b) { return a == b ? 1.0f : __builtin_amdgcn_exp2f(a - b); }

// What the lengths on the device say of one request.
struct Share {
    int begin, tokens, context;   // its first row of query, new and cached tokens
    int first_tile, tiles;        // tiles of keys that any of its new tokens sees
    uint32_t row_tiles, splits, each;  // workgroups' rows; parts of its keys, and tiles in a part
    uint32_t first, first_slot;   // number of its first workgroup, and of its first part
};
struct Plan {
    uint32_t row_tiles;  // of the largest request
    uint32_t target;     // workgroups that the tiles are shared out over, before each request's are rounded up; 0: one part a request
    uint32_t least;      // tiles of a part at least
    uint32_t slots;      // parts that there is room for
    uint32_t chunk;      // shares that lie on one XCD side by side
};

__device__ __forceinline__ Share lengths_of(const QuantizedAttentionArgs& a, uint32_t request, int rows_a_tile) {
    Share s{};
    s.begin = min(max(a.query_starts[request], 0), static_cast<int>(a.tokens));
    const int end = min(max(a.query_starts[request + 1], s.begin), static_cast<int>(a.tokens));
    s.tokens = min(end - s.begin, static_cast<int>(a.max_query_len));
    s.context = max(a.context_lens[request], 0);
    const unsigned long long most = min(static_cast<unsigned long long>(a.table_columns) * a.block_size.by, static_cast<unsigned long long>(a.max_key_len));
    const int keys = static_cast<int>(min(static_cast<unsigned long long>(s.context) + s.tokens, most));
    const int first = a.window != 0 && s.context >= static_cast<int>(a.window) ? s.context - static_cast<int>(a.window) + 1 : 0;
    s.first_tile = first / kTile;
    s.tiles = s.tokens > 0 && keys > first ? (keys - 1) / kTile - s.first_tile + 1 : 0;
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

// The request of workgroup `of` (or of request number `of`), and its share.  A part has the same number of tiles for all requests,
// evened out within a request.  Every wavefront works this out for itself, 64 requests at a time.
template <bool kByRequest>
__device__ __forceinline__ bool find_share(const QuantizedAttentionArgs& a, const Plan& plan, int rows_a_tile, uint32_t of, uint32_t* request, Share* out) {
    const uint32_t heads = a.cache.kv_heads;
    if (plan.target == 0) {
        const uint32_t r = kByRequest ? of : of / (heads * plan.row_tiles);
        if (r >= a.requests) return false;
        *request = r;
        *out = lengths_of(a, r, rows_a_tile);
        out->splits = 1;
        out->each = static_cast<uint32_t>(out->tiles);
        out->first = r * heads * plan.row_tiles;
        out->row_tiles = plan.row_tiles;  // (its numbering; rows past its own are empty)
        return true;
    }
    const int lane = static_cast<int>(threadIdx.x) & 63;
    Share mine{};
    float work = 0.0f;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 64) {
        if (r0 + lane < a.requests) {
            mine = lengths_of(a, r0 + lane, rows_a_tile);
            work += static_cast<float>(mine.tiles) * static_cast<float>(mine.row_tiles);
        }
    }
    work = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sum_up_to(work)), 63));
    // (a thousandth more than the quotient, for the floats' error: the parts are no more than plan.target and one a request)
    const float quotient = work * static_cast<float>(heads) * 1.001f / static_cast<float>(plan.target);
    const uint32_t tiles = max(static_cast<uint32_t>(fminf(quotient, 0x1p30f)) + 1, plan.least);
    uint32_t before = 0, slots_before = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 64) {
        uint32_t count = 0, slots = 0;
        mine.splits = 0;
        if (r0 + lane < a.requests) {
            if (a.requests > 64) mine = lengths_of(a, r0 + lane, rows_a_tile);
            mine.splits = mine.tiles > 0 ? (static_cast<uint32_t>(mine.tiles) + tiles - 1) / tiles : 1;
            mine.each = (static_cast<uint32_t>(mine.tiles) + mine.splits - 1) / mine.splits;
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
            out->first_tile = __builtin_amdgcn_readlane(mine.first_tile, l);
            out->tiles = __builtin_amdgcn_readlane(mine.tiles, l);
            out->row_tiles = __builtin_amdgcn_readlane(mine.row_tiles, l);
            out->splits = __builtin_amdgcn_readlane(mine.splits, l);
            out->each = __builtin_amdgcn_readlane(mine.each, l);
            out->first = __builtin_amdgcn_readlane(mine.first, l);
            out->first_slot = __builtin_amdgcn_readlane(mine.first_slot, l);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        slots_before += __builtin_amdgcn_readlane(slots_upto, 63);
    }
    return false;
}

__device__ __forceinline__ void store4(const QuantizedAttentionArgs& a, size_t token, uint32_t head, int d, f32x4 x, float total, bool saw) {
    const size_t to = token * a.out_token_stride + static_cast<size_t>(head) * a.out_head_stride + d;
    const float by = saw ? 1.0f / total : 0.0f;
    if (a.type == 0) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + to) = x * by;
    } else {
        uint32_t two[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float u = x[2 * i] * by, v = x[2 * i + 1] * by;
            if (a.type == 30) two[i] = pack(u, v);
            else two[i] = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(u))) | (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v))) << 16);
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + to) = uint2{two[0], two[1]};
    }
}

template <int kBytes>
struct Bytes;
template <>
struct Bytes<4> { typedef uint32_t type __attribute__((ext_vector_type(1))); };
template <>
struct Bytes<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <>
struct Bytes<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };

// 16 (4) bytes a lane from memory to 1 KiB (256 bytes) of LDS from `to` on (a uniform address), lane after lane; lanes that are off
// leave their bytes as they are.
__device__ __forceinline__ void load_to_lds(uint32_t to, const uint4* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds(uint32_t to, const float* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}
// The same of 16 bytes `past` bytes behind a uniform address.
__device__ __forceinline__ void load_to_lds(uint32_t to, const uint4* from, uint32_t past) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(past), "s"(from) : "memory", "m0");
}
// s_waitcnt for "at most kLeft vector memory operations outstanding" (nothing else waited for).
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLeft) : "memory");
}

// Where 16-byte piece `piece` of row `row` of a tile lies in LDS, in pieces.  The pieces of a row are in an order of its own, so that
// one piece of 16 rows falls on all banks (256 bytes of them).
template <int kDim>
__device__ __forceinline__ int piece_at(int row, int piece) {
    constexpr int kPieces = kDim / 16, kRowsOfBanks = 16 / kPieces;
    return row * kPieces + (piece ^ (row / kRowsOfBanks & (kPieces - 1)));
}

constexpr int kMostWaves = 8;
constexpr int stages_of(int dim) { return dim == 64 ? 4 : 2; }
constexpr int most_waves(int dim) { return dim == 256 ? 4 : kMostWaves; }
constexpr int sums_stride(int dim) { return dim + 4; }
constexpr int tile_bytes(int dim) { return kTile * dim * 2 + 2 * kTile * 4; }
// Of a wavefront: the ring of keys, values and their scales, and in its place, in the end, its sums.
constexpr int wave_lds(int dim, int rows) {
    const int ring = stages_of(dim) * tile_bytes(dim), sums = rows * (sums_stride(dim) * 4 + static_cast<int>(sizeof(Part)));
    return ((ring > sums ? ring : sums) + 1023) / 1024 * 1024;
}

// kDim: the head's values, rounded up to a size that is here (the rest are zeros).  kTerms: of the queries, 1 bf16, 2 f16, 3 f32.  kQ:
// sixteens of rows.
template <int kDim, bool kE4m3, int kTerms, int kQ>
__global__ __launch_bounds__(64 * most_waves(kDim)) void quantized_attention_kernel(QuantizedAttentionArgs a, Plan plan, float* part_out, Part* parts) {
    constexpr int kWeights = kTerms > 2 ? kTerms : 2, kSteps = kDim / 32, kVec = kDim / 16, kWords = kVec / 4, kPieces = kDim / 16, kRows = 16 * kQ;
    constexpr int kLoads = kTile * kPieces / 64, kRowsALoad = 64 / kPieces;  // of keys, and of values: 1 KiB each
    typedef typename Bytes<kVec>::type Value;
    constexpr int kStages = stages_of(kDim), kWaveLds = wave_lds(kDim, kRows);
    extern __shared__ __attribute__((aligned(1024))) char lds[];

    const uint32_t number = xcd_share(blockIdx.x, plan.chunk);
    uint32_t request;
    Share share;
    if (!find_share<false>(a, plan, kRows, number, &request, &share)) return;
    const uint32_t inside = number - share.first, row_tile = inside % share.row_tiles, kv_head = inside / share.row_tiles % a.cache.kv_heads;
    const uint32_t split = inside / share.row_tiles / a.cache.kv_heads, slot = share.first_slot + inside;
    const int group = static_cast<int>(a.group), rows = share.tokens * group, first_row = static_cast<int>(row_tile) * kRows;
    if (first_row >= rows || (share.splits > 1 && slot >= plan.slots)) return;
    const int here = min(kRows, rows - first_row);  // rows of this workgroup
    const int tid = static_cast<int>(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, waves = static_cast<int>(blockDim.x) >> 6;
    const int column = lane & 15, quarter = lane >> 4, head_dim = static_cast<int>(a.cache.head_dim);

    // ---- the keys of this part that any of these rows sees, and this wavefront's of them
    const int first_position = share.context + first_row / group, last_position = share.context + (first_row + here - 1) / group;
    const unsigned long long most = min(static_cast<unsigned long long>(a.table_columns) * a.block_size.by, static_cast<unsigned long long>(a.max_key_len));
    const int keys = static_cast<int>(min(static_cast<unsigned long long>(last_position) + 1, most));  // seen by none from here on
    const uint32_t limit = a.window != 0 ? a.window : 0x80000000u;                                      // a key is seen where position - key is below
    int tile = share.first_tile + static_cast<int>(split * share.each);
    int end = min(min(tile + static_cast<int>(share.each), share.first_tile + share.tiles), static_cast<int>((static_cast<uint32_t>(keys) + kTile - 1) / kTile));
    if (a.window != 0 && first_position >= static_cast<int>(a.window)) tile = max(tile, (first_position - static_cast<int>(a.window) + 1) / kTile);
    if (end > tile) {
        const int each = (end - tile + waves - 1) / waves;
        tile += wave * each;
        end = min(tile + each, end);
    }

    // 64 entries of the block table from `window_at` on, one a lane, and which of them name a block; the first are asked for before
    // the queries, whose way from memory nothing here waits for
    const int* table = a.block_tables + static_cast<size_t>(request) * a.table_columns;
    const uint32_t last_block = keys > 0 ? divide(static_cast<uint32_t>(keys - 1), a.block_size) : 0;
    uint32_t window = 0, window_at = 0, window_end = 0;  // (keys from window_end on are not in it)
    unsigned long long named = 0;
    const auto entries_from = [&](uint32_t first_key) {
        window_at = divide(first_key, a.block_size);
        window_end = (window_at + 64) * a.block_size.by;  // (below 2^32: a bound of the keys times the block size)
        return window_at + lane <= last_block ? static_cast<uint32_t>(table[window_at + lane]) : ~0u;
    };
    const auto keep = [&](uint32_t block) {
        named = __ballot(block < a.cache.blocks);
        window = block < a.cache.blocks ? block : 0;
    };
    const uint32_t first_entries = tile < end ? entries_from(static_cast<uint32_t>(tile) * kTile) : ~0u;

    // ---- the rows: their queries
    u32x4 raw[kQ][kSteps / 2][kTerms == 3 ? 4 : 2];
    int position[kQ];
    float slope[kQ];
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        const bool real = qt * 16 + column < here;
        const int row = first_row + (real ? qt * 16 + column : 0), token = row / group, head = static_cast<int>(kv_head) * group + row % group;
        position[qt] = real ? share.context + token : -1;  // (a row that is none sees nothing)
        slope[qt] = a.slopes != nullptr ? a.slopes[head] * kLog2e : 0.0f;
        const size_t from = static_cast<size_t>(share.begin + token) * a.query_token_stride + static_cast<size_t>(head) * a.query_head_stride;
#pragma unroll
        for (int b = 0; b < kSteps / 2; ++b) {
            const int d = 64 * b + 16 * quarter;
            const char* p = static_cast<const char*>(a.query) + (from + d) * (kTerms == 3 ? 4 : 2);
#pragma unroll
            for (int i = 0; i < (kTerms == 3 ? 4 : 2); ++i) raw[qt][b][i] = real && d < head_dim ? reinterpret_cast<const u32x4*>(p)[i] : u32x4{0, 0, 0, 0};
        }
    }

    char* const ring = lds + wave * kWaveLds;
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)ring)));
    // Where a lane's bytes of load i lie behind its first row's, where the rows of a load are in one block; whether there are any (the
    // ring holds zeros for what is past a head's end).
    const bool in_one = a.block_size.by % kRowsALoad == 0 && a.cache.slot_stride < (1u << 20);
    // (Loads that turn lanes off cost: 64 requests of 100 to 4000 keys take 75 us instead of 68 with them, so whole heads do without.
    // Every load has rows' first pieces, so that none is left out and the waits below count them all.)
    const bool whole_heads = head_dim == kDim;
    uint32_t lane_at[kLoads];
    bool has[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int row = i * kRowsALoad + lane / kPieces, piece = piece_at<kDim>(row, lane % kPieces) % kPieces;
        lane_at[i] = (static_cast<uint32_t>(lane / kPieces) * a.cache.slot_stride + piece) * 16;
        has[i] = piece * 16 < head_dim;
    }
    if (head_dim < kDim) {
        for (int i = lane; i < kWaveLds / 16; i += 64) reinterpret_cast<u32x4*>(ring)[i] = u32x4{0, 0, 0, 0};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    // Requests tile t into a stage; its keys that have a place are returned, in the order of the products' rows.  (A key without one
    // is not seen by any row: what is loaded for it, the first block's, may be anything.)
    auto request_tile = [&](int t, int stage) -> uint32_t {
        const uint32_t first_key = static_cast<uint32_t>(t) * kTile;
        if (first_key + kTile > window_end) {
            keep(entries_from(first_key));
        }
        const uint32_t to = ring_at + stage * tile_bytes(kDim);
        const uint32_t head_at = kv_head * a.cache.head_stride;
        if (in_one) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t key = first_key + i * kRowsALoad, column_of = divide(key, a.block_size);
                const uint32_t block = __builtin_amdgcn_readlane(window, column_of - window_at);
                const uint32_t place = block * a.cache.block_stride + (key - column_of * a.block_size.by) * a.cache.slot_stride + head_at;
                if (whole_heads) {
                    load_to_lds(to + i * 1024, a.cache.keys + place, lane_at[i]);
                    load_to_lds(to + kTile * kDim + i * 1024, a.cache.values + place, lane_at[i]);
                } else if (has[i]) {
                    load_to_lds(to + i * 1024, a.cache.keys + place, lane_at[i]);
                    load_to_lds(to + kTile * kDim + i * 1024, a.cache.values + place, lane_at[i]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int row = i * kRowsALoad + lane / kPieces, piece = piece_at<kDim>(row, lane % kPieces) % kPieces;
                const uint32_t key = first_key + row, column_of = divide(key, a.block_size);
                const uint32_t block = static_cast<uint32_t>(__shfl(static_cast<int>(window), static_cast<int>(column_of - window_at)));
                const uint32_t place = block * a.cache.block_stride + (key - column_of * a.block_size.by) * a.cache.slot_stride + head_at + piece;
                if (whole_heads) {
                    load_to_lds(to + i * 1024, a.cache.keys + place);
                    load_to_lds(to + kTile * kDim + i * 1024, a.cache.values + place);
                } else if (has[i]) {
                    load_to_lds(to + i * 1024, a.cache.keys + place);
                    load_to_lds(to + kTile * kDim + i * 1024, a.cache.values + place);
                }
            }
        }
        // the scales, keys' and then values'
        const uint32_t key = first_key + (lane & 16) + 4 * (lane & 3) + (lane >> 2 & 3), column_of = divide(key, a.block_size);
        const uint32_t block = static_cast<uint32_t>(__shfl(static_cast<int>(window), static_cast<int>(column_of - window_at)));
        const uint32_t place = block * a.cache.scale_block_stride + (key - column_of * a.block_size.by) * a.cache.scale_slot_stride + kv_head * a.cache.scale_head_stride;
        load_to_lds(to + 2 * kTile * kDim, (lane < 32 ? a.cache.key_scales : a.cache.value_scales) + place);
        return static_cast<uint32_t>(__ballot((named >> (column_of - window_at) & 1) != 0 && static_cast<int>(key) < keys));
    };
    keep(first_entries);
    uint32_t held[kStages] = {};  // of the tiles on their way, the next one's first
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) {
        const uint32_t got = tile + i < end ? request_tile(tile + i, i) : 0;
#pragma unroll
        for (int j = 0; j < kStages; ++j) held[j] = j == i ? got : held[j];
    }

    // What the products of a row are multiplied by, beside the keys' scales.
    const bool caps = a.softcap > 0.0f;
    const float unit = caps ? a.scale / a.softcap : a.scale * kLog2e, cap = a.softcap * kLog2e;
    float row_unit[kQ];
    bf16x8 query[kE4m3 ? kQ : 1][kE4m3 ? kSteps : 1][kTerms];
    i32x4 digits[kE4m3 ? 1 : kQ][kE4m3 ? 1 : kDim / 64][3];
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        row_unit[qt] = unit;
        float v[kE4m3 ? 1 : kDim / 4];
        uint32_t most_bits = 0;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float value;
                if (kTerms == 3) {
                    const uint32_t bits = raw[qt][s / 2][(s % 2) * 2 + j / 4][j % 4];  // (a bit_cast of the element itself reads the first)
                    value = __builtin_bit_cast(float, bits);
                } else {
                    const uint16_t bits = static_cast<uint16_t>(raw[qt][s / 2][s % 2][j / 2] >> (16 * (j % 2)));
                    value = kTerms == 1 ? static_cast<float>(__builtin_bit_cast(__bf16, bits)) : static_cast<float>(__builtin_bit_cast(_Float16, bits));
                }
                if constexpr (kE4m3) {
#pragma unroll
                    for (int term = 0; term < kTerms; ++term) {
                        query[qt][s][term][j] = static_cast<__bf16>(value);
                        value -= static_cast<float>(query[qt][s][term][j]);
                    }
                } else {
                    v[8 * s + j] = value;
                    most_bits = max(most_bits, __builtin_bit_cast(uint32_t, value) & 0x7FFFFFFFu);
                }
            }
        }
        if constexpr (!kE4m3) {
            // The row's largest value goes to [2^21, 2^22): whole numbers of three digits to the base 256, each an i8.
            most_bits = row_max_bits(most_bits);
            const int exponent = most_bits == 0 ? 0 : __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, most_bits)) - 22;
            row_unit[qt] = most_bits >= 0x7F800000u ? __builtin_nanf("") : unit * __builtin_amdgcn_ldexpf(1.0f, exponent);
#pragma unroll
            for (int b = 0; b < kDim / 64; ++b) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t words[3] = {0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int whole = static_cast<int>(__builtin_rintf(__builtin_amdgcn_ldexpf(v[16 * b + 4 * w + j], -exponent)));
                        const int high = (whole + 0x8080) >> 16, rest = whole - high * 65536, middle = (rest + 0x80) >> 8, low = rest - middle * 256;
                        words[0] |= (static_cast<uint32_t>(high) & 0xFF) << (8 * j);
                        words[1] |= (static_cast<uint32_t>(middle) & 0xFF) << (8 * j);
                        words[2] |= (static_cast<uint32_t>(low) & 0xFF) << (8 * j);
                    }
#pragma unroll
                    for (int digit = 0; digit < 3; ++digit) digits[qt][b][digit][w] = static_cast<int>(words[digit]);
                }
            }
        }
    }

    f32x4 out[kQ][kVec];
    float reference[kQ], sum[kQ];
    uint32_t saw[kQ];
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        reference[qt] = -__builtin_inff();
        sum[qt] = 0.0f;
        saw[qt] = 0;
#pragma unroll
        for (int t = 0; t < kVec; ++t) out[qt][t] = f32x4{0, 0, 0, 0};
    }

    int stage = 0;
    for (; tile < end; ++tile) {
        if (tile + kStages - 1 < end) wait_loads<(kStages - 1) * (2 * kLoads + 1)>();
        else wait_loads<0>();
        const char* const at = ring + stage * tile_bytes(kDim);
        const uint32_t there = held[0];
        // everything of the tile into registers
        u32x4 key[2][kDim / 64];
        Value value[8];
        f32x4 key_scale[2], value_scale[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int key_row = half * 16 + 4 * (column & 3) + (column >> 2);
#pragma unroll
            for (int b = 0; b < kDim / 64; ++b) key[half][b] = *reinterpret_cast<const u32x4*>(at + piece_at<kDim>(key_row, 4 * b + quarter) * 16);
            key_scale[half] = *reinterpret_cast<const f32x4*>(at + 2 * kTile * kDim + (half * 16 + quarter * 4) * 4);
            value_scale[half] = *reinterpret_cast<const f32x4*>(at + 2 * kTile * kDim + (32 + half * 16 + quarter * 4) * 4);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int row = j / 4 * 16 + j % 4 * 4 + quarter;
            value[j] = *reinterpret_cast<const Value*>(at + kTile * kDim + piece_at<kDim>(row, kVec * column / 16) * 16 + kVec * column % 16);
        }
#pragma unroll
        for (int i = 0; i + 1 < kStages; ++i) held[i] = held[i + 1];
        if (tile + kStages < end) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read
            held[kStages - 1] = request_tile(tile + kStages, stage);
        }
        stage = stage + 1 == kStages ? 0 : stage + 1;

        const int first_key = tile * kTile;
        // every row sees every key
        const bool clean = there == ~0u && first_key + kTile - 1 <= first_position && static_cast<uint32_t>(last_position - first_key) < limit;
        f32x4 score[kQ][2];
        if constexpr (kE4m3) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const u32x4 codes = key[half][s / 2];
                    const bf16x8 k = operand_of(codes[(s % 2) * 2], codes[(s % 2) * 2 + 1]);
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; --term) {  // the small terms first
#pragma unroll
                        for (int qt = 0; qt < kQ; ++qt)
                            score[qt][half] = product(k, query[qt][s][term], s == 0 && term == kTerms - 1 ? f32x4{0, 0, 0, 0} : score[qt][half]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int qt = 0; qt < kQ; ++qt) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    i32x4 whole[3];
#pragma unroll
                    for (int b = 0; b < kDim / 64; ++b) {
#pragma unroll
                        for (int digit = 0; digit < 3; ++digit)
                            whole[digit] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, key[half][b]), digits[qt][b][digit], b == 0 ? i32x4{0, 0, 0, 0} : whole[digit], 0, 0, 0);
                    }
                    // (a digit's sum is below 2^22: two of them fit 32 bits)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        score[qt][half][j] = __builtin_fmaf(static_cast<float>(whole[0][j]), 65536.0f, static_cast<float>(whole[1][j] * 256 + whole[2][j]));
                }
            }
        }
        uint32_t seen[kQ];
        bf16x8 weight[kQ][kWeights];
#pragma unroll
        for (int qt = 0; qt < kQ; ++qt) {
            float x[8], by[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = score[qt][j / 4][j % 4] * (key_scale[j / 4][j % 4] * row_unit[qt]);
                by[j] = value_scale[j / 4][j % 4];
            }
            if (caps) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = cap * hyperbolic(x[j]);
            }
            const int distance = position[qt] - first_key - quarter;  // to this lane's first key
            if (a.slopes != nullptr) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __builtin_fmaf(-slope[qt], static_cast<float>(distance - (j / 4 * 16 + j % 4 * 4)), x[j]);
            }
            seen[qt] = 0xFF;
            if (!clean) {
                // Whole numbers and selections, no branches: of a test by && the compiler (ROCm 7.2) made code that takes the weights of the
                // keys j = 0 that have no block but are near enough into the rows' sums (heads of up to 64, e4m3, the first sixteen of 32 rows).
                const uint32_t named = there >> (quarter * 4);
                seen[qt] = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t near_enough = static_cast<uint32_t>(distance - (j / 4 * 16 + j % 4 * 4)) < limit;
                    seen[qt] |= (near_enough & (named >> (j / 4 * 16 + j % 4))) << j;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool sees = (seen[qt] >> j & 1) != 0;
                    x[j] = sees ? x[j] : -__builtin_inff();
                    by[j] = sees ? by[j] : 0.0f;
                }
            }
            saw[qt] |= seen[qt];
            const float peak = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            if (__any(peak > reference[qt] + kSlack)) {
                const float highest = row_max(peak);
                if (highest > reference[qt] + kSlack) {  // each row by itself: no other row's keys move its bits
                    const float kept = reference[qt] == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(reference[qt] - highest);
                    reference[qt] = highest;
                    sum[qt] *= kept;
#pragma unroll
                    for (int t = 0; t < kVec; ++t) out[qt][t] *= kept;
                }
            }
            const float shift = reference[qt] == -__builtin_inff() ? 0.0f : reference[qt];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = __builtin_amdgcn_exp2f(x[j] - shift);
                sum[qt] += p;
                float rest = p * by[j];
#pragma unroll
                for (int term = 0; term < kWeights; ++term) {
                    weight[qt][term][j] = static_cast<__bf16>(rest);
                    rest -= static_cast<float>(weight[qt][term][j]);
                }
            }
        }
        // A row that does not see a value must not get 0 times no number from it: in tiles where some row may not see such codes they
        // are taken as zeros, and the rows that see them are made no numbers here.
        if (kE4m3 && !clean) {
            uint32_t any = 0;
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
#pragma unroll
                for (int j = 0; j < 8; ++j) any |= ((value[j][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;  // a byte's top bit: its code is no number
            }
            if (__any(any != 0)) {
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    uint32_t bad[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        bad[j] = (((value[j][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;  // 1 in such a byte
                        value[j][w] &= ~(bad[j] * 0xFFu);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        bf16x8 is;
#pragma unroll
                        for (int j = 0; j < 8; ++j) is[j] = static_cast<__bf16>(static_cast<float>(bad[j] >> (8 * i) & 1));
#pragma unroll
                        for (int qt = 0; qt < kQ; ++qt) {
                            bf16x8 sees;
#pragma unroll
                            for (int j = 0; j < 8; ++j) sees[j] = static_cast<__bf16>(static_cast<float>(seen[qt] >> j & 1));
                            const f32x4 count = product(is, sees, f32x4{0, 0, 0, 0});
#pragma unroll
                            for (int j = 0; j < 4; ++j) out[qt][4 * w + i][j] += count[j] > 0.0f ? __builtin_nanf("") : 0.0f;
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            uint32_t operand[4][4];  // [value of the word][pair of keys]
#pragma unroll
            for (int pair = 0; pair < 4; ++pair) {
                const uint32_t one = value[2 * pair][w], other = value[2 * pair + 1][w];
                if (kE4m3) {
                    const uint32_t low = __builtin_amdgcn_perm(other, one, 0x05010400u), high = __builtin_amdgcn_perm(other, one, 0x07030602u);
                    operand[0][pair] = two_e4m3<false>(low);
                    operand[1][pair] = two_e4m3<true>(low);
                    operand[2][pair] = two_e4m3<false>(high);
                    operand[3][pair] = two_e4m3<true>(high);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) operand[i][pair] = pack(one_i8(one, i), one_i8(other, i));
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bf16x8 v = __builtin_bit_cast(bf16x8, u32x4{operand[i][0], operand[i][1], operand[i][2], operand[i][3]});
#pragma unroll
                for (int term = kWeights - 1; term >= 0; --term) {
#pragma unroll
                    for (int qt = 0; qt < kQ; ++qt) out[qt][4 * w + i] = product(v, weight[qt][term], out[qt][4 * w + i]);
                }
            }
        }
    }

    // ---- the wavefronts' sums together, each in its ring's place: [row][values], and [row] behind them
    constexpr int kStride = sums_stride(kDim);
    const auto sums_of = [&](int w) { return reinterpret_cast<float*>(lds + w * kWaveLds); };
    const auto parts_of = [&](int w) { return reinterpret_cast<Part*>(lds + w * kWaveLds + kRows * kStride * 4); };
#pragma unroll
    for (int qt = 0; qt < kQ; ++qt) {
        const float total = row_sum(sum[qt]);
        const bool row_saw = row_max(saw[qt] != 0 ? 1.0f : 0.0f) > 0.0f;
        const int r = qt * 16 + column;
        if (r >= here) continue;
        float* to = sums_of(wave) + r * kStride;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int w = 0; w < kWords; ++w)
                *reinterpret_cast<f32x4*>(to + kVec * (4 * quarter + i) + 4 * w) = f32x4{out[qt][4 * w][i], out[qt][4 * w + 1][i], out[qt][4 * w + 2][i], out[qt][4 * w + 3][i]};
        }
        if (quarter == 0) parts_of(wave)[r] = Part{!row_saw ? -__builtin_inff() : reference[qt] == -__builtin_inff() ? kLowest : reference[qt], total};
    }
    __syncthreads();
    for (int item = tid; item < here * (kDim / 4); item += static_cast<int>(blockDim.x)) {
        const int r = item / (kDim / 4), d = item % (kDim / 4) * 4;
        if (d >= head_dim) continue;
        float highest = -__builtin_inff();
        for (int w = 0; w < waves; ++w) highest = fmaxf(highest, parts_of(w)[r].most);
        f32x4 x{0, 0, 0, 0};
        float all = 0.0f;
        for (int w = 0; w < waves; ++w) {
            const Part part = parts_of(w)[r];
            if (part.most == -__builtin_inff()) continue;
            const float by = exp2_between(part.most, highest);
            all = __builtin_fmaf(part.sum, by, all);
            const f32x4 y = *reinterpret_cast<const f32x4*>(sums_of(w) + r * kStride + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(y[j], by, x[j]);
        }
        if (share.splits > 1) {
            *reinterpret_cast<f32x4*>(part_out + (static_cast<size_t>(slot) * kRows + r) * a.cache.head_dim + d) = x;
            if (d == 0) parts[static_cast<size_t>(slot) * kRows + r] = Part{highest, all};
        } else {
            const int whole = first_row + r;
            store4(a, static_cast<size_t>(share.begin + whole / group), kv_head * a.group + static_cast<uint32_t>(whole % group), d, x, all, highest != -__builtin_inff());
        }
    }
}

// Of a few parts a wavefront has a row, of more a workgroup: their weights first, then every group of lanes has parts in turn, a lane
// four values.  The first parts' sums are asked for before their weights are known: one way to memory instead of two (64 parts of 56
// rows 5.5 us instead of 7.3; 16 parts or so of 16 x 140 rows 5.6 us by wavefronts, 11.2 by workgroups).
constexpr uint32_t kMostParts = 1100;  // of a request: plan.target is 1024 at most
constexpr uint32_t kFewParts = 32;
__global__ __launch_bounds__(256) void join_quantized_parts_kernel(QuantizedAttentionArgs a, Plan plan, int rows_a_tile, const float* part_out, const Part* parts) {
    __shared__ float by[kMostParts];
    __shared__ float numbers[8];
    __shared__ f32x4 sums[256];
    uint32_t request;
    Share share;
    if (!find_share<true>(a, plan, rows_a_tile, blockIdx.y, &request, &share) || share.splits <= 1) return;
    const uint32_t heads = a.cache.kv_heads, fours = a.cache.head_dim / 4, lanes = fours <= 16 ? 16 : fours <= 32 ? 32 : 64, groups = 256 / lanes;
    const uint32_t tid = threadIdx.x, rows = static_cast<uint32_t>(share.tokens) * a.group, splits = min(share.splits, kMostParts);
    // (starts that fall, which no batch has, could count rows twice and ask for more parts than there is room for)
    if (share.first_slot + static_cast<uint64_t>(share.row_tiles) * splits * heads > plan.slots) return;
    const uint32_t lane = tid % lanes;
    constexpr uint32_t kAhead = 8;
    f32x4 ahead[kAhead], x;
    // (also of a part without weight: a value that is no number shows whichever part has it; parts that saw nothing hold zeros)
    const auto take = [&](f32x4 y, float w) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(y[j], w, x[j]);
    };
    const auto put = [&](uint32_t kv_head, uint32_t row, float all, float highest) {
        store4(a, static_cast<size_t>(share.begin) + row / a.group, kv_head * a.group + row % a.group, static_cast<int>(4 * lane), x, all, highest != -__builtin_inff());
    };
    const auto first_part = [&](uint32_t kv_head, uint32_t row) {
        return (share.first_slot + static_cast<size_t>(kv_head) * share.row_tiles + row / rows_a_tile) * rows_a_tile + row % rows_a_tile;
    };
    const size_t apart = static_cast<size_t>(heads) * share.row_tiles * rows_a_tile;
    if (splits <= kFewParts) {
        const uint32_t at = tid & 63, first = at / lanes, in_wave = 64 / lanes;
        for (uint32_t number = blockIdx.x * 4 + (tid >> 6); number < rows * heads; number += gridDim.x * 4) {
            const uint32_t kv_head = number / rows, row = number % rows;
            const size_t part = first_part(kv_head, row);
            const auto sums_at = [&](uint32_t s) {
                return lane < fours && s < splits ? *reinterpret_cast<const f32x4*>(part_out + (part + s * apart) * a.cache.head_dim + 4 * lane) : f32x4{0, 0, 0, 0};
            };
            const Part own = at < splits ? parts[part + at * apart] : Part{-__builtin_inff(), 0.0f};
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) ahead[i] = sums_at(first + i * in_wave);
            float highest = own.most;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) highest = fmaxf(highest, __shfl_xor(highest, d));
            const float weight = own.most == -__builtin_inff() ? 0.0f : exp2_between(own.most, highest);
            float all = own.sum * weight;  // (a part that saw nothing has a sum of zero)
#pragma unroll
            for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
            x = f32x4{0, 0, 0, 0};
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) take(ahead[i], __shfl(weight, static_cast<int>(first + i * in_wave)));  // (below 64; zero from `splits` on)
            for (uint32_t s = first + kAhead * in_wave; s - first < splits; s += in_wave) take(sums_at(s), __shfl(weight, static_cast<int>(s)));
            for (uint32_t d = lanes; d < 64; d *= 2) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float v = x[j];
                    x[j] = v + __shfl_xor(v, static_cast<int>(d));
                }
            }
            if (at < fours) put(kv_head, row, all, highest);
        }
        return;
    }
    for (uint32_t number = blockIdx.x; number < rows * heads; number += gridDim.x) {
        const uint32_t kv_head = number / rows, row = number % rows, first = tid / lanes;
        const size_t part = first_part(kv_head, row);
        const auto part_at = [&](uint32_t s) { return part + s * apart; };
        const auto sums_at = [&](uint32_t s) { return *reinterpret_cast<const f32x4*>(part_out + part_at(s) * a.cache.head_dim + 4 * lane); };
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) ahead[i] = lane < fours && first + i * groups < splits ? sums_at(first + i * groups) : f32x4{0, 0, 0, 0};
        constexpr uint32_t kOwn = (kMostParts + 255) / 256;
        Part own[kOwn];
        float highest = -__builtin_inff(), all = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) own[i] = tid + i * 256 < splits ? parts[part_at(tid + i * 256)] : Part{-__builtin_inff(), 0.0f};
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) highest = fmaxf(highest, own[i].most);
#pragma unroll
        for (int d = 1; d < 64; d *= 2) highest = fmaxf(highest, __shfl_xor(highest, d));
        if ((tid & 63) == 0) numbers[tid >> 6] = highest;
        __syncthreads();
        highest = fmaxf(fmaxf(numbers[0], numbers[1]), fmaxf(numbers[2], numbers[3]));
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
            const float w = own[i].most == -__builtin_inff() ? 0.0f : exp2_between(own[i].most, highest);
            if (tid + i * 256 < splits) by[tid + i * 256] = w;
            all = __builtin_fmaf(own[i].sum, w, all);  // (a part that saw nothing has a sum of zero)
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
        if ((tid & 63) == 0) numbers[4 + (tid >> 6)] = all;
        __syncthreads();
        all = (numbers[4] + numbers[5]) + (numbers[6] + numbers[7]);
        x = f32x4{0, 0, 0, 0};
        if (lane < fours) {
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) take(ahead[i], first + i * groups < splits ? by[first + i * groups] : 0.0f);
#pragma unroll 4
            for (uint32_t s = first + kAhead * groups; s < splits; s += groups) take(sums_at(s), by[s]);
        }
        sums[tid] = x;
        __syncthreads();
        if (tid < fours) {
            for (uint32_t g = 1; g < groups; ++g) x += sums[g * lanes + tid];
            put(kv_head, row, all, highest);
        }
        __syncthreads();
    }
}

struct Shape {
    int dim, sixteens, waves;
    Plan plan;
    uint64_t groups, join_groups;
    int rows_a_tile() const { return 16 * sixteens; }
};

constexpr uint32_t kMostShared = 1024;  // requests: every wavefront reads their lengths, 64 at a time

Shape shape_of(const QuantizedAttentionArgs& a, int compute_units) {
    Shape s;
    s.dim = a.cache.head_dim <= 64 ? 64 : a.cache.head_dim <= 128 ? 128 : 256;
    s.waves = 4;
    const uint64_t rows = static_cast<uint64_t>(a.max_query_len) * a.group;
    // In 32 rows a key is read once for twice as many; with no more than sixteen of them half the products are idle (16 requests of 4 tokens, 4
    // heads a key head, on 1000 keys: 16.8 us in sixteens, 20.7 in 32 rows; of 8 tokens on 500 keys 13.2 and 17.4; of 3 to 7 tokens, 5 heads, on 300
    // to 9000 keys 43.1 and 42.7).
    s.sixteens = rows <= 16 || s.dim == 256 ? 1 : 2;
    const uint64_t tile_rows = s.rows_a_tile(), most_row_tiles = (rows + tile_rows - 1) / tile_rows;
    uint64_t row_tiles = static_cast<uint64_t>(a.tokens) * a.group / tile_rows + a.requests;  // of the batch: a request's last may be part empty
    if (row_tiles > a.requests * most_row_tiles) row_tiles = a.requests * most_row_tiles;
    const uint64_t base = row_tiles * a.cache.kv_heads;
    uint64_t keys = a.max_key_len;
    if (a.window != 0 && keys > static_cast<uint64_t>(a.window) + a.max_query_len) keys = static_cast<uint64_t>(a.window) + a.max_query_len;
    const uint64_t tiles = keys / kTile + 2;
    s.plan.row_tiles = static_cast<uint32_t>(most_row_tiles);
    s.plan.least = 8;  // (of 4, 8 and 16: 1 request of 4000 keys and 8 key heads 15.0, 13.4 and 15.9 us, of 1000 12.0, 13.2 and 15.8; 8 of 6 tokens on 1000 24, 19 and 22)
    s.plan.target = 0;
    // Contexts are shared out where row tiles would leave units idle, or where long ones of few requests would be waited for.  In one part
    // and shared out (heads of 128, 8 key heads and 1 token where no others are named, bf16 on whole numbers): 2 requests of 700 keys
    // 12.8 and 13.2 us, of 900 14.9 and 13.1; 16 of 500 to 900 keys and 4 key heads 14.7 and 13.5; 8 of 4 to 8 tokens on 500 to 1000 keys 21.5
    // and 19.7; 30 of 2500 keys 38 and 43, of 4000 55 and 58; 64 of 100 to 3000 keys 52 and 51, of 100 to 8000 152 and 128; 100 of 300 to 3000
    // keys 90 and 87, of 300 to 5500 159 and 148; 200 of 500 to 8000 keys in random order 368 and 381, in rising order 386 and 372.
    //
    // Workgroups that keys are shared out over, one, two, four and eight a unit: 2 requests of 131000 keys and 4 key heads
    // 56, 61, 62 and 71 us; 30 requests of 3000 to 9000 keys 120, 101, 90 and 90; 16 of 300 to 9000 keys and 4 key heads 43, 31, 31 and 36: two with few
    // requests and heads, four with many and enough tiles, whose unequal work evens out (16 tiles a unit; 30 requests of 4000 keys and
    // 2 key heads 25 us with four, 30 with two; 16 of 1000 keys and 4 16.2 and 13.6).  Then, below half as many heads as units, wavefronts in
    // pairs, since a part has few tiles for each (alone, in pairs, in fours: 16 requests of 3 to 7 tokens on 300 to 9000 keys, 4 key heads,
    // 54, 43 and 49 us without a window; 30 of 3000 to 9000 keys, 8 key heads, 105, 98 and 89; 2 of 131000, 4 key heads, 87, 65 and 60).
    // Of heads of 256 a unit's LDS holds four wavefronts: as two pairs (2 requests of 60000 to 90000 keys 69 us, in fours 75).
    const uint64_t units = static_cast<uint64_t>(compute_units < 256 ? compute_units : 256), pairs = static_cast<uint64_t>(a.requests) * a.cache.kv_heads;
    const uint64_t enough = base < units / 2 ? 24 : base < 2 * units ? 100 : 160;  // tiles of the longest context
    if (a.requests <= kMostShared && base < 4 * units && tiles > enough) {
        const bool many = pairs >= units / 8 && base * tiles >= 16 * units;
        s.plan.target = static_cast<uint32_t>(many ? 4 * units : 2 * units);
        if (s.dim == 256 || (many && pairs < units / 2)) s.waves = 2;
    } else if (base < units) {
        s.waves = most_waves(s.dim);
    }
    s.groups = s.plan.target == 0 ? a.requests * most_row_tiles * a.cache.kv_heads : base + s.plan.target;
    s.plan.slots = s.plan.target == 0 ? 0 : static_cast<uint32_t>(s.groups);
    const uint64_t chunk = xcd_chunk(most_row_tiles, a.cache.kv_heads, s.groups);
    s.plan.chunk = static_cast<uint32_t>(chunk);
    s.groups = (s.groups + 8 * chunk - 1) / (8 * chunk) * (8 * chunk);
    s.join_groups = rows * a.cache.kv_heads;
    // Mostly few parts: a workgroup has four rows, one a wavefront (8 requests of 6 tokens on 3000 keys 31.3 us, with four times the workgroups
    // 32.3).  Of many parts a row is a workgroup's (1 request of 60000 keys 37 us, 45 with a quarter of them; of 1 key head 23 and 52).
    if (base * 16 >= s.plan.target) s.join_groups = (s.join_groups + 3) / 4;
    if (s.join_groups > 4096) s.join_groups = 4096;
    return s;
}

size_t part_out_bytes(const QuantizedAttentionArgs& a, const Shape& s) {
    return (static_cast<size_t>(s.plan.slots) * s.rows_a_tile() * a.cache.head_dim * sizeof(float) + 255) / 256 * 256;
}

template <int kDim, bool kE4m3, int kTerms, int kQ>
hipError_t attend(hipStream_t stream, const QuantizedAttentionArgs& a, const Shape& s, void* workspace) {
    static LdsLimit limit;
    static_assert(most_waves(kDim) * wave_lds(kDim, 16 * kQ) <= 160 * 1024, "a compute unit's LDS");
    const size_t lds = static_cast<size_t>(s.waves) * wave_lds(kDim, 16 * kQ);
    const auto kernel = quantized_attention_kernel<kDim, kE4m3, kTerms, kQ>;
    hipError_t e = allow_lds(kernel, lds, &limit);
    if (e != hipSuccess) return e;
    float* part_out = static_cast<float*>(workspace);
    Part* parts = s.plan.slots != 0 ? reinterpret_cast<Part*>(static_cast<char*>(workspace) + part_out_bytes(a, s)) : nullptr;
    kernel<<<static_cast<uint32_t>(s.groups), 64 * s.waves, lds, stream>>>(a, s.plan, part_out, parts);
    e = hipGetLastError();
    if (e != hipSuccess || s.plan.slots == 0) return e;
    join_quantized_parts_kernel<<<dim3(static_cast<uint32_t>(s.join_groups), a.requests), 256, 0, stream>>>(a, s.plan, s.rows_a_tile(), part_out, parts);
    return hipGetLastError();
}

template <int kDim, bool kE4m3, int kTerms>
hipError_t attend_rows(hipStream_t stream, const QuantizedAttentionArgs& a, const Shape& s, void* workspace) {
    if constexpr (kDim != 256) {
        if (s.sixteens == 2) return attend<kDim, kE4m3, kTerms, 2>(stream, a, s, workspace);
    }
    return attend<kDim, kE4m3, kTerms, 1>(stream, a, s, workspace);
}

template <int kDim, bool kE4m3>
hipError_t attend_types(hipStream_t stream, const QuantizedAttentionArgs& a, const Shape& s, void* workspace) {
    if (a.type == 0) return attend_rows<kDim, kE4m3, 3>(stream, a, s, workspace);
    if (a.type == 1) return attend_rows<kDim, kE4m3, 2>(stream, a, s, workspace);
    return attend_rows<kDim, kE4m3, 1>(stream, a, s, workspace);
}

}  // namespace

size_t quantized_attention_workspace_bytes(const QuantizedAttentionArgs& args, int compute_units) {
    const Shape s = shape_of(args, compute_units);
    return s.plan.slots == 0 ? 0 : part_out_bytes(args, s) + static_cast<size_t>(s.plan.slots) * s.rows_a_tile() * sizeof(Part);
}

bool quantized_attention_fits_a_launch(const QuantizedAttentionArgs& args, int compute_units) {
    const Shape s = shape_of(args, compute_units);
    return fits_a_launch(s.groups, 64 * static_cast<uint64_t>(s.waves));
}

hipError_t launch_quantized_attention(hipStream_t stream, const QuantizedAttentionArgs& args, void* workspace, int compute_units) {
    const Shape s = shape_of(args, compute_units);
    if (s.dim == 64) return args.cache.e4m3 ? attend_types<64, true>(stream, args, s, workspace) : attend_types<64, false>(stream, args, s, workspace);
    if (s.dim == 128) return args.cache.e4m3 ? attend_types<128, true>(stream, args, s, workspace) : attend_types<128, false>(stream, args, s, workspace);
    return args.cache.e4m3 ? attend_types<256, true>(stream, args, s, workspace) : attend_types<256, false>(stream, args, s, workspace);
}

}  // namespace afhip
