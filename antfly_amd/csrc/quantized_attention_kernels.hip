// Attention of a batch's new tokens over an 8-bit paged key / value cache.
//
//   out[t][h] = sum_j p_j u_j v_j / sum_j p_j,   p_j = exp(s_j - m),   s_j from scale * k_scale_j * (q . k_j),   u_j the value's scale
//
// One pass over the keys with a running reference m and sum of the softmax.  The rows of one key head are its query heads' tokens
// packed together (row = token * group + head in group), sixteen to a wavefront, so a key is read once for all of them.
//
// The products are on the 16 x 16 x 32 bf16 matrix instructions with the keys as the first operand: K Q^T has one row of the packed
// queries to a lane (column = lane % 16) and four consecutive keys in its registers, and these are, after the softmax, the second
// operand of V^T P^T as they stand.  Codes go from memory into registers and to bf16 there, which holds every one of them exactly: 16
// bytes a lane of a key, and of a value one, two or four dwords of eight keys, whose bytes are put side by side key by key before
// the conversion (the order of the head's values over lanes and products is free: value kVec * column + t is in product t).  So
// nothing is staged in LDS but a tile's places and scales, which lie one key a lane as they arrive and are needed four a lane.
// F32 queries and the weights beside them are three terms of bf16, f16 two, each a product of its own.
//
// A wavefront steps over tiles of 32 keys, the next one's codes requested before it works on one, the block table a tile before
// that.  Wavefronts of a workgroup take tiles in turn and add up in LDS; long contexts are shared out over workgroups by the
// lengths that the device holds, and a second kernel joins the parts.
#include "quantized_launch.h"

#include <hip/hip_runtime.h>

namespace afhip {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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
template <bool kE4m3>
__device__ __forceinline__ bf16x8 operand_of(uint32_t low, uint32_t high) {
    u32x4 r;
    if (kE4m3) r = u32x4{two_e4m3<false>(low), two_e4m3<true>(low), two_e4m3<false>(high), two_e4m3<true>(high)};
    else r = u32x4{pack(one_i8(low, 0), one_i8(low, 1)), pack(one_i8(low, 2), one_i8(low, 3)), pack(one_i8(high, 0), one_i8(high, 1)), pack(one_i8(high, 2), one_i8(high, 3))};
    return __builtin_bit_cast(bf16x8, r);
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
};

__device__ __forceinline__ Share lengths_of(const QuantizedAttentionArgs& a, uint32_t request) {
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
    s.row_tiles = (static_cast<uint32_t>(s.tokens) * a.group + 15) / 16;
    return s;
}

template <typename T>
__device__ __forceinline__ T sum_up_to(T v) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const T below = __shfl_up(v, d);
        if (lane >= d) v += below;
    }
    return v;
}

// The request of workgroup `of` (or of request number `of`), and its share.  A part has the same number of tiles for all requests,
// evened out within a request.  Every wavefront works this out for itself, 64 requests at a time.
template <bool kByRequest>
__device__ __forceinline__ bool find_share(const QuantizedAttentionArgs& a, const Plan& plan, uint32_t of, uint32_t* request, Share* out) {
    const uint32_t heads = a.cache.kv_heads;
    if (plan.target == 0) {
        const uint32_t r = kByRequest ? of : of / (heads * plan.row_tiles);
        if (r >= a.requests) return false;
        *request = r;
        *out = lengths_of(a, r);
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
            mine = lengths_of(a, r0 + lane);
            work += static_cast<float>(mine.tiles) * static_cast<float>(mine.row_tiles);
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) work += __shfl_xor(work, d);
    // (a thousandth more than the quotient, for the floats' error: the parts are no more than plan.target and one a request)
    const float quotient = work * static_cast<float>(heads) * 1.001f / static_cast<float>(plan.target);
    const uint32_t tiles = max(static_cast<uint32_t>(fminf(quotient, 0x1p30f)) + 1, plan.least);
    uint32_t before = 0, slots_before = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 64) {
        uint32_t count = 0, slots = 0;
        mine.splits = 0;
        if (r0 + lane < a.requests) {
            if (a.requests > 64) mine = lengths_of(a, r0 + lane);
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

// A tile on its way: its codes, and what one lane holds of its keys (lanes 0 to 31 keys' scales, 32 to 63 values').
template <int kDim>
struct Tile {
    typedef typename Bytes<kDim / 16>::type Value;
    u32x4 key[2][kDim / 64];
    Value value[8];
    float scale;
    uint32_t held;  // its keys that have a place
};

constexpr int kMostWaves = 8;
constexpr int kWaveLds = 3 * kTile * 4;  // of a wavefront: its tile's places and scales
constexpr int waves_of(int dim) { return dim == 256 ? 4 : kMostWaves; }

// kDim: the head's values, rounded up to a size that is here (the rest are zeros).  kTerms: 1 bf16, 2 f16, 3 f32 queries.
template <int kDim, bool kE4m3, int kTerms>
__global__ __launch_bounds__(64 * waves_of(kDim)) void quantized_attention_kernel(QuantizedAttentionArgs a, Plan plan, float* part_out, Part* parts) {
    constexpr int kSteps = kDim / 32, kVec = kDim / 16, kWords = kVec / 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint32_t(*const place_of)[kTile] = reinterpret_cast<uint32_t(*)[kTile]>(lds);  // [wave][key]
    float(*const scale_of)[2 * kTile] = reinterpret_cast<float(*)[2 * kTile]>(lds + (blockDim.x >> 6) * (kTile * 4));

    const uint32_t number = ((blockIdx.x >> 3) / plan.row_tiles * 8 + (blockIdx.x & 7)) * plan.row_tiles + (blockIdx.x >> 3) % plan.row_tiles;
    uint32_t request;
    Share share;
    if (!find_share<false>(a, plan, number, &request, &share)) return;
    const uint32_t inside = number - share.first, row_tile = inside % share.row_tiles, split = inside / share.row_tiles % share.splits;
    const uint32_t kv_head = inside / share.row_tiles / share.splits, slot = share.first_slot + inside;
    const int group = static_cast<int>(a.group), rows = share.tokens * group, first_row = static_cast<int>(row_tile) * 16;
    if (first_row >= rows || (share.splits > 1 && slot >= plan.slots)) return;
    const int here = min(16, rows - first_row);  // rows of this workgroup
    const int tid = static_cast<int>(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, waves = static_cast<int>(blockDim.x) >> 6;
    const int column = lane & 15, quarter = lane >> 4;

    // ---- the rows: their queries, requested first
    const bool real = column < here;
    const int row = first_row + (real ? column : 0), token = row / group, head = static_cast<int>(kv_head) * group + row % group;
    const int position = real ? share.context + token : -1;  // (a row that is none sees nothing)
    u32x4 raw[kSteps / 2][kTerms == 3 ? 4 : 2];
    {
        const size_t from = static_cast<size_t>(share.begin + token) * a.query_token_stride + static_cast<size_t>(head) * a.query_head_stride;
#pragma unroll
        for (int b = 0; b < kSteps / 2; ++b) {
            const int d = 64 * b + 16 * quarter;
            const char* p = static_cast<const char*>(a.query) + (from + d) * (kTerms == 3 ? 4 : 2);
#pragma unroll
            for (int i = 0; i < (kTerms == 3 ? 4 : 2); ++i) raw[b][i] = real && d < static_cast<int>(a.cache.head_dim) ? reinterpret_cast<const u32x4*>(p)[i] : u32x4{0, 0, 0, 0};
        }
    }
    const float slope = a.slopes != nullptr ? a.slopes[head] * kLog2e : 0.0f;

    // ---- the keys of this part that any of these rows sees
    const int first_position = share.context + first_row / group, last_position = share.context + (first_row + here - 1) / group;
    const unsigned long long most = min(static_cast<unsigned long long>(a.table_columns) * a.block_size.by, static_cast<unsigned long long>(a.max_key_len));
    const int keys = static_cast<int>(min(static_cast<unsigned long long>(last_position) + 1, most));  // seen by none from here on
    const uint32_t limit = a.window != 0 ? a.window : 0x80000000u;                                      // a key is seen where position - key is below
    int tile = share.first_tile + static_cast<int>(split * share.each);
    const int end = min(min(tile + static_cast<int>(share.each), share.first_tile + share.tiles), (keys + kTile - 1) / kTile);
    if (a.window != 0 && first_position >= static_cast<int>(a.window)) tile = max(tile, (first_position - static_cast<int>(a.window) + 1) / kTile);
    tile += wave;

    const int* table = a.block_tables + static_cast<size_t>(request) * a.table_columns;
    const uint32_t mine = lane & 31;
    uint32_t entry = ~0u;  // the block of this lane's key, of the next tile to be requested
    auto find = [&](int t) {
        const uint32_t key = static_cast<uint32_t>(t) * kTile + mine;
        entry = static_cast<int>(key) < keys ? static_cast<uint32_t>(table[divide(key, a.block_size)]) : ~0u;
    };
    auto request_tile = [&](int t, Tile<kDim>& to) {
        const uint32_t key = static_cast<uint32_t>(t) * kTile + mine;
        const uint32_t past = key - divide(key, a.block_size) * a.block_size.by;
        const bool there = entry < a.cache.blocks;
        to.held = static_cast<uint32_t>(__ballot(there));
        // (a key without a place is not seen by any row: what is loaded for it, the cache's first, may be anything)
        const uint32_t block = there ? entry : 0, within = there ? past : 0;
        const uint32_t place = block * a.cache.block_stride + within * a.cache.slot_stride + kv_head * a.cache.head_stride;
        const uint32_t scale_at = block * a.cache.scale_block_stride + within * a.cache.scale_slot_stride + kv_head * a.cache.scale_head_stride;
        to.scale = (lane < 32 ? a.cache.key_scales : a.cache.value_scales)[scale_at];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lane < 32) place_of[wave][mine] = place;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint4* from = a.cache.keys + place_of[wave][half * 16 + column];
#pragma unroll
            for (int b = 0; b < kDim / 64; ++b) {
                if (64 * b + 16 * quarter < static_cast<int>(a.cache.head_dim)) to.key[half][b] = *reinterpret_cast<const u32x4*>(from + 4 * b + quarter);
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const u32x4 places = *reinterpret_cast<const u32x4*>(&place_of[wave][half * 16 + quarter * 4]);
            if (kVec * column < static_cast<int>(a.cache.head_dim)) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    to.value[half * 4 + j] = *reinterpret_cast<const typename Tile<kDim>::Value*>(reinterpret_cast<const char*>(a.cache.values + places[j]) + kVec * column);
            }
        }
    };

    Tile<kDim> ping, pong;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int b = 0; b < kDim / 64; ++b) ping.key[half][b] = pong.key[half][b] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ping.value[j] = pong.value[j] = typename Tile<kDim>::Value(0u);
    if (tile < end) {
        find(tile);
        request_tile(tile, ping);
        if (tile + waves < end) find(tile + waves);
    }

    bf16x8 query[kSteps][kTerms];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (kTerms == 3) {
                const uint32_t bits = raw[s / 2][(s % 2) * 2 + j / 4][j % 4];  // (a bit_cast of the element itself reads the first)
                float rest = __builtin_bit_cast(float, bits);
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    query[s][term][j] = static_cast<__bf16>(rest);
                    rest -= static_cast<float>(query[s][term][j]);
                }
            } else {
                const uint16_t bits = static_cast<uint16_t>(raw[s / 2][s % 2][j / 2] >> (16 * (j % 2)));
                if (kTerms == 1) {
                    query[s][0][j] = __builtin_bit_cast(__bf16, bits);
                } else {
                    const float v = static_cast<float>(__builtin_bit_cast(_Float16, bits));
                    query[s][0][j] = static_cast<__bf16>(v);
                    query[s][kTerms - 1][j] = static_cast<__bf16>(v - static_cast<float>(query[s][0][j]));
                }
            }
        }
    }

    const bool caps = a.softcap > 0.0f;
    const float unit = caps ? a.scale / a.softcap : a.scale * kLog2e, cap = a.softcap * kLog2e;
    f32x4 out[kVec];
#pragma unroll
    for (int t = 0; t < kVec; ++t) out[t] = f32x4{0, 0, 0, 0};
    float reference = -__builtin_inff(), sum = 0.0f;
    bool saw = false;

    auto work = [&](int t, Tile<kDim>& at) {
        const int first_key = t * kTile;
        // every row sees every key
        const bool clean = at.held == ~0u && first_key + kTile - 1 <= first_position && static_cast<uint32_t>(last_position - first_key) < limit;
        scale_of[wave][lane] = at.scale;
        f32x4 score[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const u32x4 codes = at.key[half][s / 2];
                const bf16x8 key = operand_of<kE4m3>(codes[(s % 2) * 2], codes[(s % 2) * 2 + 1]);
#pragma unroll
                for (int term = kTerms - 1; term >= 0; --term) score[half] = product(key, query[s][term], score[half]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float x[8], value_scale[8];
        uint32_t seen = 0xFF;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const f32x4 k = *reinterpret_cast<const f32x4*>(&scale_of[wave][half * 16 + quarter * 4]);
            const f32x4 v = *reinterpret_cast<const f32x4*>(&scale_of[wave][32 + half * 16 + quarter * 4]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[half * 4 + j] = score[half][j] * (k[j] * unit);
                value_scale[half * 4 + j] = v[j];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (caps) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = cap * hyperbolic(x[j]);
        }
        const int my_key = first_key + quarter * 4;
        if (a.slopes != nullptr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __builtin_fmaf(-slope, static_cast<float>(position - my_key - (j / 4 * 16 + j % 4)), x[j]);
        }
        if (!clean) {
            seen = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = j / 4 * 16 + j % 4;
                const bool sees = static_cast<uint32_t>(position - my_key - key) < limit && (at.held >> (quarter * 4 + key) & 1) != 0;
                seen |= static_cast<uint32_t>(sees) << j;
                if (!sees) x[j] = -__builtin_inff();
            }
        }
        saw |= seen != 0;
        const float peak = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if (__any(peak > reference + kSlack)) {
            const float highest = row_max(peak);
            if (highest > reference + kSlack) {  // each row by itself: no other row's keys move its bits
                const float by = reference == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(reference - highest);
                reference = highest;
                sum *= by;
#pragma unroll
                for (int t = 0; t < kVec; ++t) out[t] *= by;
            }
        }
        const float shift = reference == -__builtin_inff() ? 0.0f : reference;
        bf16x8 weight[kTerms];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float p = __builtin_amdgcn_exp2f(x[j] - shift);
            sum += p;
            float rest = p * value_scale[j];
            if (!clean && (seen >> j & 1) == 0) rest = 0.0f;
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
                weight[term][j] = static_cast<__bf16>(rest);
                rest -= static_cast<float>(weight[term][j]);
            }
        }
        // A row that does not see a value must not get 0 times no number from it: such codes are taken as zeros in tiles where some
        // row may not see them, and the rows that do are made no numbers afterwards.
        uint32_t none[kE4m3 ? kWords : 1] = {};  // of each of the lane's values: whether a key's code is no number, bit 8 * byte + j ... by word
        bool any_none = false;
        if (kE4m3 && !clean) {
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t odd = ((at.value[j][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;  // a byte's top bit: its code is no number
                    any_none |= odd != 0;
                }
            }
            any_none = __any(any_none);
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            uint32_t codes[8], bad[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) codes[j] = at.value[j][w];
            if (kE4m3 && any_none) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    bad[j] = (((codes[j] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;  // 1 in such a byte
                    codes[j] &= ~(bad[j] * 0xFFu);
                }
            }
            uint32_t operand[4][4];  // [value of the word][pair of keys]
#pragma unroll
            for (int pair = 0; pair < 4; ++pair) {
                if (kE4m3) {
                    const uint32_t low = __builtin_amdgcn_perm(codes[2 * pair + 1], codes[2 * pair], 0x05010400u);
                    const uint32_t high = __builtin_amdgcn_perm(codes[2 * pair + 1], codes[2 * pair], 0x07030602u);
                    operand[0][pair] = two_e4m3<false>(low);
                    operand[1][pair] = two_e4m3<true>(low);
                    operand[2][pair] = two_e4m3<false>(high);
                    operand[3][pair] = two_e4m3<true>(high);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) operand[i][pair] = pack(one_i8(codes[2 * pair], i), one_i8(codes[2 * pair + 1], i));
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bf16x8 value = __builtin_bit_cast(bf16x8, u32x4{operand[i][0], operand[i][1], operand[i][2], operand[i][3]});
#pragma unroll
                for (int term = kTerms - 1; term >= 0; --term) out[4 * w + i] = product(value, weight[term], out[4 * w + i]);
            }
            if (kE4m3 && any_none) {
                bf16x8 sees;
#pragma unroll
                for (int j = 0; j < 8; ++j) sees[j] = static_cast<__bf16>(static_cast<float>(seen >> j & 1));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bf16x8 is;
#pragma unroll
                    for (int j = 0; j < 8; ++j) is[j] = static_cast<__bf16>(static_cast<float>(bad[j] >> (8 * i) & 1));
                    const f32x4 count = product(is, sees, f32x4{0, 0, 0, 0});
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (count[j] > 0.0f) out[4 * w + i][j] = __builtin_nanf("");
                    }
                }
            }
        }
        (void)none;
    };

    while (tile < end) {
        if (tile + waves < end) {
            request_tile(tile + waves, pong);
            if (tile + 2 * waves < end) find(tile + 2 * waves);
        }
        work(tile, ping);
        tile += waves;
        if (tile >= end) break;
        if (tile + waves < end) {
            request_tile(tile + waves, ping);
            if (tile + 2 * waves < end) find(tile + 2 * waves);
        }
        work(tile, pong);
        tile += waves;
    }

    // ---- the wavefronts' sums together
    float* const sums = reinterpret_cast<float*>(lds + waves * kWaveLds);  // [wave][row][kDim + 4]
    constexpr int kStride = kDim + 4;
    Part* const wave_parts = reinterpret_cast<Part*>(sums + waves * here * kStride);  // [wave][row]
    const float total = row_sum(sum);
    const bool row_saw = row_max(saw ? 1.0f : 0.0f) > 0.0f;
    if (real) {
        float* to = sums + (wave * here + column) * kStride;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int w = 0; w < kWords; ++w)
                *reinterpret_cast<f32x4*>(to + kVec * (4 * quarter + i) + 4 * w) = f32x4{out[4 * w][i], out[4 * w + 1][i], out[4 * w + 2][i], out[4 * w + 3][i]};
        }
        if (quarter == 0) wave_parts[wave * here + column] = Part{!row_saw ? -__builtin_inff() : reference == -__builtin_inff() ? kLowest : reference, total};
    }
    __syncthreads();
    for (int item = tid; item < here * (kDim / 4); item += static_cast<int>(blockDim.x)) {
        const int r = item / (kDim / 4), d = item % (kDim / 4) * 4;
        if (d >= static_cast<int>(a.cache.head_dim)) continue;
        float highest = -__builtin_inff();
        for (int w = 0; w < waves; ++w) highest = fmaxf(highest, wave_parts[w * here + r].most);
        f32x4 x{0, 0, 0, 0};
        float all = 0.0f;
        for (int w = 0; w < waves; ++w) {
            const Part part = wave_parts[w * here + r];
            if (part.most == -__builtin_inff()) continue;
            const float by = exp2_between(part.most, highest);
            all = __builtin_fmaf(part.sum, by, all);
            const f32x4 y = *reinterpret_cast<const f32x4*>(sums + (w * here + r) * kStride + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(y[j], by, x[j]);
        }
        if (share.splits > 1) {
            *reinterpret_cast<f32x4*>(part_out + (static_cast<size_t>(slot) * 16 + r) * a.cache.head_dim + d) = x;
            if (d == 0) parts[static_cast<size_t>(slot) * 16 + r] = Part{highest, all};
        } else {
            const int whole = first_row + r;
            store4(a, static_cast<size_t>(share.begin + whole / group), kv_head * a.group + static_cast<uint32_t>(whole % group), d, x, all, highest != -__builtin_inff());
        }
    }
}

// A workgroup has sixteen rows of a request and a key head: a thread four values of a row, over all parts.
__global__ __launch_bounds__(256) void join_quantized_parts_kernel(QuantizedAttentionArgs a, Plan plan, const float* part_out, const Part* parts) {
    uint32_t request;
    Share share;
    if (!find_share<true>(a, plan, blockIdx.y, &request, &share) || share.splits <= 1) return;
    const uint32_t heads = a.cache.kv_heads, fours = a.cache.head_dim / 4;
    for (uint32_t number = blockIdx.x; number < share.row_tiles * heads; number += gridDim.x) {
        const uint32_t kv_head = number / share.row_tiles, row_tile = number % share.row_tiles;
        const uint32_t rows = min(16u, static_cast<uint32_t>(share.tokens) * a.group - row_tile * 16);
        const size_t first_slot = share.first_slot + static_cast<size_t>(kv_head) * share.splits * share.row_tiles + row_tile;
        for (uint32_t item = threadIdx.x; item < rows * fours; item += 256) {
            const uint32_t r = item / fours, d = item % fours * 4;
            float highest = -__builtin_inff(), all = 0.0f;
            f32x4 x{0, 0, 0, 0};
            for (uint32_t s = 0; s < share.splits; ++s) highest = fmaxf(highest, parts[(first_slot + static_cast<size_t>(s) * share.row_tiles) * 16 + r].most);
            for (uint32_t s = 0; s < share.splits; ++s) {
                const size_t at = (first_slot + static_cast<size_t>(s) * share.row_tiles) * 16 + r;
                const Part part = parts[at];
                if (part.most == -__builtin_inff()) continue;
                const float by = exp2_between(part.most, highest);
                all = __builtin_fmaf(part.sum, by, all);
                const f32x4 y = *reinterpret_cast<const f32x4*>(part_out + at * a.cache.head_dim + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(y[j], by, x[j]);
            }
            const uint32_t whole = row_tile * 16 + r;
            store4(a, static_cast<size_t>(share.begin) + whole / a.group, kv_head * a.group + whole % a.group, static_cast<int>(d), x, all, highest != -__builtin_inff());
        }
    }
}

struct Shape {
    int dim, waves;
    Plan plan;
    uint64_t groups, join_groups;
};

constexpr uint32_t kMostShared = 1024;  // requests: every wavefront reads their lengths, 64 at a time

Shape shape_of(const QuantizedAttentionArgs& a, int compute_units) {
    Shape s;
    s.dim = a.cache.head_dim <= 64 ? 64 : a.cache.head_dim <= 128 ? 128 : 256;
    s.waves = 4;
    const uint64_t rows = static_cast<uint64_t>(a.max_query_len) * a.group, most_row_tiles = (rows + 15) / 16;
    uint64_t row_tiles = static_cast<uint64_t>(a.tokens) * a.group / 16 + a.requests;  // of the batch: a request's last may be part empty
    if (row_tiles > a.requests * most_row_tiles) row_tiles = a.requests * most_row_tiles;
    const uint64_t base = row_tiles * a.cache.kv_heads;
    uint64_t keys = a.max_key_len;
    if (a.window != 0 && keys > static_cast<uint64_t>(a.window) + a.max_query_len) keys = static_cast<uint64_t>(a.window) + a.max_query_len;
    const uint64_t tiles = keys / kTile + 2;
    s.plan.row_tiles = static_cast<uint32_t>(most_row_tiles);
    s.plan.least = 8;
    s.plan.target = 0;
    const uint64_t resident = 4 * static_cast<uint64_t>(compute_units);
    if (a.requests <= kMostShared && base < 2 * resident && tiles > 16) s.plan.target = static_cast<uint32_t>(resident);
    s.groups = s.plan.target == 0 ? a.requests * most_row_tiles * a.cache.kv_heads : base + s.plan.target;
    s.plan.slots = s.plan.target == 0 ? 0 : static_cast<uint32_t>(s.groups);
    s.groups = (s.groups + 8 * most_row_tiles - 1) / (8 * most_row_tiles) * (8 * most_row_tiles);
    s.join_groups = most_row_tiles * a.cache.kv_heads;
    if (s.join_groups > 4096) s.join_groups = 4096;
    return s;
}

size_t part_out_bytes(const QuantizedAttentionArgs& a, const Shape& s) { return (static_cast<size_t>(s.plan.slots) * 16 * a.cache.head_dim * sizeof(float) + 255) / 256 * 256; }

template <int kDim, bool kE4m3, int kTerms>
hipError_t attend(hipStream_t stream, const QuantizedAttentionArgs& a, const Shape& s, void* workspace) {
    static LdsLimit limit;
    const uint64_t rows = static_cast<uint64_t>(a.max_query_len) * a.group, here = rows < 16 ? rows : 16;
    const size_t lds = static_cast<size_t>(s.waves) * (kWaveLds + here * ((kDim + 4) * sizeof(float) + sizeof(Part)));
    const auto kernel = quantized_attention_kernel<kDim, kE4m3, kTerms>;
    static_assert(waves_of(kDim) * (kWaveLds + 16 * ((kDim + 4) * sizeof(float) + sizeof(Part))) <= 160 * 1024, "a compute unit's LDS");
    hipError_t e = allow_lds(kernel, lds, &limit);
    if (e != hipSuccess) return e;
    float* part_out = static_cast<float*>(workspace);
    Part* parts = s.plan.slots != 0 ? reinterpret_cast<Part*>(static_cast<char*>(workspace) + part_out_bytes(a, s)) : nullptr;
    kernel<<<static_cast<uint32_t>(s.groups), 64 * s.waves, lds, stream>>>(a, s.plan, part_out, parts);
    e = hipGetLastError();
    if (e != hipSuccess || s.plan.slots == 0) return e;
    join_quantized_parts_kernel<<<dim3(static_cast<uint32_t>(s.join_groups), a.requests), 256, 0, stream>>>(a, s.plan, part_out, parts);
    return hipGetLastError();
}

template <int kDim, bool kE4m3>
hipError_t attend_types(hipStream_t stream, const QuantizedAttentionArgs& a, const Shape& s, void* workspace) {
    if (a.type == 0) return attend<kDim, kE4m3, 3>(stream, a, s, workspace);
    if (a.type == 1) return attend<kDim, kE4m3, 2>(stream, a, s, workspace);
    return attend<kDim, kE4m3, 1>(stream, a, s, workspace);
}

}  // namespace

size_t quantized_attention_workspace_bytes(const QuantizedAttentionArgs& args, int compute_units) {
    const Shape s = shape_of(args, compute_units);
    return s.plan.slots == 0 ? 0 : part_out_bytes(args, s) + static_cast<size_t>(s.plan.slots) * 16 * sizeof(Part);
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
