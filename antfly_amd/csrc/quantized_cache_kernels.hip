// What lies between a projection and the attention over a paged cache: norms of queries and keys head by head, their rotation by
// the tokens' positions, and keys and values written to a 16-bit or 8-bit cache; and the way back from an 8-bit cache.
//
//   y = x / sqrt(mean x^2 + eps) * w;   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * frequency
//   m = max |x| over a head:   scale = m / L,  code = x (L / m),  L = 127 or 448
//
// A head is a group of 8, 16 or 32 lanes with eight values each: its sum of squares and its maximum are three to five exchanges of
// registers.  A lane's eight values are four pairs of the rotation (two runs of four values), so a pair never leaves its lane.  The
// angles are the same for all heads of a token: a workgroup's threads make one each, while the first heads' values are on their way,
// and every lane keeps those of its four pairs for the heads it takes (made by each lane, 2111 tokens of 32 heads took 5 % longer).
// Registers are kept to eight wavefronts a SIMD: 7500 tokens of 48 heads take 60 us instead of 64 with seven, the 2111 3 % longer.
// Bound by the bytes: 7500 tokens of 32 and 8 heads of 128, f32 in, bf16 queries out, keys and values to e4m3, 60 us, 4.4 TB/s; 4000
// tokens of 8 heads of 128 stored and 30001 loaded, 57 us, 4.0 TB/s; 2111 tokens of 28 and 4 heads, three axes, 13.8 us.  A few tokens
// cost a launch (one: 4.0 us).
#include "quantized_launch.h"

#include <hip/hip_runtime.h>

namespace afhip {

namespace {

constexpr int kThreads = 256;
constexpr float kTiniest = 0x1p-100f;  // a head's maximum counts as at least this: its scale and the reciprocal stay normal numbers
constexpr uint32_t kInfinity = 0x7f800000u;

typedef float f32x4 __attribute__((ext_vector_type(4)));

// `what(v, another lane's v)` over the lanes of a group of kLanes, in all of them.
template <int kControl>
__device__ __forceinline__ uint32_t other(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kControl, 0xF, 0xF, false));
}
template <int kLanes, typename What>
__device__ __forceinline__ uint32_t over_group(uint32_t v, What what) {
    v = what(v, other<0xB1>(v));   // lane ^ 1
    v = what(v, other<0x4E>(v));   // lane ^ 2
    v = what(v, other<0x141>(v));  // the other four of eight
    if (kLanes > 8) v = what(v, other<0x140>(v));  // the other eight of sixteen
    if (kLanes > 16) v = what(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
    return v;
}
template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
    return __builtin_bit_cast(float, over_group<kLanes>(__builtin_bit_cast(uint32_t, v), [](uint32_t a, uint32_t b) {
                                  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
                              }));
}
template <int kLanes>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    return over_group<kLanes>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

struct __attribute__((packed, aligned(4))) Four { float v[4]; };  // weights and frequencies lie on any 4 bytes

template <int kType>
__device__ __forceinline__ f32x4 load4(const void* base, size_t element) {
    if (kType == 0) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + element);
    const uint2 raw = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + element);
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint16_t h = static_cast<uint16_t>((i < 2 ? raw.x : raw.y) >> (16 * (i & 1)));
        v[i] = kType == 30 ? __builtin_bit_cast(float, static_cast<uint32_t>(h) << 16) : static_cast<float>(__builtin_bit_cast(_Float16, h));
    }
    return v;
}

__device__ __forceinline__ uint32_t pack16(float a, float b, bool bf16) {
    if (bf16) {
        const __bf16 x = static_cast<__bf16>(a), y = static_cast<__bf16>(b);
        return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, x)) | (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, y)) << 16);
    }
    const _Float16 x = static_cast<_Float16>(a), y = static_cast<_Float16>(b);
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, x)) | (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, y)) << 16);
}
// type: 0 f32, 1 f16, 30 bf16
__device__ __forceinline__ void store4(void* base, size_t element, f32x4 v, int type) {
    if (type == 0) *reinterpret_cast<f32x4*>(static_cast<float*>(base) + element) = v;
    else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + element) = uint2{pack16(v[0], v[1], type == 30), pack16(v[2], v[3], type == 30)};
}

// sin and cos of position * frequency.  The product with 1 / (2 pi) is held in two 64-bit numbers (a position of 31 bits times a
// frequency of 24 has 55, and 28 of the quotient's go with the whole turns: in one number the angle is off by 8 steps of 2^-24 at
// positions of 2^31), so that what is left of the turn, at most an eighth, is good to f32's last bit.  Then the two Taylor series in
// quarter turns, whose first terms left out are below 2e-9 and 2e-10.
__device__ __forceinline__ void sine_cosine(int position, float frequency, float* sine, float* cosine) {
    constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnRest = -0x1.6b01ec5417056p-57;  // 1 / (2 pi)
    const double f = static_cast<double>(frequency), p = static_cast<double>(position);
    const double step = f * kTurn, step_rest = __builtin_fma(f, kTurn, -step) + f * kTurnRest;
    const double turns = p * step, turns_rest = __builtin_fma(p, step, -turns) + p * step_rest;
    const double rest = (turns - __builtin_rint(turns)) + turns_rest;
    const double quarters = 4.0 * (rest - __builtin_rint(rest)), whole = __builtin_rint(quarters);
    const float x = static_cast<float>(quarters - whole), z = x * x;
    const int quarter = static_cast<int>(whole);
    // (pi / 2)^n / n!
    const float s = x * __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.60441185e-4f, -4.68175414e-3f), 7.96926262e-2f), -6.45964098e-1f), 1.57079633f);
    const float c = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -2.52020424e-5f, 9.19260274e-4f), -2.08634807e-2f), 2.53669508e-1f), -1.23370055f), 1.0f);
    const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
    *sine = quarter & 2 ? -a : a;
    *cosine = (quarter + 1) & 2 ? -b : b;
}

struct Codes {
    uint32_t first, second;  // of a lane's two runs of four values
    float scale;
};
template <int kLanes>
__device__ __forceinline__ Codes quantize(f32x4 a, f32x4 b, bool e4m3) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = a[i], y = b[i];  // (a bit_cast of a[i] itself reads a[0])
        // (the bits of magnitudes are in their order, no numbers last)
        most = max(most, max(__builtin_bit_cast(uint32_t, x) & 0x7fffffffu, __builtin_bit_cast(uint32_t, y) & 0x7fffffffu));
    }
    most = group_max<kLanes>(most);
    if (most >= kInfinity) return Codes{0, 0, __builtin_nanf("")};
    const float m = fmaxf(__builtin_bit_cast(float, most), kTiniest), largest = e4m3 ? 448.0f : 127.0f, by = largest / m;
    a *= by;
    b *= by;
    Codes c;
    c.scale = m / largest;
    if (e4m3) {
        c.first = __builtin_amdgcn_cvt_pk_fp8_f32(a[2], a[3], __builtin_amdgcn_cvt_pk_fp8_f32(a[0], a[1], 0, false), true);
        c.second = __builtin_amdgcn_cvt_pk_fp8_f32(b[2], b[3], __builtin_amdgcn_cvt_pk_fp8_f32(b[0], b[1], 0, false), true);
    } else {
        c.first = c.second = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c.first |= (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(a[i]))) & 0xFF) << (8 * i);
            c.second |= (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(b[i]))) & 0xFF) << (8 * i);
        }
    }
    return c;
}

// Items of a token: its queries' heads, its keys', its values'.  A workgroup has tokens_a_group tokens and groups_a_token groups of
// lanes for each, which take the items of its chunk (blockIdx.y) in turn.
template <int kType, int kLanes>
__global__ __launch_bounds__(kThreads, 8) void heads_kernel(HeadsArgs a) {
    __shared__ float2 turned[kThreads * 4];  // sines and cosines of [token][pair]: 32, 16 or 8 tokens of up to 32, 64 or 128
    const uint32_t lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, own_token = group / a.groups_a_token;
    const uint32_t token = blockIdx.x * a.tokens_a_group + own_token;
    const bool idle = group >= a.tokens_a_group * a.groups_a_token || token >= a.tokens;
    const uint32_t items = a.heads + a.kv_heads + a.value_heads;
    const uint32_t last = min(items, (blockIdx.y + 1) * a.chunk);
    // the lane's two runs of four values, and its four pairs
    const uint32_t rotary = a.rotary_dim, first_pair = 4 * lane;
    const bool works = 8 * lane < a.head_dim, turns = 8 * lane < rotary;
    const uint32_t d0 = turns && !a.interleaved ? 4 * lane : 8 * lane, d1 = turns && !a.interleaved ? rotary / 2 + 4 * lane : 8 * lane + 4;
    // a head's values, asked for before the angles are formed
    f32x4 next_x{0, 0, 0, 0}, next_y{0, 0, 0, 0};
    const auto request = [&](uint32_t item) {
        const bool is_query = item < a.heads, is_value = item >= a.heads + a.kv_heads;
        const uint32_t head = is_query ? item : is_value ? item - a.heads - a.kv_heads : item - a.heads;
        const HeadRows& from = is_query ? a.query : is_value ? a.value : a.key;
        const size_t at = static_cast<size_t>(token) * from.token_stride + static_cast<size_t>(head) * from.head_stride;
        if (works && item < last) {
            next_x = load4<kType>(from.data, at + d0);
            next_y = load4<kType>(from.data, at + d1);
        }
    };
    const uint32_t first_item = blockIdx.y * a.chunk + group % a.groups_a_token;
    if (!idle) request(first_item);
    if (a.positions != nullptr) {
        const uint32_t pairs = rotary / 2;
        for (uint32_t i = threadIdx.x; i < a.tokens_a_group * pairs; i += kThreads) {
            const uint32_t of = a.tokens_a_group == 1 ? 0 : i / pairs, pair = i - of * pairs, its = blockIdx.x * a.tokens_a_group + of;
            if (its >= a.tokens) break;
            const int position = a.positions[a.one_axis ? its : static_cast<size_t>(a.pair_axes[pair]) * a.tokens + its];
            float2 both;
            sine_cosine(position, a.frequencies[pair], &both.x, &both.y);
            turned[i] = both;
        }
        __syncthreads();
    }
    if (idle) return;
    float sine[4], cosine[4];
    if (turns) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const float2 both = turned[own_token * (rotary / 2) + first_pair + p];
            sine[p] = both.x;
            cosine[p] = both.y;
        }
    }
    const float inverse_dim = 1.0f / static_cast<float>(a.head_dim);
    const int target = static_cast<int>(a.target);
    uint32_t block = 0, inside = 0;
    bool there = true;
    if (target != static_cast<int>(HeadTarget::arrays)) {
        const uint32_t slot = static_cast<uint32_t>(a.slots[token]), block_size = target >= static_cast<int>(HeadTarget::i8_cache) ? a.quantized.block_size : a.cache.block_size;
        block = slot / block_size;
        inside = slot - block * block_size;
        there = block < (target >= static_cast<int>(HeadTarget::i8_cache) ? a.quantized.blocks : a.cache.blocks);
    }
    for (uint32_t item = first_item; item < last; item += a.groups_a_token) {
        const bool is_query = item < a.heads, is_value = item >= a.heads + a.kv_heads;
        const uint32_t head = is_query ? item : is_value ? item - a.heads - a.kv_heads : item - a.heads;
        f32x4 x = next_x, y = next_y;
        request(item + a.groups_a_token);
        if (!is_value) {
            const float* weight = is_query ? a.query_weight : a.key_weight;
            if (weight != nullptr) {
                const float squares = (x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]) + ((y[0] * y[0] + y[1] * y[1]) + (y[2] * y[2] + y[3] * y[3]));
                const float by = __builtin_amdgcn_rsqf(group_sum<kLanes>(squares) * inverse_dim + a.epsilon);  // (off by an f32 step)
                if (works) {
                    const Four first = *reinterpret_cast<const Four*>(weight + d0), second = *reinterpret_cast<const Four*>(weight + d1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = x[i] * by * first.v[i];
                        y[i] = y[i] * by * second.v[i];
                    }
                }
            }
            if (turns) {
                const f32x4 u = x, v = y;
                if (a.interleaved) {
                    x = f32x4{u[0] * cosine[0] - u[1] * sine[0], u[0] * sine[0] + u[1] * cosine[0], u[2] * cosine[1] - u[3] * sine[1], u[2] * sine[1] + u[3] * cosine[1]};
                    y = f32x4{v[0] * cosine[2] - v[1] * sine[2], v[0] * sine[2] + v[1] * cosine[2], v[2] * cosine[3] - v[3] * sine[3], v[2] * sine[3] + v[3] * cosine[3]};
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = u[i] * cosine[i] - v[i] * sine[i];
                        y[i] = u[i] * sine[i] + v[i] * cosine[i];
                    }
                }
            }
        }
        if (is_query || target == static_cast<int>(HeadTarget::arrays)) {
            const HeadRows& to = is_query ? a.out_query : a.out_key;
            const size_t out = static_cast<size_t>(token) * to.token_stride + static_cast<size_t>(head) * to.head_stride;
            if (works) {
                store4(to.data, out + d0, x, a.out_type);
                store4(to.data, out + d1, y, a.out_type);
            }
        } else if (target >= static_cast<int>(HeadTarget::i8_cache)) {
            const QuantizedView& q = a.quantized;
            const Codes c = quantize<kLanes>(x, y, q.e4m3);
            if (!there) continue;
            char* codes = reinterpret_cast<char*>((is_value ? q.values : q.keys) + (static_cast<size_t>(block) * q.block_stride + static_cast<size_t>(inside) * q.slot_stride +
                                                                                     static_cast<size_t>(head) * q.head_stride));
            if (works) {
                *reinterpret_cast<uint32_t*>(codes + d0) = c.first;
                *reinterpret_cast<uint32_t*>(codes + d1) = c.second;
            }
            if (lane == 0)
                (is_value ? q.value_scales : q.key_scales)[static_cast<size_t>(block) * q.scale_block_stride + static_cast<size_t>(inside) * q.scale_slot_stride +
                                                           static_cast<size_t>(head) * q.scale_head_stride] = c.scale;
        } else if (there && works) {
            const size_t out = (static_cast<size_t>(block) * a.cache.block_stride + static_cast<size_t>(inside) * a.cache.slot_stride +
                                static_cast<size_t>(head) * a.cache.head_stride) * 8;
            void* to = is_value ? a.cache.values : a.cache.keys;
            const int type = target == static_cast<int>(HeadTarget::bf16_cache) ? 30 : 1;
            store4(to, out + d0, x, type);
            store4(to, out + d1, y, type);
        }
    }
}

// A lane reads eight codes of each of kTogether heads, requested together, and writes eight values of each.
template <int kLanes, int kTogether>
__global__ __launch_bounds__(kThreads) void quantized_load_kernel(QuantizedView cache, int type, HeadRows keys, HeadRows values, const int* slots, uint32_t tokens,
                                                                 uint32_t items) {
    const uint32_t lane = threadIdx.x % kLanes, first = (blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes) * kTogether;
    if (first >= items || 8 * lane >= cache.head_dim) return;
    const uint32_t both = 2 * cache.kv_heads;
    uint32_t token[kTogether], head[kTogether];
    bool is_value[kTogether], there[kTogether];
    uint2 codes[kTogether];
    float scale[kTogether];
    uint32_t at_token = first / both, at_item = first % both;
#pragma unroll
    for (int t = 0; t < kTogether; ++t) {
        token[t] = at_token;
        is_value[t] = at_item >= cache.kv_heads;
        head[t] = is_value[t] ? at_item - cache.kv_heads : at_item;
        there[t] = first + t < items;
        if (++at_item == both) {
            at_item = 0;
            ++at_token;
        }
    }
    uint32_t slot[kTogether];
#pragma unroll
    for (int t = 0; t < kTogether; ++t) slot[t] = there[t] ? static_cast<uint32_t>(slots[token[t]]) : ~0u;
#pragma unroll
    for (int t = 0; t < kTogether; ++t) {
        const uint32_t block = slot[t] / cache.block_size, inside = slot[t] % cache.block_size;
        there[t] = there[t] && block < cache.blocks;
        if (!there[t]) continue;
        const uint4* from = (is_value[t] ? cache.values : cache.keys) +
                            (static_cast<size_t>(block) * cache.block_stride + static_cast<size_t>(inside) * cache.slot_stride + static_cast<size_t>(head[t]) * cache.head_stride);
        codes[t] = reinterpret_cast<const uint2*>(from)[lane];
        scale[t] = (is_value[t] ? cache.value_scales : cache.key_scales)[static_cast<size_t>(block) * cache.scale_block_stride +
                                                                        static_cast<size_t>(inside) * cache.scale_slot_stride +
                                                                        static_cast<size_t>(head[t]) * cache.scale_head_stride];
    }
#pragma unroll
    for (int t = 0; t < kTogether; ++t) {
        if (!there[t]) continue;
        f32x4 v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t four = h == 0 ? codes[t].x : codes[t].y;
            if (cache.e4m3) {
                const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(four), false), high = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(four), true);
                v[h] = f32x4{low[0], low[1], high[0], high[1]};
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[h][i] = static_cast<float>(static_cast<int8_t>(four >> (8 * i)));
            }
            v[h] *= scale[t];
        }
        const HeadRows& to = is_value[t] ? values : keys;
        const size_t out = static_cast<size_t>(token[t]) * to.token_stride + static_cast<size_t>(head[t]) * to.head_stride + 8 * lane;
        if (type == 0) {
            store4(to.data, out, v[0], 0);
            store4(to.data, out + 4, v[1], 0);
        } else {
            const bool bf16 = type == 30;
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(to.data) + out) = uint4{pack16(v[0][0], v[0][1], bf16), pack16(v[0][2], v[0][3], bf16), pack16(v[1][0], v[1][1], bf16), pack16(v[1][2], v[1][3], bf16)};
        }
    }
}

int lanes_of(uint32_t head_dim) { return head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32; }

template <int kType>
hipError_t heads(hipStream_t stream, const HeadsArgs& a, dim3 grid) {
    switch (lanes_of(a.head_dim)) {
        case 8: heads_kernel<kType, 8><<<grid, kThreads, 0, stream>>>(a); break;
        case 16: heads_kernel<kType, 16><<<grid, kThreads, 0, stream>>>(a); break;
        default: heads_kernel<kType, 32><<<grid, kThreads, 0, stream>>>(a); break;
    }
    return hipGetLastError();
}

template <int kTogether>
hipError_t load(hipStream_t stream, const QuantizedView& cache, int type, const HeadRows& keys, const HeadRows& values, const int* slots, uint32_t tokens) {
    const uint32_t items = tokens * 2 * cache.kv_heads, lanes = lanes_of(cache.head_dim), each = kThreads / lanes * kTogether;
    const uint32_t grid = static_cast<uint32_t>((static_cast<uint64_t>(items) + each - 1) / each);
    switch (lanes) {
        case 8: quantized_load_kernel<8, kTogether><<<grid, kThreads, 0, stream>>>(cache, type, keys, values, slots, tokens, items); break;
        case 16: quantized_load_kernel<16, kTogether><<<grid, kThreads, 0, stream>>>(cache, type, keys, values, slots, tokens, items); break;
        default: quantized_load_kernel<32, kTogether><<<grid, kThreads, 0, stream>>>(cache, type, keys, values, slots, tokens, items); break;
    }
    return hipGetLastError();
}

struct HeadsGrid {
    uint32_t groups, items, groups_a_token, tokens_a_group;
    uint64_t x;
    HeadsGrid(uint32_t tokens, uint32_t all, uint32_t head_dim) : groups(kThreads / lanes_of(head_dim)), items(all) {
        groups_a_token = items < groups ? items : groups;
        tokens_a_group = groups / groups_a_token;
        x = (static_cast<uint64_t>(tokens) + tokens_a_group - 1) / tokens_a_group;
    }
};

}  // namespace

bool heads_fit_a_launch(uint32_t tokens, uint32_t items, uint32_t head_dim) {
    const HeadsGrid grid(tokens, items, head_dim);
    // (a token's chunks are no more than its items over its groups)
    return fits_a_launch(grid.x, kThreads) && (items + grid.groups_a_token - 1) / grid.groups_a_token <= 65535;
}

hipError_t launch_heads(hipStream_t stream, int type, const HeadsArgs& args, int compute_units) {
    HeadsArgs a = args;
    const HeadsGrid grid(a.tokens, a.heads + a.kv_heads + a.value_heads, a.head_dim);
    a.groups_a_token = grid.groups_a_token;
    a.tokens_a_group = grid.tokens_a_group;
    // A token's heads are one workgroup's, which makes the angles once, unless there are too few tokens to fill the units (in chunks and in
    // one workgroup, 32 heads and 8 of keys and values, f32 into an e4m3 cache: 1 token 4.0 and 5.6 us, 200 tokens 4.7 and 6.3, 500 5.8 and 7.0,
    // 1000 9.7 and 9.4, 2000 16.6 and 15.0).
    const uint32_t rounds = (grid.items + grid.groups_a_token - 1) / grid.groups_a_token;
    const uint64_t wanted = 8 * static_cast<uint64_t>(compute_units);
    uint32_t chunks = grid.x >= wanted ? 1 : static_cast<uint32_t>((wanted + grid.x - 1) / grid.x);
    if (chunks > rounds || a.positions == nullptr) chunks = rounds;
    a.chunk = (rounds + chunks - 1) / chunks * grid.groups_a_token;
    const dim3 shape(static_cast<uint32_t>(grid.x), (grid.items + a.chunk - 1) / a.chunk);
    return type == 0 ? heads<0>(stream, a, shape) : type == 1 ? heads<1>(stream, a, shape) : heads<30>(stream, a, shape);
}

hipError_t launch_quantized_load(hipStream_t stream, const QuantizedView& cache, int type, const HeadRows& keys, const HeadRows& values,
                                 const int* slots, uint32_t tokens, int compute_units) {
    // Eight heads a group of lanes where that still gives every unit eight workgroups: 30001 tokens of 8 heads of 128 39 us instead of 55;
    // a step that stores and loads 64 tokens takes 10.6 us that way instead of 5.7.
    const uint64_t groups = static_cast<uint64_t>(tokens) * 2 * cache.kv_heads * lanes_of(cache.head_dim) / kThreads;
    return groups >= 64 * static_cast<uint64_t>(compute_units) ? load<8>(stream, cache, type, keys, values, slots, tokens) : load<1>(stream, cache, type, keys, values, slots, tokens);
}

}  // namespace afhip
