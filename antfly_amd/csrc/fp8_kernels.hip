// Matrix product in 8-bit floating point with a scale per block of 128:
//
//   Y[r][o] = sum over blocks b of  x_scale[r][b] * w_scale[o / 128][b] * (sum over k in b of  x[r][k] * w[o][k])
//
// The codes are widened to f16, which holds every e4m3 number exactly (v_cvt_scalef32_pk_f16_fp8, two a lane and
// instruction), and multiplied on the f16 matrix instructions, whose products are exact and whose sums are f32.  The 8-bit
// instructions (v_mfma_scale_f32_*_f8f6f4, and the older v_mfma_f32_*_fp8_fp8 alike) would do twice the products a cycle,
// but what they add is cut some 17 bits below the largest product of an instruction: on codes of all sizes the result is
// off by 5e-5 of its norm, where f32 sums are off by 3e-7.  The block's sum is then multiplied by the two scales and added to the
// result in f32 on the vector ALU.  The weights are the first operand and the activations the second, so a lane's results all
// belong to one row of X: its scale is one register, the weights' is the same for the whole wavefront, and a block costs one
// multiplication and one fused multiply-add a result.
//
// The order of the values of K inside an instruction is free as long as both operands keep it: a lane takes whole 16-byte
// pieces as they lie in memory.
#include "device_common.h"
#include "fp8_launch.h"

#include <hip/hip_runtime.h>

namespace afhip {

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kMost = 448.0f;           // of e4m3
constexpr float kTiniest = 0x1p-100f;     // a block's maximum counts as at least this: its scale and the reciprocal stay normal numbers

// Eight codes as f16.
__device__ __forceinline__ f16x8 widen(uint32_t lo, uint32_t hi) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ---- quantizer: eight lanes a block, four values of each 32 to a lane
__global__ __launch_bounds__(256) void quantize_fp8_kernel(uint8_t* q, float* scales, const float* x, size_t blocks, int row_blocks, int in_dim) {
    const size_t at = static_cast<size_t>(blockIdx.x) * 32 + threadIdx.x / 8;
    if (at >= blocks) return;
    const size_t row = at / row_blocks;
    const int block = static_cast<int>(at % row_blocks), part = threadIdx.x & 7;
    const size_t from = row * in_dim;
    float4 v[4];
    float most = kTiniest;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = block * kFp8Block + i * 32 + part * 4;
        v[i] = k < in_dim ? *reinterpret_cast<const float4*>(x + from + k) : float4{0, 0, 0, 0};
        most = fmaxf(most, fmaxf(fmaxf(__builtin_fabsf(v[i].x), __builtin_fabsf(v[i].y)), fmaxf(__builtin_fabsf(v[i].z), __builtin_fabsf(v[i].w))));
    }
    most = max_over_8(most);
    const float by = kMost / most;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = block * kFp8Block + i * 32 + part * 4;
        int code = __builtin_amdgcn_cvt_pk_fp8_f32(v[i].x * by, v[i].y * by, 0, false);
        code = __builtin_amdgcn_cvt_pk_fp8_f32(v[i].z * by, v[i].w * by, code, true);
        if (k < in_dim) *reinterpret_cast<int*>(q + from + k) = code;
    }
    if (part == 0) scales[at] = most / kMost;
}

// ---- few rows: operands from memory into registers
//
// A workgroup has 16 kN columns of W and 16 kM rows of X; its wavefronts share out the blocks of K (in turn) and add up in
// LDS.  kAhead blocks are requested at a time.
template <int kM, int kN, int kWaves, int kAhead>
__global__ __launch_bounds__(kWaves * 64) void matmul_fp8_rows_kernel(Fp8Matmul a) {
    __shared__ float sums[kWaves][16 * kM][16 * kN + 4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, column = lane & 15, quarter = lane >> 4;
    const int first_o = blockIdx.x * 16 * kN, first_r = blockIdx.y * 16 * kM;
    const int blocks = fp8_blocks(a.in_dim);
    const uint4* w[kN];
    const uint4* x[kM];
    const float* x_scale[kM];
    const float* w_scale[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        w[n] = reinterpret_cast<const uint4*>(a.w + static_cast<size_t>(min(first_o + n * 16 + column, a.out_dim - 1)) * a.in_dim);
        w_scale[n] = a.w_scales + static_cast<size_t>(min(first_o + n * 16, a.out_dim - 1) / kFp8Block) * blocks;
    }
#pragma unroll
    for (int m = 0; m < kM; ++m) {
        const size_t row = min(first_r + m * 16 + column, a.rows - 1);
        x[m] = reinterpret_cast<const uint4*>(a.x + row * a.in_dim);
        x_scale[m] = a.x_scales + row * blocks;
    }
    f32x4 total[kN][kM];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int m = 0; m < kM; ++m) total[n][m] = f32x4{0, 0, 0, 0};
    }
    const int pieces = a.in_dim / 16;
    const uint4 zero{0, 0, 0, 0};
    for (int b0 = wave; b0 < blocks; b0 += kWaves * kAhead) {
        uint4 wv[kAhead][kN][2], xv[kAhead][kM][2];
        float ws[kAhead][kN], xs[kAhead][kM];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int b = b0 + i * kWaves;
            const int p0 = b * 8 + quarter, p1 = p0 + 4;
            const bool first = b < blocks && p0 < pieces, second = b < blocks && p1 < pieces;
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                wv[i][n][0] = first ? w[n][p0] : zero;
                wv[i][n][1] = second ? w[n][p1] : zero;
                ws[i][n] = b < blocks ? w_scale[n][b] : 0.0f;
            }
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                xv[i][m][0] = first ? x[m][p0] : zero;
                xv[i][m][1] = second ? x[m][p1] : zero;
                xs[i][m] = b < blocks ? x_scale[m][b] : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            f32x4 dot[kN][kM];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                f16x8 wide_w[kN], wide_x[kM];
#pragma unroll
                for (int n = 0; n < kN; ++n) wide_w[n] = k & 1 ? widen(wv[i][n][k / 2].z, wv[i][n][k / 2].w) : widen(wv[i][n][k / 2].x, wv[i][n][k / 2].y);
#pragma unroll
                for (int m = 0; m < kM; ++m) wide_x[m] = k & 1 ? widen(xv[i][m][k / 2].z, xv[i][m][k / 2].w) : widen(xv[i][m][k / 2].x, xv[i][m][k / 2].y);
#pragma unroll
                for (int n = 0; n < kN; ++n) {
#pragma unroll
                    for (int m = 0; m < kM; ++m)
                        dot[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wide_w[n], wide_x[m], k == 0 ? f32x4{0, 0, 0, 0} : dot[n][m], 0, 0, 0);
                }
            }
#pragma unroll
            for (int n = 0; n < kN; ++n) {
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    const float scale = xs[i][m] * ws[i][n];
#pragma unroll
                    for (int j = 0; j < 4; ++j) total[n][m][j] = __builtin_fmaf(dot[n][m][j], scale, total[n][m][j]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int m = 0; m < kM; ++m) *reinterpret_cast<f32x4*>(&sums[wave][m * 16 + column][n * 16 + quarter * 4]) = total[n][m];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * kM * kN; i += kWaves * 64) {
        const int m = i / (16 * kN), n = i % (16 * kN), row = first_r + m, o = first_o + n;
        if (row >= a.rows || o >= a.out_dim) continue;
        float v = 0.0f;
#pragma unroll
        for (int s = 0; s < kWaves; ++s) v += sums[s][m][n];
        const size_t to = static_cast<size_t>(row) * a.out_dim + o;
        a.y[to] = finish_output(a.ep, o, to, v);
    }
}

// ---- many rows: tiles through LDS
//
// 128 rows of X and 128 columns of W a workgroup, four wavefronts with 64 x 64 results each; a block of K (128 bytes a row)
// at a time, the next one on its way from memory straight into the other half of LDS.  16-byte piece p of row r lies at
// place p ^ (r % 8): eight lanes that read the same piece of eight rows fall on other banks.
__device__ const uint4 kZeroPiece{0, 0, 0, 0};  // what pieces past in_dim are loaded from

__global__ __launch_bounds__(256) void matmul_fp8_tile_kernel(Fp8Matmul a) {
    __shared__ __attribute__((aligned(16))) char lds[2][2][128 * 128];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first_o = blockIdx.x * 128, first_r = blockIdx.y * 128;
    const int blocks = fp8_blocks(a.in_dim), pieces = a.in_dim / 16;
    const int wave_o = (wave & 1) * 64, wave_r = (wave >> 1) * 64;
    const float* w_scale = a.w_scales + static_cast<size_t>(blockIdx.x) * blocks;
    const float* x_scale[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) x_scale[m] = a.x_scales + static_cast<size_t>(min(first_r + wave_r + m * 32 + (lane & 31), a.rows - 1)) * blocks;

    auto request = [&](int b, int half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int slot = i * 256 + wave * 64 + lane, row = slot >> 3, piece = b * 8 + ((slot & 7) ^ (row & 7));
            const uint4* w = reinterpret_cast<const uint4*>(a.w + static_cast<size_t>(min(first_o + row, a.out_dim - 1)) * a.in_dim) + piece;
            const uint4* x = reinterpret_cast<const uint4*>(a.x + static_cast<size_t>(min(first_r + row, a.rows - 1)) * a.in_dim) + piece;
            if (piece >= pieces) w = x = &kZeroPiece;
            char* to = lds[half][0] + (i * 256 + wave * 64) * 16;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)w, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)x, (__attribute__((address_space(3))) void*)(to + 128 * 128), 16, 0, 0);
        }
    };
    f32x16 total[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int m = 0; m < 2; ++m) total[n][m] = f32x16{};
    }
    request(0, 0);
    for (int b = 0; b < blocks; ++b) {
        const float xs[2] = {x_scale[0][b], x_scale[1][b]}, ws = w_scale[b];
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // the wavefront's own bytes of this block are in LDS (a barrier alone does not wait for them)
        __syncthreads();                                    // everyone's are, and the other half has been read
        if (b + 1 < blocks) request(b + 1, (b + 1) & 1);
        const char* at = lds[b & 1][0];
        f32x16 dot[2][2];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // 32 of K: a 16-byte piece a lane, two instructions' worth
            f16x8 w[2][2], x[2][2];
            const int piece = k * 2 + (lane >> 5);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int wr = wave_o + t * 32 + (lane & 31), xr = wave_r + t * 32 + (lane & 31);
                const uint4 wp = *reinterpret_cast<const uint4*>(at + wr * 128 + (piece ^ (wr & 7)) * 16);
                const uint4 xp = *reinterpret_cast<const uint4*>(at + 128 * 128 + xr * 128 + (piece ^ (xr & 7)) * 16);
                w[t][0] = widen(wp.x, wp.y);
                w[t][1] = widen(wp.z, wp.w);
                x[t][0] = widen(xp.x, xp.y);
                x[t][1] = widen(xp.z, xp.w);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
                        dot[n][m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w[n][half], x[m][half], k + half == 0 ? f32x16{} : dot[n][m], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const float scale = xs[m] * ws;
#pragma unroll
                for (int j = 0; j < 16; ++j) total[n][m][j] = __builtin_fmaf(dot[n][m][j], scale, total[n][m][j]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const int row = first_r + wave_r + m * 32 + (lane & 31);
        if (row >= a.rows) continue;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int o = first_o + wave_o + n * 32 + (j >> 2) * 8 + (lane >> 5) * 4 + (j & 3);
                const size_t to = static_cast<size_t>(row) * a.out_dim + o;
                if (o < a.out_dim) a.y[to] = finish_output(a.ep, o, to, total[n][m][j]);
            }
        }
    }
}

template <int kM, int kN, int kWaves, int kAhead>
hipError_t rows_kernel(hipStream_t stream, const Fp8Matmul& a) {
    const dim3 grid((a.out_dim + 16 * kN - 1) / (16 * kN), (a.rows + 16 * kM - 1) / (16 * kM));
    matmul_fp8_rows_kernel<kM, kN, kWaves, kAhead><<<grid, kWaves * 64, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize_fp8(hipStream_t stream, uint8_t* q, float* scales, const float* x, size_t rows, int in_dim) {
    const int row_blocks = fp8_blocks(in_dim);
    const size_t blocks = rows * row_blocks;
    quantize_fp8_kernel<<<static_cast<uint32_t>((blocks + 31) / 32), 256, 0, stream>>>(q, scales, x, blocks, row_blocks, in_dim);
    return hipGetLastError();
}

hipError_t launch_matmul_fp8(hipStream_t stream, const Fp8Matmul& a) {
    if (a.rows <= 16) return rows_kernel<1, 1, 8, 4>(stream, a);
    if (a.rows <= 32) return rows_kernel<2, 2, 8, 2>(stream, a);
    const int64_t tiles = static_cast<int64_t>((a.out_dim + 127) / 128) * ((a.rows + 127) / 128);
    if (a.rows <= 64 || tiles < gemv_compute_units()) return rows_kernel<4, 2, 4, 2>(stream, a);
    const dim3 grid((a.out_dim + 127) / 128, (a.rows + 127) / 128);
    matmul_fp8_tile_kernel<<<grid, 256, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace afhip
