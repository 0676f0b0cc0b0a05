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
#include <math.h>

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
//
// Bound by memory: 5 bytes a value, once.  Whole 128-byte lines in and 32-byte pieces out; the block's maximum takes three moves
// between neighbouring lanes.  2048 x 4096: 10 us (4.2 TB/s); 333 x 2000: 3 us, a launch's own time.
struct BlockPart {
    float4 v[4];
    __device__ __forceinline__ void load(const float* row, int block, int part, int in_dim) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = block * kFp8Block + i * 32 + part * 4;
            v[i] = k < in_dim ? *reinterpret_cast<const float4*>(row + k) : float4{0, 0, 0, 0};
        }
    }
    // four codes for each of the four parts; returns the block's scale
    __device__ __forceinline__ float quantize(int* codes) const {
        float most = kTiniest;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            most = fmaxf(most, fmaxf(fmaxf(__builtin_fabsf(v[i].x), __builtin_fabsf(v[i].y)), fmaxf(__builtin_fabsf(v[i].z), __builtin_fabsf(v[i].w))));
        most = max_over_8(most);
        const float by = kMost / most;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int low = __builtin_amdgcn_cvt_pk_fp8_f32(v[i].x * by, v[i].y * by, 0, false);
            codes[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[i].z * by, v[i].w * by, low, true);
        }
        return most / kMost;
    }
};

__global__ __launch_bounds__(256) void quantize_fp8_kernel(uint8_t* q, float* scales, const float* x, size_t blocks, int row_blocks, int in_dim) {
    const size_t at = static_cast<size_t>(blockIdx.x) * 32 + threadIdx.x / 8;
    if (at >= blocks) return;
    const size_t row = at / row_blocks;
    const int block = static_cast<int>(at % row_blocks), part = threadIdx.x & 7;
    BlockPart x_part;
    x_part.load(x + row * in_dim, block, part, in_dim);
    int codes[4];
    const float scale = x_part.quantize(codes);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = block * kFp8Block + i * 32 + part * 4;
        if (k < in_dim) *reinterpret_cast<int*>(q + row * in_dim + k) = codes[i];
    }
    if (part == 0) scales[at] = scale;
}

// ---- what both kernels share
//
// Codes come from memory straight into LDS, whole 128-byte blocks of a row, 1 KiB (eight rows) an instruction.  16-byte piece p
// of row r lies at place p ^ (r / 2 % 8) of the row's 128 bytes: the same piece of 16 rows, what an operand's lanes read, falls
// on all banks (two rows to 256 bytes).
__device__ const uint4 kNothing{0, 0, 0, 0};  // what pieces past in_dim are loaded from

__device__ __forceinline__ void load_to_lds(uint32_t to, const void* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void load_dword_to_lds(uint32_t to, const void* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}
// s_waitcnt for "at most kLeft vector memory operations outstanding" (nothing else waited for).
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLeft) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p));
}

// One float by a scalar load (a vector load would stand in the queue behind the blocks on their way, and wait for them).  The
// address is the same for the whole wavefront.
__device__ __forceinline__ float load_uniform(const float* p) { return *(const __attribute__((address_space(4))) float*)p; }

// Rows [first, first + 8) of a block to LDS (eight lanes a row); `rows`: how many the matrix has, `pieces`: of a row.
__device__ __forceinline__ void request_rows(uint32_t to, const uint8_t* matrix, int first, int in_tile, int rows, int in_dim, int block, int lane) {
    const int row = lane >> 3, piece = block * 8 + ((lane & 7) ^ ((in_tile + row) >> 1 & 7));
    const uint8_t* from = matrix + static_cast<size_t>(min(first + row, rows - 1)) * in_dim + piece * 16;
    load_to_lds(to, piece * 16 < in_dim ? static_cast<const void*>(from) : &kNothing);
}
__device__ __forceinline__ uint4 read_piece(const char* tile, int row, int piece) {
    return *reinterpret_cast<const uint4*>(tile + row * 128 + (piece ^ (row >> 1 & 7)) * 16);
}

// ---- few rows
//
// Bound by the weights' bytes, which all rows of a workgroup share.  A workgroup has 16 columns of W and 16 kM rows of X.  Its
// wavefronts share out the blocks of K in turn and add up at the end: each works alone, with a ring of kStages blocks in LDS (its
// W, X and X's scales) and no barrier in the loop, so that a few columns are enough to keep a compute unit's memory queue full.
// K = 4096, 14336 columns (59 MB, 11.4 us at a copy's rate): 1 row 11.9 us (4.9 TB/s), 16 rows 12.6, 32 rows 17.8, 48 rows 20.8;
// past one sixteen it is X, read by every workgroup from L2 into LDS, that takes the time.
template <int kM, int kWaves, int kStages>
__global__ __launch_bounds__(kWaves * 64) void matmul_fp8_rows_kernel(Fp8Matmul a) {
    constexpr int kRows = 16 * kM, kStage = 2048 + kRows * 128 + 256;  // W, X, a scale a row
    constexpr int kLoads = 2 + 2 * kM + 1;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, column = lane & 15, quarter = lane >> 4;
    const int first_o = blockIdx.x * 16, first_r = blockIdx.y * kRows;
    const int blocks = fp8_blocks(a.in_dim);
    const float* w_scale = a.w_scales + static_cast<size_t>(first_o / kFp8Block) * blocks;
    char* ring = lds + wave * (kStages * kStage);
    const uint32_t ring_at = lds_address(ring);
    const float* x_scale = a.x_scales + static_cast<size_t>(min(first_r + min(lane, kRows - 1), a.rows - 1)) * blocks;

    auto request = [&](int block, int stage) {
        const uint32_t to = ring_at + stage * kStage;
#pragma unroll
        for (int i = 0; i < 2; ++i) request_rows(to + i * 1024, a.w, first_o + i * 8, i * 8, a.out_dim, a.in_dim, block, lane);
#pragma unroll
        for (int i = 0; i < 2 * kM; ++i) request_rows(to + 2048 + i * 1024, a.x, first_r + i * 8, i * 8, a.rows, a.in_dim, block, lane);
        load_dword_to_lds(to + 2048 + kRows * 128, x_scale + block);
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (wave + i * kWaves < blocks) request(wave + i * kWaves, i);
    }
    f32x4 total[kM];
#pragma unroll
    for (int m = 0; m < kM; ++m) total[m] = f32x4{0, 0, 0, 0};
    int stage = 0, free_stage = kStages - 1;
    float ws_ahead = wave < blocks ? load_uniform(w_scale + wave) : 0.0f;
    for (int b = wave; b < blocks; b += kWaves) {
        if (b + (kStages - 2) * kWaves < blocks) wait_loads<kLoads * (kStages - 2)>();
        else wait_loads<0>();
        if (b + (kStages - 1) * kWaves < blocks) request(b + (kStages - 1) * kWaves, free_stage);
        const char* w = ring + stage * kStage;
        const char* x = w + 2048;
        const float* scales = reinterpret_cast<const float*>(x + kRows * 128);
        stage = stage + 1 == kStages ? 0 : stage + 1;
        free_stage = free_stage + 1 == kStages ? 0 : free_stage + 1;
        const float ws = ws_ahead;
        if (b + kWaves < blocks) ws_ahead = load_uniform(w_scale + b + kWaves);
        f32x4 dot[kM];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint4 wp = read_piece(w, column, k * 4 + quarter);
            const f16x8 w0 = widen(wp.x, wp.y), w1 = widen(wp.z, wp.w);
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                const uint4 xp = read_piece(x + m * 2048, column, k * 4 + quarter);
                dot[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w0, widen(xp.x, xp.y), k == 0 ? f32x4{0, 0, 0, 0} : dot[m], 0, 0, 0);
                dot[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w1, widen(xp.z, xp.w), dot[m], 0, 0, 0);
            }
        }
#pragma unroll
        for (int m = 0; m < kM; ++m) {
            const float scale = scales[m * 16 + column] * ws;
#pragma unroll
            for (int j = 0; j < 4; ++j) total[m][j] = __builtin_fmaf(dot[m][j], scale, total[m][j]);
        }
    }
    constexpr int kPitch = 20;  // floats of a row's 16 columns
    float* sums = reinterpret_cast<float*>(lds);  // [kWaves][kRows][kPitch]
    __syncthreads();                              // everyone is done with the ring
#pragma unroll
    for (int m = 0; m < kM; ++m) *reinterpret_cast<f32x4*>(sums + (wave * kRows + m * 16 + column) * kPitch + quarter * 4) = total[m];
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * 16; i += kWaves * 64) {
        const int m = i / 16, n = i % 16, row = first_r + m, o = first_o + n;
        if (row >= a.rows || o >= a.out_dim) continue;
        float v = 0.0f;
#pragma unroll
        for (int s = 0; s < kWaves; ++s) v += sums[(s * kRows + m) * kPitch + n];
        const size_t to = static_cast<size_t>(row) * a.out_dim + o;
        a.y[to] = finish_output(a.ep, o, to, v);
    }
}

// ---- few values of X: quantized by every workgroup itself
//
// While the first blocks of W are on their way, a workgroup quantizes all of X (up to 16 rows, kFusedValues values) into LDS: one
// launch instead of two, and X read by every workgroup from L2.  1 row: 4096 x 4096 5.2 us (3.2 TB/s: start, one round
// trip to memory and the sums are most of it), 4096 x 14336 12.3 us (4.8 TB/s).
template <int kWaves, int kStages>
__global__ __launch_bounds__(kWaves * 64) void linear_fp8_rows_kernel(Fp8Matmul a, const float* input) {
    constexpr int kLoads = 2;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, column = lane & 15, quarter = lane >> 4;
    const int first_o = blockIdx.x * 16, blocks = fp8_blocks(a.in_dim);
    const float* w_scale = a.w_scales + static_cast<size_t>(first_o / kFp8Block) * blocks;
    char* ring = lds + wave * (kStages * 2048);
    const uint32_t ring_at = lds_address(ring);
    const int x_pitch = blocks * kFp8Block + 16;  // bytes of a row of codes: rows fall on other banks
    char* x_codes = lds + kWaves * kStages * 2048;
    float* x_scales = reinterpret_cast<float*>(x_codes + a.rows * x_pitch);  // [rows][blocks]

    const int parts = a.rows * blocks, part = threadIdx.x & 7;
    BlockPart first_part;
    const int mine = threadIdx.x / 8;
    if (mine < parts) first_part.load(input + static_cast<size_t>(mine / blocks) * a.in_dim, mine % blocks, part, a.in_dim);
    auto request = [&](int block, int stage) {
#pragma unroll
        for (int i = 0; i < 2; ++i) request_rows(ring_at + stage * 2048 + i * 1024, a.w, first_o + i * 8, i * 8, a.out_dim, a.in_dim, block, lane);
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (wave + i * kWaves < blocks) request(wave + i * kWaves, i);
    }
    for (int at = mine; at < parts; at += kWaves * 8) {
        const int row = at / blocks, block = at % blocks;
        if (at != mine) first_part.load(input + static_cast<size_t>(row) * a.in_dim, block, part, a.in_dim);
        int codes[4];
        const float scale = first_part.quantize(codes);
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<int*>(x_codes + row * x_pitch + block * kFp8Block + i * 32 + part * 4) = codes[i];
        if (part == 0) x_scales[at] = scale;
    }
    __syncthreads();
    const int row = min(column, a.rows - 1);
    const char* x = x_codes + row * x_pitch;
    f32x4 total{0, 0, 0, 0};
    int stage = 0, free_stage = kStages - 1;
    float ws_ahead = wave < blocks ? load_uniform(w_scale + wave) : 0.0f;
    for (int b = wave; b < blocks; b += kWaves) {
        if (b + (kStages - 2) * kWaves < blocks) wait_loads<kLoads * (kStages - 2)>();
        else wait_loads<0>();
        if (b + (kStages - 1) * kWaves < blocks) request(b + (kStages - 1) * kWaves, free_stage);
        const char* w = ring + stage * 2048;
        stage = stage + 1 == kStages ? 0 : stage + 1;
        free_stage = free_stage + 1 == kStages ? 0 : free_stage + 1;
        const float ws = ws_ahead;
        if (b + kWaves < blocks) ws_ahead = load_uniform(w_scale + b + kWaves);
        f32x4 dot{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint4 wp = read_piece(w, column, k * 4 + quarter);
            const uint4 xp = *reinterpret_cast<const uint4*>(x + b * kFp8Block + (k * 4 + quarter) * 16);
            dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(wp.x, wp.y), widen(xp.x, xp.y), dot, 0, 0, 0);
            dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(wp.z, wp.w), widen(xp.z, xp.w), dot, 0, 0, 0);
        }
        const float scale = x_scales[row * blocks + b] * ws;
#pragma unroll
        for (int j = 0; j < 4; ++j) total[j] = __builtin_fmaf(dot[j], scale, total[j]);
    }
    constexpr int kPitch = 20;
    float* sums = reinterpret_cast<float*>(lds);  // [kWaves][16][kPitch]
    __syncthreads();
    *reinterpret_cast<f32x4*>(sums + (wave * 16 + column) * kPitch + quarter * 4) = total;
    __syncthreads();
    if (threadIdx.x < static_cast<unsigned>(a.rows) * 16) {
        const int m = threadIdx.x / 16, n = threadIdx.x % 16, o = first_o + n;
        if (o >= a.out_dim) return;
        float v = 0.0f;
#pragma unroll
        for (int s = 0; s < kWaves; ++s) v += sums[(s * 16 + m) * kPitch + n];
        const size_t to = static_cast<size_t>(m) * a.out_dim + o;
        a.y[to] = finish_output(a.ep, o, to, v);
    }
}

// ---- many rows
//
// kRowWaves x kColWaves wavefronts with 32 kR rows x 64 columns each, a block of K at a time from a ring of kStages in LDS that all
// of them fill and read.  Every wavefront widens its own operands: of a block's instructions about half are conversions, which
// run beside another wavefront's products.  128 x 128 with a ring of two is two workgroups a compute unit (66 KiB of LDS and 210
// registers each), whose barriers, waits and last stores fall into the other's products: 2048 x 4096 x 14336 248 us (970 TFLOP/s), a
// ring of three and one workgroup 310 us, 256 x 128 and a ring of three 278 us; a library's f16 product of that size takes 212 us.
// What is left is the matrix instructions' own time at the clock that they are given on dense data and the conversions' issue.
// 64 x 128 with a ring of three fills the units where there are few rows, and has the registers for all of a block's pieces at once
// (one workgroup a unit: 29 us instead of 35): 256 x 4096 x 4096 30 us, 128 x 128 42 (no shares).
// `sums`: blocks of K are shared out over gridDim.y workgroups, whose sums go there, [share][rows][out_dim rounded up to 4], for
// add_shares_kernel.
template <int kR, int kRowWaves, int kColWaves, int kStages>
__global__ __launch_bounds__(kRowWaves * kColWaves * 64, 2) void matmul_fp8_tile_kernel(Fp8Matmul a, int row_tiles, int col_tiles, float* sums) {
    constexpr int kWaves = kRowWaves * kColWaves, kRows = 32 * kR * kRowWaves, kCols = 64 * kColWaves;
    constexpr int kStage = (kRows + kCols) * 128 + kWaves * 256;                 // W, X, X's scales
    constexpr int kWLoads = kCols / 8 / kWaves, kXLoads = kRows / 8 / kWaves, kLoads = kWLoads + kXLoads + 1;
    constexpr int kOwn = kRows / kWaves;                                         // rows whose scales a wavefront loads
    static_assert(kOwn <= 64 && kOwn % 8 == 0 && kWLoads > 0, "");
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, column = lane & 31, half = lane >> 5;
    // An XCD has neighbouring columns of tiles, row tile by row tile: what its units load at a time fits its L2.
    const int per_xcd = (col_tiles + 7) / 8, local = blockIdx.x >> 3;
    const int col_tile = (blockIdx.x & 7) * per_xcd + local / row_tiles, row_tile = local % row_tiles;
    if (local / row_tiles >= per_xcd || col_tile >= col_tiles) return;
    const int first_o = col_tile * kCols, first_r = row_tile * kRows;
    const int wave_o = wave % kColWaves * 64, wave_r = wave / kColWaves * (32 * kR);
    const int blocks = fp8_blocks(a.in_dim), each = (blocks + gridDim.y - 1) / gridDim.y;
    const int first_block = blockIdx.y * each, end_block = min(first_block + each, blocks);  // (a last share may be empty: sums of zero)
    const float* w_scale = a.w_scales + static_cast<size_t>(min(first_o + wave_o, a.out_dim - 1) / kFp8Block) * blocks;
    const float* x_scale = a.x_scales + static_cast<size_t>(min(first_r + wave * kOwn + lane % kOwn, a.rows - 1)) * blocks;
    const uint32_t ring_at = lds_address(lds);

    auto request = [&](int block, int stage) {
        const uint32_t to = ring_at + stage * kStage;
#pragma unroll
        for (int i = 0; i < kWLoads; ++i) {
            const int at = (wave * kWLoads + i) * 8;
            request_rows(to + at * 128, a.w, first_o + at, at, a.out_dim, a.in_dim, block, lane);
        }
#pragma unroll
        for (int i = 0; i < kXLoads; ++i) {
            const int at = (wave * kXLoads + i) * 8;
            request_rows(to + (kCols + at) * 128, a.x, first_r + at, at, a.rows, a.in_dim, block, lane);
        }
        load_dword_to_lds(to + (kCols + kRows) * 128 + wave * 256, x_scale + block);
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (first_block + i < end_block) request(first_block + i, i);
    }
    f32x16 total[2][kR];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int m = 0; m < kR; ++m) total[n][m] = f32x16{};
    }
    int stage = 0, free_stage = kStages - 1;
    float ws_ahead = first_block < end_block ? load_uniform(w_scale + first_block) : 0.0f;
    for (int b = first_block; b < end_block; ++b) {
        if (b + kStages - 2 < end_block) wait_loads<kLoads * (kStages - 2)>();
        else wait_loads<0>();
        __syncthreads();  // everyone's part of the block is there, and the stage to be filled has been read
        if (b + kStages - 1 < end_block) request(b + kStages - 1, free_stage);
        const char* w = lds + stage * kStage + wave_o * 128;
        const char* x = lds + stage * kStage + (kCols + wave_r) * 128;
        const float* scales = reinterpret_cast<const float*>(lds + stage * kStage + (kCols + kRows) * 128);
        stage = stage + 1 == kStages ? 0 : stage + 1;
        free_stage = free_stage + 1 == kStages ? 0 : free_stage + 1;
        const float ws = ws_ahead;
        if (b + 1 < end_block) ws_ahead = load_uniform(w_scale + b + 1);
        float scale[kR];
#pragma unroll
        for (int m = 0; m < kR; ++m) {
            const int row = wave_r + m * 32 + column;
            scale[m] = scales[row / kOwn * 64 + row % kOwn] * ws;
        }
        f32x16 dot[2][kR];
        constexpr int kHeld = kR == 1 ? 4 : 1;  // steps whose pieces are requested together, as registers allow
#pragma unroll
        for (int k0 = 0; k0 < 4; k0 += kHeld) {  // 32 of K a step: a 16-byte piece a lane, two instructions' worth
            uint4 w_piece[kHeld][2], x_piece[kHeld][kR];
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
#pragma unroll
                for (int n = 0; n < 2; ++n) w_piece[i][n] = read_piece(w + n * 4096, column, (k0 + i) * 2 + half);
#pragma unroll
                for (int m = 0; m < kR; ++m) x_piece[i][m] = read_piece(x + m * 4096, column, (k0 + i) * 2 + half);
            }
            if (kHeld > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                f16x8 wide_w[2][2], wide_x[kR][2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    wide_w[n][0] = widen(w_piece[i][n].x, w_piece[i][n].y);
                    wide_w[n][1] = widen(w_piece[i][n].z, w_piece[i][n].w);
                }
#pragma unroll
                for (int m = 0; m < kR; ++m) {
                    wide_x[m][0] = widen(x_piece[i][m].x, x_piece[i][m].y);
                    wide_x[m][1] = widen(x_piece[i][m].z, x_piece[i][m].w);
                }
#pragma unroll
                for (int part = 0; part < 2; ++part) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
#pragma unroll
                        for (int m = 0; m < kR; ++m)
                            dot[n][m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wide_w[n][part], wide_x[m][part], k0 + i + part == 0 ? f32x16{} : dot[n][m], 0, 0, 0);
                    }
                }
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int m = 0; m < kR; ++m) {
#pragma unroll
                for (int j = 0; j < 16; ++j) total[n][m][j] = __builtin_fmaf(dot[n][m][j], scale[m], total[n][m][j]);
            }
        }
    }
    const size_t pitch = sums != nullptr ? fp8_sums_pitch(a.out_dim) : a.out_dim;
    float* y = sums != nullptr ? sums + blockIdx.y * pitch * a.rows : a.y;
    // Through LDS into whole rows of 64 columns: a lane has four neighbouring columns of every fourth row, whose bias it loads once,
    // and the residual's loads of 32 rows go out together, ahead of the stores (the residual may be Y itself).  2048 x 4096 x 14336 with
    // bias, GELU and residual 296 us; from the registers as they stand, 16 bytes of 32 rows at a time, 380 (without them the same).
    const bool fours = pitch % 4 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0 && reinterpret_cast<uintptr_t>(a.ep.residual) % 16 == 0;
    const bool finish = sums == nullptr;
    const int o = first_o + wave_o + lane % 16 * 4;
    constexpr int kPitch = 68;
    float* own = reinterpret_cast<float*>(lds) + wave * 32 * kPitch;
    f32x4 bias{0, 0, 0, 0};
    if (finish && a.ep.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j) bias[j] = o + j < a.out_dim ? a.ep.bias[o + j] : 0.0f;
    }
    __syncthreads();  // everyone is done with the ring
#pragma unroll
    for (int m = 0; m < kR; ++m) {
        const int row = first_r + wave_r + m * 32 + lane / 16;  // and every fourth from there
        f32x4 residual[8];
        if (finish && a.ep.residual != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const size_t at = static_cast<size_t>(min(row + i * 4, a.rows - 1)) * pitch;
                if (fours) {
                    residual[i] = *reinterpret_cast<const f32x4*>(a.ep.residual + at + min(o, a.out_dim - 4));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) residual[i][j] = a.ep.residual[at + min(o + j, a.out_dim - 1)];
                }
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 v;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = total[n][m][q * 4 + j];
                *reinterpret_cast<f32x4*>(own + column * kPitch + n * 32 + q * 8 + half * 4) = v;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f32x4 v = *reinterpret_cast<const f32x4*>(own + (i * 4 + lane / 16) * kPitch + lane % 16 * 4);
            if (finish) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (a.ep.bias != nullptr) v[j] += bias[j];
                    v[j] = activate(a.ep.activation, v[j]);
                    if (a.ep.residual != nullptr) v[j] += residual[i][j];
                }
            }
            if (row + i * 4 >= a.rows || o >= a.out_dim) continue;
            float* to = y + static_cast<size_t>(row + i * 4) * pitch + o;
            if (fours) {
                *reinterpret_cast<f32x4*>(to) = v;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (o + j < a.out_dim) to[j] = v[j];
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// The sums of the shares of K, in their order, and what follows them: four columns a thread, 1024 of a row a workgroup.  Bound by
// their bytes, most of them still in the caches: 8 shares of 48 x 4096 4 us.
__global__ __launch_bounds__(256) void add_shares_kernel(Fp8Matmul a, const float* sums, int shares) {
    const size_t pitch = fp8_sums_pitch(a.out_dim);
    const int parts = (a.out_dim + 1023) / 1024, row = blockIdx.x / parts, o = (blockIdx.x % parts * 256 + threadIdx.x) * 4;
    if (o >= a.out_dim) return;
    f32x4 v{0, 0, 0, 0};
#pragma unroll 4
    for (int s = 0; s < shares; ++s) v += *reinterpret_cast<const f32x4*>(sums + (static_cast<size_t>(s) * a.rows + row) * pitch + o);
    const size_t to = static_cast<size_t>(row) * a.out_dim + o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // (all loads ahead of the stores)
        if (o + j < a.out_dim) v[j] = finish_output(a.ep, o + j, to + j, v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (o + j < a.out_dim) a.y[to + j] = v[j];
    }
}

template <int kM, int kWaves, int kStages>
hipError_t rows_kernel(hipStream_t stream, const Fp8Matmul& a) {
    static LdsLimit limit;
    constexpr size_t ring = static_cast<size_t>(kWaves) * kStages * (2048 + kM * 2048 + 256), sums = static_cast<size_t>(kWaves) * 16 * kM * 20 * 4;
    constexpr size_t lds = ring > sums ? ring : sums;
    const auto kernel = matmul_fp8_rows_kernel<kM, kWaves, kStages>;
    const hipError_t e = allow_lds(kernel, lds, &limit);
    if (e != hipSuccess) return e;
    const dim3 grid((a.out_dim + 15) / 16, (a.rows + 16 * kM - 1) / (16 * kM));
    kernel<<<grid, kWaves * 64, lds, stream>>>(a);
    return hipGetLastError();
}

template <int kR, int kRowWaves, int kColWaves, int kStages>
hipError_t tile_kernel(hipStream_t stream, const Fp8Matmul& a, int shares, float* sums) {
    static LdsLimit limit;
    constexpr int kRows = 32 * kR * kRowWaves, kCols = 64 * kColWaves;
    constexpr size_t lds = kStages * ((kRows + kCols) * 128 + kRowWaves * kColWaves * 256);
    static_assert(lds >= kRowWaves * kColWaves * 32 * 68 * 4, "the results' way through LDS");
    const auto kernel = matmul_fp8_tile_kernel<kR, kRowWaves, kColWaves, kStages>;
    hipError_t e = allow_lds(kernel, lds, &limit);
    if (e != hipSuccess) return e;
    const int row_tiles = (a.rows + kRows - 1) / kRows, col_tiles = (a.out_dim + kCols - 1) / kCols;
    const dim3 grid((col_tiles + 7) / 8 * 8 * row_tiles, shares);
    kernel<<<grid, kRowWaves * kColWaves * 64, lds, stream>>>(a, row_tiles, col_tiles, shares > 1 ? sums : nullptr);
    e = hipGetLastError();
    if (e != hipSuccess || shares == 1) return e;
    add_shares_kernel<<<static_cast<uint32_t>(a.rows) * static_cast<uint32_t>((a.out_dim + 1023) / 1024), 256, 0, stream>>>(a, sums, shares);
    return hipGetLastError();
}

template <int kWaves, int kStages>
hipError_t fused_kernel(hipStream_t stream, const Fp8Matmul& a, const float* input) {
    static LdsLimit limit;
    const size_t blocks = fp8_blocks(a.in_dim);
    const size_t lds = kWaves * kStages * 2048 + a.rows * (blocks * kFp8Block + 16 + blocks * 4);
    const auto kernel = linear_fp8_rows_kernel<kWaves, kStages>;
    const hipError_t e = allow_lds(kernel, lds, &limit);
    if (e != hipSuccess) return e;
    kernel<<<(a.out_dim + 15) / 16, kWaves * 64, lds, stream>>>(a, input);
    return hipGetLastError();
}

// Workgroups of 16 columns for more than two rounds and a half on the compute units.
bool is_wide(int out_dim, int compute_units) { return (out_dim + 15) / 16 >= compute_units * 5 / 2; }

}  // namespace

hipError_t launch_quantize_fp8(hipStream_t stream, uint8_t* q, float* scales, const float* x, size_t rows, int in_dim) {
    const int row_blocks = fp8_blocks(in_dim);
    const size_t blocks = rows * row_blocks;
    quantize_fp8_kernel<<<static_cast<uint32_t>((blocks + 31) / 32), 256, 0, stream>>>(q, scales, x, blocks, row_blocks, in_dim);
    return hipGetLastError();
}

bool quantize_fp8_fits_a_launch(size_t rows, int in_dim) { return fits_a_launch((rows * fp8_blocks(in_dim) + 31) / 32, 256); }

// (512 threads: the most that a workgroup of 16 columns has)
bool linear_fp8_fused_fits_a_launch(int out_dim) { return fits_a_launch((static_cast<uint64_t>(out_dim) + 15) / 16, 512); }

bool matmul_fp8_fits_a_launch(int rows, int out_dim, const Fp8Plan& plan) {
    if (plan.kernel != kFp8Tile64 && plan.kernel != kFp8Tile128) return linear_fp8_fused_fits_a_launch(out_dim);
    const uint64_t tile = plan.kernel == kFp8Tile64 ? 64 : 128;
    return fits_a_launch((static_cast<uint64_t>(out_dim) + 1023) / 1024 * 8 * ((rows + tile - 1) / tile), 256) &&
           (plan.shares == 1 || fits_a_launch(static_cast<uint64_t>(rows) * ((static_cast<uint64_t>(out_dim) + 1023) / 1024), 256));
}

// Up to how many values of X every workgroup quantizes them itself.
constexpr int64_t kFusedValues = 16384;

bool linear_fp8_is_fused(int rows, int in_dim) { return rows <= 16 && static_cast<int64_t>(rows) * in_dim <= kFusedValues; }

hipError_t launch_linear_fp8_fused(hipStream_t stream, const Fp8Matmul& a, const float* input, int compute_units) {
    // Two workgroups or more on a unit (by LDS), and as many as leave no unit idle for long in a last round: many columns four
    // wavefronts a workgroup, few eight.  K = 4096: 1 row on 8192 columns 8.7 us with eight and 10.0 with four, 4 rows 12.8 with a
    // ring of four (one workgroup a unit) and 11.2 with three; 1 row on 14336 columns 14.5 with eight and 12.3 with four, 4 rows 21.8
    // and 15.9.
    if (is_wide(a.out_dim, compute_units)) return fused_kernel<4, 2>(stream, a, input);
    if (a.rows * a.in_dim > 8192) return fused_kernel<8, 3>(stream, a, input);
    return fused_kernel<8, 4>(stream, a, input);
}

// What the kernels take, in us, as measured (512 to 14336 columns, K = 1024 to 14336, 24 to 2048 rows): few rows pass over W
// once for each 32 or 48 of them, 4 and 5 us for 2^24 weights (less on a long K); tiles take rounds of workgroups on the compute units, a time for each block
// of K (64 rows: two workgroups a unit); sums of shares are written and read at 5 TB/s.  Below them 3 or 4 us of a launch.
Fp8Plan plan_matmul_fp8(int rows, int in_dim, int out_dim, int compute_units, size_t room) {
    // Workgroups of four wavefronts instead of eight where those of eight would leave units idle in their last rounds: K = 4096, 16
    // rows on 4096 columns 5.8 us with eight and 6.4 with four, on 14336 15.7 and 12.9; 32 rows (one workgroup of eight a unit) on 4096
    // columns 6.6 and 7.6, on 14336 20.4 and 18.0, on 57344 59 and 65; 48 rows on 4096 columns 7.7 and 8.5, on 6144 12.2 and 10.7.
    const double units = compute_units, blocks = fp8_blocks(in_dim), weights = static_cast<double>(in_dim) * out_dim;
    const auto groups = [&](int of) { return static_cast<double>((out_dim + 15) / 16) * ((rows + of - 1) / of); };
    const auto half_filled = [&](int of) { return groups(of) > 1.25 * units && groups(of) < 8 * units; };
    const Fp8Kernel rows16 = is_wide(out_dim, compute_units) ? kFp8Rows16Wide : kFp8Rows16;
    Fp8Plan best{rows16, 1};
    if (rows <= 16) return best;
    // 32 or 48 rows a workgroup: a pass over W takes less than its rows' share longer (48 rows on 4096 x 4096: 10.4 us in two passes, 7.7 in one).
    const double shorter = fmin(2.2, 4096.0 / in_dim);
    const auto passes = [&](int of, double each, double partly) {  // `each`: 2^24 weights by workgroups that fill the units
        return each * (units * 16 * in_dim / (1 << 24)) * (half_filled(of) ? partly * groups(of) / units : fmax(groups(of) / units, 0.75));
    };
    const double by32 = passes(32, 2.3 + 1.2 * shorter, 1.25), by48 = passes(48, 3.75 + 1.15 * shorter, 1.05);
    double least = 3 + fmin(by32, by48);
    if (weights > (4 << 20)) {
        best.kernel = by32 <= by48 ? (half_filled(32) ? kFp8Rows32Wide : kFp8Rows32) : (half_filled(48) ? kFp8Rows48Wide : kFp8Rows48);
    } else {
        // W stays in every XCD's L2 (4 MiB) over its passes: 16 rows a workgroup, many workgroups (of four wavefronts where they are
        // more than two a unit).  Bias, GELU and residual with it: 333 rows on 2000 x 1111 9.4 us, with eight wavefronts 10.7, 32 rows a
        // workgroup 9.5 and 12.4; 512 rows on 768 x 2304 11.6, 16.6, 11.4, 18.5.
        if (groups(16) >= 2.5 * units) best.kernel = kFp8Rows16Wide;
        least = 3 + (0.95 + 1.4 * fmin(2.2, 1024.0 / in_dim)) * ((rows + 15) / 16) * (weights / (1 << 24));
    }
    const auto tiles = [&](int of) { return static_cast<double>((out_dim + 127) / 128) * ((rows + of - 1) / of); };
    // Two workgroups a compute unit at a time, `two` a block of K; a last round of one a unit takes `one`.
    const auto rounds = [&](double n, double one, double two) {
        const double full = floor(n / (2 * units)), left = n - full * 2 * units;
        return full * two + (left > units ? two : left > 0 ? one : 0);
    };
    for (int shares = 1; shares <= 8; shares *= 2) {
        const size_t sums = Fp8Plan{kFp8Tile64, shares}.sums_bytes(rows, out_dim);
        if (shares > 1 && (sums > room || blocks < 4 * shares)) break;
        const double each = ceil(blocks / shares), rest = 4 + (shares > 1 ? 3 + 2.0 * sums / 5e6 : 0.0);
        const double t64 = rest + each * rounds(tiles(64) * shares, 0.80, 1.30), t128 = rest + each * rounds(tiles(128) * shares, 1.22, 1.98);
        if (t64 < least) least = t64, best = Fp8Plan{kFp8Tile64, shares};
        if (t128 < least) least = t128, best = Fp8Plan{kFp8Tile128, shares};
    }
    return best;
}

hipError_t launch_matmul_fp8(hipStream_t stream, const Fp8Matmul& a, const Fp8Plan& plan, float* sums) {
    switch (plan.kernel) {
        case kFp8Rows16: return rows_kernel<1, 8, 2>(stream, a);
        case kFp8Rows16Wide: return rows_kernel<1, 4, 2>(stream, a);
        case kFp8Rows32: return rows_kernel<2, 8, 2>(stream, a);
        case kFp8Rows32Wide: return rows_kernel<2, 4, 2>(stream, a);
        case kFp8Rows48: return rows_kernel<3, 8, 2>(stream, a);
        case kFp8Rows48Wide: return rows_kernel<3, 4, 2>(stream, a);
        case kFp8Tile64: return tile_kernel<1, 2, 2, 3>(stream, a, plan.shares, sums);
        default: return tile_kernel<2, 2, 2, 2>(stream, a, plan.shares, sums);
    }
}

}  // namespace afhip
