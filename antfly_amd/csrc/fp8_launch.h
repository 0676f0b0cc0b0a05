// Internal C++ interface between the 8-bit floating point kernels and the C ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "qmatmul_launch.h"

namespace afhip {

constexpr int kFp8Block = 128;  // values that share a scale

__host__ __device__ inline int fp8_blocks(int n) { return (n + kFp8Block - 1) / kFp8Block; }

// Floats of a row of the sums of K's shares: whole vectors.
__host__ __device__ inline size_t fp8_sums_pitch(int out_dim) { return (static_cast<size_t>(out_dim) + 3) / 4 * 4; }

struct Fp8Matmul {
    const uint8_t* x;       // e4m3 [rows][in_dim]
    const float* x_scales;  // [rows][blocks of in_dim]
    const uint8_t* w;       // e4m3 [out_dim][in_dim]
    const float* w_scales;  // [blocks of out_dim][blocks of in_dim]
    float* y;               // [rows][out_dim]
    Epilogue ep;
    int rows, in_dim, out_dim;
};

hipError_t launch_quantize_fp8(hipStream_t stream, uint8_t* q, float* scales, const float* x, size_t rows, int in_dim);
// Few values of X: f32, quantized in the product's own launch (a.x and a.x_scales are not read).
bool linear_fp8_is_fused(int rows, int in_dim);
hipError_t launch_linear_fp8_fused(hipStream_t stream, const Fp8Matmul& call, const float* input, int compute_units);
// Which kernel, and over how many workgroups the blocks of K are shared out; `room`: bytes for the shares' sums.
enum Fp8Kernel { kFp8Rows16, kFp8Rows16Wide, kFp8Rows32, kFp8Rows32Wide, kFp8Rows48, kFp8Rows48Wide, kFp8Tile64, kFp8Tile128 };
struct Fp8Plan {
    Fp8Kernel kernel;
    int shares;
    size_t sums_bytes(int rows, int out_dim) const { return shares > 1 ? shares * rows * fp8_sums_pitch(out_dim) * sizeof(float) : 0; }
};
Fp8Plan plan_matmul_fp8(int rows, int in_dim, int out_dim, int compute_units, size_t room);
hipError_t launch_matmul_fp8(hipStream_t stream, const Fp8Matmul& call, const Fp8Plan& plan, float* sums);
// Whether their grids are within what a launch may have.
bool quantize_fp8_fits_a_launch(size_t rows, int in_dim);
bool linear_fp8_fused_fits_a_launch(int out_dim);
bool matmul_fp8_fits_a_launch(int rows, int out_dim, const Fp8Plan& plan);

}  // namespace afhip
