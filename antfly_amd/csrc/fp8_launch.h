// Internal C++ interface between the 8-bit floating point kernels and the C ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "qmatmul_launch.h"

namespace afhip {

constexpr int kFp8Block = 128;  // values that share a scale

__host__ __device__ inline int fp8_blocks(int n) { return (n + kFp8Block - 1) / kFp8Block; }

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
hipError_t launch_matmul_fp8(hipStream_t stream, const Fp8Matmul& call);

}  // namespace afhip
