// C ABI of the 8-bit floating point product: argument checks, the quantizer, the product.
#include <hip/hip_runtime_api.h>

#include "api_internal.h"
#include "fp8_launch.h"

using namespace afhip;

namespace {

constexpr size_t kInt32Max = 0x7fffffff;

bool aligned(afhip_buffer b, size_t to) { return b.ptr != 0 && b.ptr % to == 0; }

bool holds(afhip_buffer b, size_t count, size_t size, size_t alignment) {
    size_t bytes;
    return checked_mul(count, size, &bytes) && bytes <= b.len && (count == 0 || aligned(b, alignment));
}

size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

bool dims_fit(size_t rows, size_t in_dim, size_t out_dim) {
    size_t product;
    return in_dim != 0 && in_dim % 16 == 0 && in_dim <= kInt32Max - 127 && rows <= kInt32Max - 255 && out_dim <= kInt32Max - 255 &&
           checked_mul(rows, in_dim, &product) && product < (size_t{1} << 40) && checked_mul(rows, out_dim, &product) &&
           product < (size_t{1} << 40) && checked_mul(in_dim, out_dim, &product) && product < (size_t{1} << 40);
}

size_t codes_bytes(size_t rows, size_t in_dim) { return round_up(rows * in_dim); }
size_t scales_bytes(size_t rows, size_t in_dim) { return round_up(rows * ((in_dim + 127) / 128) * 4); }

afhip_status status_of(hipError_t e) { return e == hipSuccess ? AFHIP_OK : static_cast<afhip_status>(e); }

// What both products check of everything but the activations; fills the call.
afhip_status product_args(afhip_buffer dst, afhip_buffer weight, afhip_buffer weight_scales, afhip_buffer bias, afhip_buffer residual,
                          int activation, size_t rows, size_t in_dim, size_t out_dim, Fp8Matmul* call) {
    if (activation < AFHIP_ACTIVATION_NONE || activation > AFHIP_ACTIVATION_GELU) return AFHIP_ERR_INVALID_ARGUMENT;
    if (!dims_fit(rows, in_dim, out_dim)) return AFHIP_ERR_INVALID_STATE;
    const size_t kb = (in_dim + 127) / 128;
    if (!holds(dst, rows * out_dim, 4, 4) || !holds(weight, in_dim * out_dim, 1, 16) ||
        !holds(weight_scales, (out_dim + 127) / 128 * kb, 4, 4) || (bias.ptr != 0 && !holds(bias, out_dim, 4, 4)) ||
        (residual.ptr != 0 && !holds(residual, rows * out_dim, 4, 4)))
        return AFHIP_ERR_INVALID_STATE;
    if ((rows + 15) / 16 > 65535) return AFHIP_ERR_OP_UNSUPPORTED;  // row tiles of one launch
    *call = Fp8Matmul{};
    call->w = reinterpret_cast<const uint8_t*>(weight.ptr);
    call->w_scales = reinterpret_cast<const float*>(weight_scales.ptr);
    call->y = reinterpret_cast<float*>(dst.ptr);
    call->ep.bias = reinterpret_cast<const float*>(bias.ptr);
    call->ep.residual = reinterpret_cast<const float*>(residual.ptr);
    call->ep.activation = activation;
    call->rows = static_cast<int>(rows);
    call->in_dim = static_cast<int>(in_dim);
    call->out_dim = static_cast<int>(out_dim);
    return AFHIP_OK;
}

}  // namespace

extern "C" {

afhip_status afhip_launch_quantize_fp8(void* stream, afhip_buffer q, afhip_buffer scales, afhip_buffer input, size_t rows, size_t in_dim) {
    if (!dims_fit(rows, in_dim, 1)) return AFHIP_ERR_INVALID_STATE;
    if (!holds(input, rows * in_dim, 4, 16) || !holds(q, rows * in_dim, 1, 16) || !holds(scales, rows * ((in_dim + 127) / 128), 4, 4))
        return AFHIP_ERR_INVALID_STATE;
    if (rows == 0) return AFHIP_OK;
    if (!quantize_fp8_fits_a_launch(rows, static_cast<int>(in_dim))) return AFHIP_ERR_OP_UNSUPPORTED;
    return status_of(launch_quantize_fp8(static_cast<hipStream_t>(stream), reinterpret_cast<uint8_t*>(q.ptr), reinterpret_cast<float*>(scales.ptr),
                                         reinterpret_cast<const float*>(input.ptr), rows, static_cast<int>(in_dim)));
}

size_t afhip_linear_fp8_workspace_bytes(size_t rows, size_t in_dim, size_t out_dim) {
    if (!dims_fit(rows, in_dim, out_dim) || rows == 0 || out_dim == 0) return 0;
    const int r = static_cast<int>(rows), k = static_cast<int>(in_dim), n = static_cast<int>(out_dim);
    if (linear_fp8_is_fused(r, k)) return 0;
    return codes_bytes(rows, in_dim) + scales_bytes(rows, in_dim) + plan_matmul_fp8(r, k, n, gemv_compute_units(), SIZE_MAX).sums_bytes(r, n);
}

afhip_status afhip_launch_matmul_fp8_f32(void* stream, afhip_buffer dst, afhip_buffer q, afhip_buffer q_scales, afhip_buffer weight,
                                         afhip_buffer weight_scales, afhip_buffer bias, afhip_buffer residual, int activation, size_t rows,
                                         size_t in_dim, size_t out_dim, afhip_buffer workspace) {
    Fp8Matmul call;
    const afhip_status s = product_args(dst, weight, weight_scales, bias, residual, activation, rows, in_dim, out_dim, &call);
    if (s != AFHIP_OK) return s;
    if (!holds(q, rows * in_dim, 1, 16) || !holds(q_scales, rows * ((in_dim + 127) / 128), 4, 4)) return AFHIP_ERR_INVALID_STATE;
    if (rows == 0 || out_dim == 0) return AFHIP_OK;
    call.x = reinterpret_cast<const uint8_t*>(q.ptr);
    call.x_scales = reinterpret_cast<const float*>(q_scales.ptr);
    const bool lent = workspace.ptr != 0 && workspace.ptr % 256 == 0;
    const Fp8Plan plan = plan_matmul_fp8(call.rows, call.in_dim, call.out_dim, gemv_compute_units(), lent ? workspace.len : 0);
    if (!matmul_fp8_fits_a_launch(call.rows, call.out_dim, plan)) return AFHIP_ERR_OP_UNSUPPORTED;
    return status_of(launch_matmul_fp8(static_cast<hipStream_t>(stream), call, plan, reinterpret_cast<float*>(workspace.ptr)));
}

afhip_status afhip_launch_linear_fp8_f32(void* stream, afhip_buffer dst, afhip_buffer input, afhip_buffer weight, afhip_buffer weight_scales,
                                         afhip_buffer bias, afhip_buffer residual, int activation, size_t rows, size_t in_dim,
                                         size_t out_dim, afhip_buffer workspace) {
    Fp8Matmul call;
    const afhip_status s = product_args(dst, weight, weight_scales, bias, residual, activation, rows, in_dim, out_dim, &call);
    if (s != AFHIP_OK) return s;
    if (!holds(input, rows * in_dim, 4, 16)) return AFHIP_ERR_INVALID_STATE;
    if (rows == 0 || out_dim == 0) return AFHIP_OK;
    if (linear_fp8_is_fused(call.rows, call.in_dim)) {
        if (!linear_fp8_fused_fits_a_launch(call.out_dim)) return AFHIP_ERR_OP_UNSUPPORTED;
        return status_of(launch_linear_fp8_fused(static_cast<hipStream_t>(stream), call, reinterpret_cast<const float*>(input.ptr), gemv_compute_units()));
    }
    const size_t quantized = codes_bytes(rows, in_dim) + scales_bytes(rows, in_dim);
    if (!holds(workspace, quantized, 1, 256)) return AFHIP_ERR_INVALID_STATE;
    const Fp8Plan plan = plan_matmul_fp8(call.rows, call.in_dim, call.out_dim, gemv_compute_units(), workspace.len - quantized);
    if (!quantize_fp8_fits_a_launch(rows, call.in_dim) || !matmul_fp8_fits_a_launch(call.rows, call.out_dim, plan)) return AFHIP_ERR_OP_UNSUPPORTED;
    uint8_t* codes = reinterpret_cast<uint8_t*>(workspace.ptr);
    float* scales = reinterpret_cast<float*>(workspace.ptr + codes_bytes(rows, in_dim));
    const hipError_t e = launch_quantize_fp8(static_cast<hipStream_t>(stream), codes, scales, reinterpret_cast<const float*>(input.ptr), rows,
                                             static_cast<int>(in_dim));
    if (e != hipSuccess) return static_cast<afhip_status>(e);
    call.x = codes;
    call.x_scales = scales;
    return status_of(launch_matmul_fp8(static_cast<hipStream_t>(stream), call, plan, reinterpret_cast<float*>(workspace.ptr + quantized)));
}

}  // extern "C"
