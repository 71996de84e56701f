// extern "C" layer of the feed-forward half of a transformer block: RMS norm with the residual's addition, the product of 8-bit operands
// and its quantiser, the gated transition, and the backward passes.  None of them has a counterpart in the reference.
#include <hip/hip_runtime.h>

#include <climits>

#include "api_internal.h"
#include "kutacc_hip.h"
#include "launch_internal.h"

namespace {
constexpr int64_t MAX_INDEX = INT32_MAX / 2; // extents that the kernels count in 32 bits
constexpr int64_t FP8_BLOCK = 128;

bool storage_type(int32_t dtype) { return dtype == KUTACC_DTYPE_BF16 || dtype == KUTACC_DTYPE_FP32; }
// a matrix that may be absent, and one that may not
bool optional_rows(const void *ptr, int64_t ld, int64_t size) { return ptr == nullptr || ld >= size; }
bool rows_of(const void *ptr, int64_t ld, int64_t size) { return ptr != nullptr && ld >= size; }
bool extent(int64_t v) { return v > 0 && v <= MAX_INDEX; }
int64_t blocks_of(int64_t v) { return (v + FP8_BLOCK - 1) / FP8_BLOCK; }
bool workspace_fits(const void *ptr, int64_t bytes, int64_t needed)
{
    return needed == 0 || (ptr != nullptr && bytes >= needed && (reinterpret_cast<uintptr_t>(ptr) & 255u) == 0);
}
} // namespace

extern "C" {

int kutacc_hip_rms_norm(const kutacc_hip_rms_norm_args_t *args, void *stream)
{
    if (args == nullptr) {
        return KUTACC_HIP_EINVAL;
    }
    const kutacc_hip_rms_norm_args_t &a = *args;
    if (a.rows < 0 || !extent(a.size) || !storage_type(a.dtype) || !(a.eps >= 0.f)) {
        return KUTACC_HIP_EINVAL;
    }
    if (a.rows == 0) {
        return 0;
    }
    if ((!a.out && !a.out8 && !a.sum) || (a.out8 != nullptr) != (a.scales != nullptr) || !rows_of(a.x, a.x_ld, a.size) || !optional_rows(a.residual, a.residual_ld, a.size) || !optional_rows(a.sum, a.sum_ld, a.size) ||
        !optional_rows(a.out, a.out_ld, a.size) || !optional_rows(a.out8, a.out8_ld, a.size) || !optional_rows(a.scales, a.scales_ld, blocks_of(a.size))) {
        return KUTACC_HIP_EINVAL;
    }
    if (!kutacc_launch::rms_norm_supports(a.size)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    return kutacc_launch::rms_norm(a, kutacc_api::stream_or_default(stream));
}

int64_t kutacc_hip_rms_norm_backward_workspace(int64_t rows, int64_t size)
{
    if (rows < 0 || !extent(size)) {
        return KUTACC_HIP_EINVAL;
    }
    return rows == 0 || !kutacc_launch::rms_norm_supports(size) ? 0 : kutacc_launch::rms_norm_backward_workspace(rows, size);
}

int kutacc_hip_rms_norm_backward(const kutacc_hip_rms_norm_backward_args_t *args, void *stream)
{
    if (args == nullptr) {
        return KUTACC_HIP_EINVAL;
    }
    const kutacc_hip_rms_norm_backward_args_t &a = *args;
    if (a.rows <= 0 || !extent(a.size) || !storage_type(a.dtype) || !(a.eps >= 0.f) || (!a.grad_x && !a.grad_gamma) || !rows_of(a.x, a.x_ld, a.size) ||
        !rows_of(a.grad_out, a.grad_out_ld, a.size) || !optional_rows(a.grad_sum, a.grad_sum_ld, a.size) || !optional_rows(a.grad_x, a.grad_x_ld, a.size)) {
        return KUTACC_HIP_EINVAL;
    }
    if (!kutacc_launch::rms_norm_supports(a.size)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    if (a.grad_gamma != nullptr && !workspace_fits(a.workspace, a.workspace_bytes, kutacc_launch::rms_norm_backward_workspace(a.rows, a.size))) {
        return KUTACC_HIP_EINVAL;
    }
    return kutacc_launch::rms_norm_backward(a, kutacc_api::stream_or_default(stream));
}

int kutacc_hip_quantize_fp8(const void *x, int64_t x_ld, void *out, int64_t out_ld, float *scales, int64_t scales_ld, int64_t rows, int64_t size,
                            int32_t block_rows, int32_t dtype, void *stream)
{
    if (rows < 0 || !extent(size) || !storage_type(dtype) || (block_rows != 1 && block_rows != FP8_BLOCK)) {
        return KUTACC_HIP_EINVAL;
    }
    if (rows == 0) {
        return 0;
    }
    if (!rows_of(x, x_ld, size) || !rows_of(out, out_ld, size) || !rows_of(scales, scales_ld, blocks_of(size))) {
        return KUTACC_HIP_EINVAL;
    }
    return kutacc_launch::quantize_fp8(x, x_ld, out, out_ld, scales, scales_ld, rows, size, block_rows, dtype, kutacc_api::stream_or_default(stream));
}

int kutacc_hip_linear_fp8(const kutacc_hip_linear_fp8_args_t *args, void *stream)
{
    if (args == nullptr) {
        return KUTACC_HIP_EINVAL;
    }
    const kutacc_hip_linear_fp8_args_t &a = *args;
    if (a.m < 0 || a.m > MAX_INDEX || !extent(a.n) || !extent(a.k) || !storage_type(a.dtype)) {
        return KUTACC_HIP_EINVAL;
    }
    if (a.m == 0) {
        return 0;
    }
    if (!rows_of(a.a, a.a_ld, a.k) || !rows_of(a.w, a.w_ld, a.k) || !rows_of(a.a_scales, a.a_scales_ld, blocks_of(a.k)) ||
        !rows_of(a.w_scales, a.w_scales_ld, blocks_of(a.k)) || !rows_of(a.out, a.out_ld, a.n)) {
        return KUTACC_HIP_EINVAL;
    }
    return kutacc_launch::linear_fp8(a, kutacc_api::stream_or_default(stream));
}

int64_t kutacc_hip_gated_transition_workspace(int64_t rows, int64_t c_o, int64_t c_i)
{
    if (rows < 0 || rows > MAX_INDEX || !extent(c_o) || !extent(c_i)) {
        return KUTACC_HIP_EINVAL;
    }
    return rows == 0 ? 0 : kutacc_launch::gated_transition_workspace(rows, c_o, c_i);
}

int kutacc_hip_gated_transition(const kutacc_hip_gated_transition_args_t *args, void *stream)
{
    if (args == nullptr) {
        return KUTACC_HIP_EINVAL;
    }
    const kutacc_hip_gated_transition_args_t &a = *args;
    if (a.rows < 0 || a.rows > MAX_INDEX || !extent(a.c_o) || !extent(a.c_i) || a.dtype != KUTACC_DTYPE_BF16 ||
        (a.activation != KUTACC_HIP_SILU && a.activation != KUTACC_HIP_GELU) || !a.gate_w || !a.up_w || !a.down_w) {
        return KUTACC_HIP_EINVAL;
    }
    if (a.rows == 0) {
        return 0;
    }
    if (!rows_of(a.x, a.x_ld, a.c_o) || !rows_of(a.out, a.out_ld, a.c_o) ||
        !workspace_fits(a.workspace, a.workspace_bytes, kutacc_launch::gated_transition_workspace(a.rows, a.c_o, a.c_i))) {
        return KUTACC_HIP_EINVAL;
    }
    return kutacc_launch::gated_transition(a, kutacc_api::stream_or_default(stream));
}

int64_t kutacc_hip_gated_transition_backward_workspace(int64_t rows, int64_t c_o, int64_t c_i)
{
    if (rows < 0 || rows > MAX_INDEX || !extent(c_o) || !extent(c_i)) {
        return KUTACC_HIP_EINVAL;
    }
    return rows == 0 ? 0 : kutacc_launch::gated_transition_backward_workspace(rows, c_o, c_i);
}

int kutacc_hip_gated_transition_backward(const kutacc_hip_gated_transition_backward_args_t *args, void *stream)
{
    if (args == nullptr) {
        return KUTACC_HIP_EINVAL;
    }
    const kutacc_hip_gated_transition_backward_args_t &a = *args;
    if (!extent(a.rows) || !extent(a.c_o) || !extent(a.c_i) || a.dtype != KUTACC_DTYPE_BF16 || (a.activation != KUTACC_HIP_SILU && a.activation != KUTACC_HIP_GELU) ||
        !a.gate_w || !a.up_w || !a.down_w || (!a.grad_x && !a.grad_gate_w && !a.grad_up_w && !a.grad_down_w) || !rows_of(a.x, a.x_ld, a.c_o) ||
        !rows_of(a.grad_out, a.grad_out_ld, a.c_o) || !optional_rows(a.grad_x, a.grad_x_ld, a.c_o) ||
        !workspace_fits(a.workspace, a.workspace_bytes, kutacc_launch::gated_transition_backward_workspace(a.rows, a.c_o, a.c_i))) {
        return KUTACC_HIP_EINVAL;
    }
    return kutacc_launch::gated_transition_backward(a, kutacc_api::stream_or_default(stream));
}

} // extern "C"
