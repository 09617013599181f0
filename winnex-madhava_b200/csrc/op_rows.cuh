// The 8-bit row cache as kernels see it (rows.cu, attend.cu): its checked
// view, and the arithmetic of its codes.
#pragma once

#include "op_common.cuh"

namespace mdh {
namespace op {

struct RowsView {
    uint8_t* codes;
    float* scales;      // int8: [slots][n_groups]
    int64_t slots, stride;
    int width, group, n_groups;
    bool affine;        // uint8 codes: lo + step * code
    float lo, step, inv_step;
};

// Rows start and step on 8 bytes.
inline bool rows_on_8(const RowsView& r) { return reinterpret_cast<uintptr_t>(r.codes) % 8 == 0 && r.stride % 8 == 0; }

// Checks a caller's cache and gives its view; throws MDH_ERR_INVALID_ARG.
RowsView rows_view(const mdh_rows* c);

// The larger of two values >= 0, or NaN when either is NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Scale and inverse of a group with largest magnitude a.  Below 2^-100 the
// inverse would leave the float range: such groups are stored as zeros.  An
// infinity or NaN becomes the scale itself with all codes 0, so the group
// reads back as NaN.  Products by an inverse, each rounded, and not quotients
// rounded once: they are what torch's a / 127 and 127 / a compute on a GPU, so a
// program that quantises rows there gets the same codes bit for bit.  Against
// the quotients 4% of the scales move by their last bit (largest relative error
// 1.06 instead of 0.99 times 2^-24) and 0.8 codes in a million by one.
__device__ __forceinline__ void group_scale(float a, float& scale, float& inv) {
    const bool finite = a < INFINITY, some = a >= 0x1p-100f;
    scale = !finite ? a : some ? __fmul_rn(a, 1.0f / 127.0f) : 0.0f;
    inv = finite && some ? __fmul_rn(127.0f, __frcp_rn(a)) : 0.0f;
}
// In a group without a finite inverse x may be infinite or NaN: 0 * x is then
// NaN, which converts to 0.
__device__ __forceinline__ int group_code(float x, float inv) { return __float2int_rn(__fmul_rn(x, inv)); }
__device__ __forceinline__ uint8_t affine_code(float x, float lo, float inv_step) {
    const float v = __fmul_rn(__fsub_rn(x, lo), inv_step);
    return (uint8_t)__float2int_rn(fminf(fmaxf(v, 0.0f), 255.0f));
}
__device__ __forceinline__ float affine_value(uint8_t code, float lo, float step) {
    return __fadd_rn(lo, __fmul_rn(step, (float)code));
}

}  // namespace op
}  // namespace mdh
