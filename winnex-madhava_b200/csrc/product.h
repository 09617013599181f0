// Tensor-core product with an epilogue (product.cu), used by linear.cu.
#pragma once

#include "op_common.cuh"

namespace mdh {
namespace op {

// An operand of C[m][n] = sum_k a(m, k) b(n, k): element (row, k) is at
// p[row * stride + k] (k_major) or at p[k * stride + row].
struct ProductOperand {
    const void* p;
    int64_t stride;
    bool k_major;
};

// y = act(C + bias) + residual; z = C + bias (before the activation).
// Elements are bfloat16 or float16; null parts are left out.
struct ProductEpilogue {
    const void* bias = nullptr;      // [n]
    const void* residual = nullptr;  // [m][n], residual_stride
    int64_t residual_stride = 0;
    int act = MDH_ACT_NONE;
    void* y = nullptr;  // [m][n], y_stride
    int64_t y_stride = 0;
    void* z = nullptr;  // [m][n] contiguous
};

// Scratch of one product: copies of operands that TMA cannot read in place,
// and the partial sums of a split k.
int64_t product_workspace(const ProductOperand& a, const ProductOperand& b, int64_t m, int64_t n, int64_t k);
void product(const ProductOperand& a, const ProductOperand& b, int64_t m, int64_t n, int64_t k, int32_t dtype,
             const ProductEpilogue& ep, void* ws, cudaStream_t st);

// Throws MDH_ERR_TIMEOUT when a product on the current device gave up one of its
// waits since the last call of this.
void check_product_status();
// Records what such a product does.
void set_product_expired();

// 2^x and 1 / x by the hardware (relative errors about 2^-22 and 2^-23).
__device__ __forceinline__ float fast_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float fast_inverse(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ f32x2 both(float v) { return pair(v, v); }
// e^x of both values.
__device__ __forceinline__ f32x2 exp_of(f32x2 x) {
    const float2 f = unpair(mul2(x, both(1.44269504088896341f)));
    return pair(fast_exp2(f.x), fast_exp2(f.y));
}
// The normal distribution's Phi(z), with e = e^(-z^2 / 2).  The side away from
// 0 is e R(|z|), where R(x) = Phi(-x) e^(x^2 / 2) falls slowly, like 1 / x: a
// polynomial of degree 7 in t = 1 / (1 + 0.362 x) without a constant term,
// fitted to R on [0, 14] by the largest relative error (8e-7; 1.1e-6 with
// float32's roundings).  So the left tail, and GELU there, keeps that relative
// error and what e has of its argument's roundings, z^2 / 2 times 2e-7 or so:
// far below a 16-bit result's rounding until e itself ends (z = -13.2).
__device__ __forceinline__ f32x2 normal_cdf(f32x2 z, f32x2 e) {
    const float2 f = unpair(z);
    const f32x2 x = pair(fabsf(f.x), fabsf(f.y));
    const float2 d = unpair(fma2(x, both(0.362f), both(1.0f)));
    const f32x2 t = pair(fast_inverse(d.x), fast_inverse(d.y));
    f32x2 p = fma2(both(0.0479382612f), t, both(-0.180009604f));
    p = fma2(p, t, both(0.176617175f));
    p = fma2(p, t, both(0.0288315415f));
    p = fma2(p, t, both(0.139429674f));
    p = fma2(p, t, both(0.142689317f));
    p = fma2(p, t, both(0.144503906f));
    const float2 tail = unpair(mul2(mul2(p, t), e));
    return pair(f.x < 0.0f ? tail.x : 1.0f - tail.x, f.y < 0.0f ? tail.y : 1.0f - tail.y);
}
__device__ __forceinline__ f32x2 logistic(f32x2 z) {
    const float2 d = unpair(add2(exp_of(mul2(z, both(-1.0f))), both(1.0f)));
    return pair(fast_inverse(d.x), fast_inverse(d.y));
}
__device__ __forceinline__ f32x2 activate(f32x2 z, int act) {
    if (act == MDH_ACT_RELU) {
        const float2 f = unpair(z);
        return pair(f.x < 0.0f ? 0.0f : f.x, f.y < 0.0f ? 0.0f : f.y);  // NaN stays NaN
    }
    if (act == MDH_ACT_GELU) return mul2(z, normal_cdf(z, exp_of(mul2(mul2(z, z), both(-0.5f)))));
    if (act == MDH_ACT_SILU) {
        // z logistic(z); where e^-z leaves the float range the factor is 0 and so is the value.
        return mul2(z, logistic(z));
    }
    return z;
}
// Infinities become numbers so large that every slope has its limit there (0
// times infinity would be NaN); NaN stays.
__device__ __forceinline__ float bounded(float z) {
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(z), "f"(1e30f));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(z), "f"(-1e30f));
    return z;
}
// act'(z).  z comes as it was kept, in 16 bits: a float16 z is infinite past
// 65,504, where the value that the forward pass went on with was finite.
__device__ __forceinline__ f32x2 activation_slope(f32x2 z, int act) {
    if (act == MDH_ACT_GELU || act == MDH_ACT_SILU) {
        const float2 f = unpair(z);
        z = pair(bounded(f.x), bounded(f.y));
    }
    if (act == MDH_ACT_RELU) {
        const float2 f = unpair(z);
        return pair(f.x > 0.0f ? 1.0f : 0.0f, f.y > 0.0f ? 1.0f : 0.0f);
    }
    if (act == MDH_ACT_GELU) {
        const f32x2 e = exp_of(mul2(mul2(z, z), both(-0.5f)));
        return fma2(mul2(z, both(0.39894228040143268f)), e, normal_cdf(z, e));
    }
    if (act == MDH_ACT_SILU) {
        const f32x2 g = logistic(z);  // g (1 + z (1 - g))
        return fma2(mul2(g, z), add2(both(1.0f), mul2(g, both(-1.0f))), g);
    }
    return both(1.0f);
}
__device__ __forceinline__ float activate(float z, int act) { return unpair(activate(both(z), act)).x; }

}  // namespace op
}  // namespace mdh
