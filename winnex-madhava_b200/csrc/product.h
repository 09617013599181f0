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

// Throws MDH_ERR_TIMEOUT when an earlier product gave up one of its waits.
void check_product_status();

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case MDH_ACT_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays NaN
        case MDH_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case MDH_ACT_SILU: return z / (1.0f + expf(-z));
        default: return z;
    }
}

}  // namespace op
}  // namespace mdh
