// Linear layer with bias, activation and residual in the product's epilogue,
// and its gradients.
//
//   z = x w^T + b,  y = act(z) + residual
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = sum_rows dz
#include <algorithm>

#include "product.h"

namespace mdh {
namespace {

using namespace op;

__device__ __forceinline__ float activation_slope(float z, int act) {
    switch (act) {
        case MDH_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case MDH_ACT_GELU:
            return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
        case MDH_ACT_SILU: {
            const float e = 1.0f / (1.0f + expf(-z));
            return e * (1.0f + z * (1.0f - e));
        }
        default: return 1.0f;
    }
}

// dz [rows][n] = dy act'(z) (dz null: not stored), and part[block][n] = the
// column sums of a block's rows.
constexpr int kSlopeRows = 64;
template <class T>
__global__ void __launch_bounds__(256)
    k_slope(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ z, int act, int64_t rows, int64_t n,
            T* __restrict__ dz, int64_t dz_stride, float* __restrict__ part) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    const int64_t r0 = (int64_t)blockIdx.y * kSlopeRows, r1 = min(r0 + kSlopeRows, rows);
    float sum = 0.0f;
    for (int64_t r = r0; r < r1; r++) {
        float v = to_f32(dy[r * dy_stride + c]);
        if (act != MDH_ACT_NONE) v *= activation_slope(to_f32(z[r * n + c]), act);
        sum += v;
        if (dz) dz[r * dz_stride + c] = from_f32<T>(v);
    }
    if (part) part[blockIdx.y * n + c] = sum;
}

template <class T>
__global__ void __launch_bounds__(256) k_join(const float* __restrict__ part, int64_t blocks, int64_t n,
                                              T* __restrict__ out) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    float v = 0.0f;
    for (int64_t i = 0; i < blocks; i++) v += part[i * n + c];
    out[c] = from_f32<T>(v);
}

void check_linear(const void* x, int64_t x_stride, const void* w, int64_t w_stride, int32_t dtype, int32_t act,
                  int64_t rows, int32_t inner, int32_t outer) {
    MDH_REQUIRE(dtype == MDH_BF16 || dtype == MDH_F16, MDH_ERR_INVALID_ARG,
                "linear: dtype must be bfloat16 or float16");
    MDH_REQUIRE(act >= MDH_ACT_NONE && act <= MDH_ACT_SILU, MDH_ERR_INVALID_ARG, "linear: unknown activation");
    MDH_REQUIRE(rows >= 0 && inner >= 1 && outer >= 1, MDH_ERR_INVALID_ARG,
                "linear: rows must be >= 0, inner and outer >= 1");
    MDH_REQUIRE(rows <= INT32_MAX / 2, MDH_ERR_UNSUPPORTED, "linear: rows are limited to 2^30");
    MDH_REQUIRE(w && (rows == 0 || x), MDH_ERR_INVALID_ARG, "linear: null x or w");
    MDH_REQUIRE((rows <= 1 || x_stride >= inner) && (outer == 1 || w_stride >= inner), MDH_ERR_INVALID_ARG,
                "linear: row stride below the inner size");
}

bool enough(const void* ws, int64_t have, int64_t need) { return need == 0 || (ws && aligned16(ws) && have >= need); }

// The backward pass's scratch: dz (rows of a 16-byte stride) where there is
// an activation, the partial column sums, and the products' own scratch,
// which the second product takes over from the first.
struct BackwardLayout {
    int64_t dz_stride, part, product, bytes;
};
BackwardLayout backward_layout(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* w,
                               int64_t w_stride, int32_t activation, int64_t rows, int32_t inner, int32_t outer) {
    BackwardLayout l;
    l.dz_stride = round_up(outer, 8);
    const bool has_dz = activation != MDH_ACT_NONE;
    l.part = has_dz ? round_up(rows * l.dz_stride * 2, 128) : 0;
    l.product = l.part + round_up(ceil_div(rows, kSlopeRows) * outer * 4, 128);
    // Any 16-byte aligned address stands for dz: only its alignment is looked at.
    const void* g = has_dz ? nullptr : dy;
    const int64_t gs = has_dz ? l.dz_stride : dy_stride;
    const int64_t a = product_workspace({g, gs, true}, {w, w_stride, false}, rows, inner, outer);
    const int64_t b = product_workspace({g, gs, false}, {x, x_stride, false}, outer, inner, rows);
    l.bytes = l.product + std::max(a, b);
    return l;
}

template <class F>
void by_half(int32_t t, F&& fn) {
    if (t == MDH_BF16) fn(bf16{});
    else fn(f16{});
}

}  // namespace
}  // namespace mdh

using namespace mdh;

extern "C" {

int64_t mdh_linear_forward_workspace(const void* x, int64_t x_stride, const void* w, int64_t w_stride, int64_t rows,
                                     int32_t inner, int32_t outer) {
    return product_workspace({x, x_stride, true}, {w, w_stride, true}, rows, outer, inner);
}

mdh_status mdh_linear_forward(const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* bias,
                              const void* residual, int64_t residual_stride, int32_t dtype, int32_t activation,
                              int64_t rows, int32_t inner, int32_t outer, void* y, int64_t y_stride, void* z_out,
                              void* ws, int64_t ws_bytes, void* stream) {
    return guarded([&] {
        check_linear(x, x_stride, w, w_stride, dtype, activation, rows, inner, outer);
        MDH_REQUIRE(rows <= 1 || (y_stride >= outer && (!residual || residual_stride >= outer)), MDH_ERR_INVALID_ARG,
                    "linear: row stride below the outer size");
        current_device();
        if (rows == 0) return;
        MDH_REQUIRE(y, MDH_ERR_INVALID_ARG, "linear: null output");
        check_product_status();
        MDH_REQUIRE(enough(ws, ws_bytes, mdh_linear_forward_workspace(x, x_stride, w, w_stride, rows, inner, outer)),
                    MDH_ERR_INVALID_ARG, "linear: workspace too small or not 16-byte aligned");
        ProductEpilogue ep;
        ep.bias = bias;
        ep.residual = residual;
        ep.residual_stride = residual_stride;
        ep.act = activation;
        ep.y = y;
        ep.y_stride = y_stride;
        ep.z = z_out;
        product({x, x_stride, true}, {w, w_stride, true}, rows, outer, inner, dtype, ep, ws, (cudaStream_t)stream);
    });
}

int64_t mdh_linear_backward_workspace(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                                      const void* w, int64_t w_stride, int32_t activation, int64_t rows, int32_t inner,
                                      int32_t outer) {
    if (rows <= 0 || outer <= 0 || inner <= 0) return 0;
    return backward_layout(dy, dy_stride, x, x_stride, w, w_stride, activation, rows, inner, outer).bytes;
}

mdh_status mdh_linear_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* w,
                               int64_t w_stride, const void* z, int32_t dtype, int32_t activation, int64_t rows,
                               int32_t inner, int32_t outer, void* dx, void* dw, void* db, void* ws, int64_t ws_bytes,
                               void* stream) {
    return guarded([&] {
        check_linear(x, x_stride, w, w_stride, dtype, activation, rows, inner, outer);
        MDH_REQUIRE(rows <= 1 || dy_stride >= outer, MDH_ERR_INVALID_ARG, "linear: row stride below the outer size");
        MDH_REQUIRE(rows == 0 || (dy && (activation == MDH_ACT_NONE || z)), MDH_ERR_INVALID_ARG,
                    "linear: null dy, or no z for the activation's slope");
        current_device();
        const cudaStream_t st = (cudaStream_t)stream;
        if (rows == 0) {
            if (dw) MDH_CUDA(cudaMemsetAsync(dw, 0, (size_t)inner * outer * 2, st));
            if (db) MDH_CUDA(cudaMemsetAsync(db, 0, (size_t)outer * 2, st));
            return;
        }
        check_product_status();
        const BackwardLayout lay = backward_layout(dy, dy_stride, x, x_stride, w, w_stride, activation, rows, inner, outer);
        MDH_REQUIRE(enough(ws, ws_bytes, lay.bytes), MDH_ERR_INVALID_ARG,
                    "linear: workspace too small or not 16-byte aligned");
        char* base = static_cast<char*>(ws);
        by_half(dtype, [&](auto zero) {
            using T = decltype(zero);
            T* dz = activation == MDH_ACT_NONE ? nullptr : reinterpret_cast<T*>(base);
            float* part = reinterpret_cast<float*>(base + lay.part);
            const int64_t blocks = ceil_div(rows, kSlopeRows);
            if (dz || db) {
                const dim3 grid((unsigned)ceil_div(outer, 256), (unsigned)blocks);
                k_slope<T><<<grid, 256, 0, st>>>((const T*)dy, dy_stride, (const T*)z, activation, rows, outer, dz,
                                                 lay.dz_stride, db ? part : nullptr);
                check_launch();
            }
            if (db) {
                k_join<T><<<(unsigned)ceil_div(outer, 256), 256, 0, st>>>(part, blocks, outer, (T*)db);
                check_launch();
            }
            const void* g = dz ? dz : dy;
            const int64_t gs = dz ? lay.dz_stride : dy_stride;
            ProductEpilogue ep;
            ep.y_stride = inner;
            if (dx) {
                ep.y = dx;
                product({g, gs, true}, {w, w_stride, false}, rows, inner, outer, dtype, ep, base + lay.product, st);
            }
            if (dw) {
                ep.y = dw;
                product({g, gs, false}, {x, x_stride, false}, outer, inner, rows, dtype, ep, base + lay.product, st);
            }
        });
    });
}

}  // extern "C"
