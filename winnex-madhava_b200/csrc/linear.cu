// Linear layer with bias, activation and residual in the product's epilogue,
// and its gradients.
//
//   z = x w^T + b,  y = act(z) + residual
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = sum_rows dz
#include "op_common.cuh"

namespace mdh {
namespace {

using namespace op;

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case MDH_ACT_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays NaN
        case MDH_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case MDH_ACT_SILU: return z / (1.0f + expf(-z));
        default: return z;
    }
}
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

// An operand of a product: element (row, k) at p[row * row_stride + k * k_stride].
template <class T>
struct Operand {
    const T* p;
    int64_t row_stride, k_stride;
    __device__ __forceinline__ float at(int64_t row, int64_t k) const { return to_f32(p[row * row_stride + k * k_stride]); }
};

template <class T>
struct Epilogue {
    const T* bias;
    const T* residual;
    int64_t residual_stride;
    int act;
    T* y;
    int64_t y_stride;
    T* z;
};

constexpr int kTile = 64, kDepth = 16;

// C[m][n] = sum_k a(m, k) b(n, k): a 64 x 64 tile of a block, 4 x 4 outputs of a thread.
template <class T>
__global__ void __launch_bounds__(256) k_product(Operand<T> a, Operand<T> b, int64_t m, int64_t n, int64_t k,
                                                 Epilogue<T> ep) {
    __shared__ float sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
    const int64_t m0 = (int64_t)blockIdx.x * kTile, n0 = (int64_t)blockIdx.y * kTile;
    const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < k; k0 += kDepth) {
        for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
            const int r = i / kDepth, c = i % kDepth;
            sa[c][r] = m0 + r < m && k0 + c < k ? a.at(m0 + r, k0 + c) : 0.0f;
            sb[c][r] = n0 + r < n && k0 + c < k ? b.at(n0 + r, k0 + c) : 0.0f;
        }
        __syncthreads();
        for (int c = 0; c < kDepth; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] += sa[c][tm + 16 * i] * sb[c][tn + 16 * j];
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int64_t r = m0 + tm + 16 * i, c = n0 + tn + 16 * j;
            if (r >= m || c >= n) continue;
            float z = acc[i][j] + (ep.bias ? to_f32(ep.bias[c]) : 0.0f);
            if (ep.z) ep.z[r * n + c] = from_f32<T>(z);
            z = activate(z, ep.act);
            if (ep.residual) z += to_f32(ep.residual[r * ep.residual_stride + c]);
            ep.y[r * ep.y_stride + c] = from_f32<T>(z);
        }
}

// dz [rows][n] = dy act'(z) (dz null: not stored), and part[block][n] = the
// column sums of a block's rows.
constexpr int kSlopeRows = 64;
template <class T>
__global__ void __launch_bounds__(256)
    k_slope(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ z, int act, int64_t rows, int64_t n,
            T* __restrict__ dz, float* __restrict__ part) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    const int64_t r0 = (int64_t)blockIdx.y * kSlopeRows, r1 = min(r0 + kSlopeRows, rows);
    float sum = 0.0f;
    for (int64_t r = r0; r < r1; r++) {
        float v = to_f32(dy[r * dy_stride + c]);
        if (act != MDH_ACT_NONE) v *= activation_slope(to_f32(z[r * n + c]), act);
        sum += v;
        if (dz) dz[r * n + c] = from_f32<T>(v);
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

template <class T>
void product(Operand<T> a, Operand<T> b, int64_t m, int64_t n, int64_t k, const Epilogue<T>& ep, cudaStream_t st) {
    const dim3 grid((unsigned)ceil_div(m, kTile), (unsigned)ceil_div(n, kTile));
    k_product<T><<<grid, 256, 0, st>>>(a, b, m, n, k, ep);
    check_launch();
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

template <class F>
void by_half(int32_t t, F&& fn) {
    if (t == MDH_BF16) fn(bf16{});
    else fn(f16{});
}

}  // namespace
}  // namespace mdh

using namespace mdh;

extern "C" {

int64_t mdh_linear_forward_workspace(const void*, int64_t, const void*, int64_t, int64_t, int32_t, int32_t) { return 0; }

mdh_status mdh_linear_forward(const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* bias,
                              const void* residual, int64_t residual_stride, int32_t dtype, int32_t activation,
                              int64_t rows, int32_t inner, int32_t outer, void* y, int64_t y_stride, void* z_out,
                              void* ws, int64_t ws_bytes, void* stream) {
    (void)ws;
    (void)ws_bytes;
    return guarded([&] {
        check_linear(x, x_stride, w, w_stride, dtype, activation, rows, inner, outer);
        MDH_REQUIRE(rows <= 1 || (y_stride >= outer && (!residual || residual_stride >= outer)), MDH_ERR_INVALID_ARG,
                    "linear: row stride below the outer size");
        current_device();
        if (rows == 0) return;
        MDH_REQUIRE(y, MDH_ERR_INVALID_ARG, "linear: null output");
        by_half(dtype, [&](auto zero) {
            using T = decltype(zero);
            const Epilogue<T> ep{(const T*)bias, (const T*)residual, residual_stride, activation, (T*)y, y_stride,
                                 (T*)z_out};
            product<T>({(const T*)x, x_stride, 1}, {(const T*)w, w_stride, 1}, rows, outer, inner, ep,
                       (cudaStream_t)stream);
        });
    });
}

int64_t mdh_linear_backward_workspace(const void*, int64_t, const void*, int64_t, const void*, int64_t,
                                      int32_t activation, int64_t rows, int32_t, int32_t outer) {
    if (rows <= 0 || outer <= 0) return 0;
    return round_up(activation == MDH_ACT_NONE ? 0 : rows * outer * 2, 16) + ceil_div(rows, kSlopeRows) * outer * 4;
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
        const int64_t need = mdh_linear_backward_workspace(dy, dy_stride, x, x_stride, w, w_stride, activation, rows,
                                                           inner, outer);
        MDH_REQUIRE(ws && aligned16(ws) && ws_bytes >= need, MDH_ERR_INVALID_ARG,
                    "linear: workspace too small or not 16-byte aligned");
        by_half(dtype, [&](auto zero) {
            using T = decltype(zero);
            T* dz = activation == MDH_ACT_NONE ? nullptr : (T*)ws;
            float* part = (float*)((char*)ws + round_up(dz ? rows * outer * 2 : 0, 16));
            const int64_t blocks = ceil_div(rows, kSlopeRows);
            if (dz || db) {
                const dim3 grid((unsigned)ceil_div(outer, 256), (unsigned)blocks);
                k_slope<T><<<grid, 256, 0, st>>>((const T*)dy, dy_stride, (const T*)z, activation, rows, outer, dz,
                                                 db ? part : nullptr);
                check_launch();
            }
            if (db) {
                k_join<T><<<(unsigned)ceil_div(outer, 256), 256, 0, st>>>(part, blocks, outer, (T*)db);
                check_launch();
            }
            const T* g = dz ? dz : (const T*)dy;
            const int64_t gs = dz ? outer : dy_stride;
            if (dx)
                product<T>({g, gs, 1}, {(const T*)w, 1, w_stride}, rows, inner, outer,
                           {nullptr, nullptr, 0, MDH_ACT_NONE, (T*)dx, inner, nullptr}, st);
            if (dw)
                product<T>({g, 1, gs}, {(const T*)x, 1, x_stride}, outer, inner, rows,
                           {nullptr, nullptr, 0, MDH_ACT_NONE, (T*)dw, inner, nullptr}, st);
        });
    });
}

}  // extern "C"
