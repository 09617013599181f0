// Linear layer with bias, activation and residual in the product's epilogue,
// and its gradients.
//
//   z = x w^T + b,  y = act(z) + residual
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = sum_rows dz
//
// Two roundings to 16 bits stand between the passes.  dz is an operand of the
// tensor cores, which take no other type: with it a gradient's relative error
// is 2.35e-3 in bfloat16 and 2.9e-4 in float16, where rounding the result alone
// gives 1.65e-3 and 2.1e-4.  z is kept between the passes in the operands' type,
// as its layer's activations are: 2.41e-3 and 3.0e-4 with both, for half of the
// memory and of the passes over it (67 MB each at 16,384 x 2,048).
#include <algorithm>

#include "product.h"

namespace mdh {
namespace {

using namespace op;

// dz [rows][n] = dy act'(z) (dz null: not stored), and part[block][n] = the
// column sums of a block's rows.  A lane holds 8 columns, a warp every eighth
// of the block's rows; the next three are on their way into the thread's own
// shared memory.  Bound by memory, three passes over [rows][n]: 16,384 x 2,048
// with GELU 38 us on B200 (5.3 TB/s; 61 us without the copies ahead).
constexpr int kSlopeRows = 64, kSlopeStages = 4;
// 8 16-bit elements as they lie in memory, zeros past `left`.
template <class T>
struct Chunk {
    Pack<T, kChunk> raw;
    __device__ __forceinline__ void load(const T* p, int left, bool vec) {
        if (vec && left >= kChunk) {
            raw = load_pack<T, kChunk>(p);
        } else {
#pragma unroll
            for (int j = 0; j < kChunk; j++) raw.v[j] = j < left ? p[j] : from_f32<T>(0.0f);
        }
    }
    __device__ __forceinline__ f32x2 pair_at(int j) const { return pair(to_f32(raw.v[2 * j]), to_f32(raw.v[2 * j + 1])); }
};
template <class T>
__global__ void __launch_bounds__(256, 4)
    k_slope(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ z, int act, int64_t rows, int64_t n,
            T* __restrict__ dz, int64_t dz_stride, float* __restrict__ part, bool vec_dy, bool vec_z) {
    __shared__ Pack<T, kChunk> ring[kSlopeStages][2][256];
    __shared__ float sums[8][32 * kChunk];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t c = ((int64_t)blockIdx.y * 32 + lane) * kChunk;
    const int left = (int)min((int64_t)kChunk, n - c);
    const int64_t r0 = (int64_t)blockIdx.x * kSlopeRows, r1 = min(r0 + kSlopeRows, rows);
    f32x2 sum[kChunk / 2] = {};
    auto run = [&](auto known) {  // the activation as a compile-time value
        constexpr int ACT = decltype(known)::value;
        const bool whole = vec_dy && vec_z && left == kChunk;
        auto fetch = [&](int stage, int64_t r) {
            if (whole && r < r1) {
                copy_async<16>(&ring[stage][0][threadIdx.x], dy + r * dy_stride + c);
                if (ACT != MDH_ACT_NONE) copy_async<16>(&ring[stage][1][threadIdx.x], z + r * n + c);
            }
            copy_commit();
        };
        for (int k = 0; k < kSlopeStages - 1; k++) fetch(k, r0 + warp + 8 * k);
        int stage = 0;
        for (int64_t r = r0 + warp; r < r1; r += 8) {
            Chunk<T> dd, zz;
            copy_wait<kSlopeStages - 2>();
            if (whole) {
                dd.raw = ring[stage][0][threadIdx.x];
                if (ACT != MDH_ACT_NONE) zz.raw = ring[stage][1][threadIdx.x];
            } else {
                dd.load(dy + r * dy_stride + c, left, vec_dy);
                if (ACT != MDH_ACT_NONE) zz.load(z + r * n + c, left, vec_z);
            }
            fetch((stage + kSlopeStages - 1) % kSlopeStages, r + 8 * (kSlopeStages - 1));
            stage = (stage + 1) % kSlopeStages;
            float v[kChunk];
#pragma unroll
            for (int j = 0; j < kChunk / 2; j++) {
                f32x2 d = dd.pair_at(j);
                if (ACT != MDH_ACT_NONE) d = mul2(d, activation_slope(zz.pair_at(j), ACT));
                sum[j] = add2(sum[j], d);
                const float2 f = unpair(d);
                v[2 * j] = f.x, v[2 * j + 1] = f.y;
            }
            if (dz) store_chunk(dz + r * dz_stride + c, left, true, v);
        }
        copy_wait<0>();
    };
    if (left > 0) {
        if (act == MDH_ACT_RELU) run(std::integral_constant<int, MDH_ACT_RELU>{});
        else if (act == MDH_ACT_GELU) run(std::integral_constant<int, MDH_ACT_GELU>{});
        else if (act == MDH_ACT_SILU) run(std::integral_constant<int, MDH_ACT_SILU>{});
        else run(std::integral_constant<int, MDH_ACT_NONE>{});
    }
    if (!part) return;
#pragma unroll
    for (int j = 0; j < kChunk / 2; j++) *reinterpret_cast<float2*>(&sums[warp][lane * kChunk + 2 * j]) = unpair(sum[j]);
    __syncthreads();
    const int64_t at = (int64_t)blockIdx.y * 32 * kChunk + threadIdx.x;
    if (at < n) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) v += sums[k][threadIdx.x];
        part[blockIdx.x * n + at] = v;
    }
}

// Column sums of part[blocks][n]: 32 columns of a block, its 32 warps each
// take every 32nd partial row, joined in order.
template <class T>
__global__ void __launch_bounds__(1024) k_join(const float* __restrict__ part, int64_t blocks, int64_t n,
                                               T* __restrict__ out) {
    __shared__ float s[32][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (c < n) {
#pragma unroll 4
        for (int64_t i = warp; i < blocks; i += 32) v += part[i * n + c];
    }
    s[warp][lane] = v;
    __syncthreads();
    if (warp != 0 || c >= n) return;
    for (int k = 1; k < 32; k++) v += s[k][lane];
    out[c] = from_f32<T>(v);
}

// The forward pass of a few rows (a query, a token): bound by reading w once
// and by latency.  A warp forms one output column for up to ROWS rows; x and w
// are read 8 elements a lane.
template <class T, int ROWS>
__global__ void __launch_bounds__(128)
    k_linear_rows(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ w, int64_t w_stride,
                  const T* __restrict__ bias, const T* __restrict__ residual, int64_t residual_stride, int act, int rows,
                  int inner, int outer, T* __restrict__ y, int64_t y_stride, T* __restrict__ z, bool vec_x, bool vec_w) {
    const int lane = threadIdx.x & 31;
    const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int m0 = blockIdx.y * ROWS, mine = m0 + lane;
    if (n >= outer) return;
    const bool writes = lane < ROWS && mine < rows;
    const float b = bias ? to_f32(bias[n]) : 0.0f;
    const float res = residual && writes ? to_f32(residual[mine * residual_stride + n]) : 0.0f;
    float acc[ROWS] = {};
#pragma unroll 2
    for (int k = lane * kChunk; k < inner; k += 32 * kChunk) {
        float wv[kChunk];
        load_chunk(w + n * w_stride + k, inner - k, vec_w, wv);
#pragma unroll
        for (int m = 0; m < ROWS; m++) {
            if (m0 + m >= rows) break;
            float xv[kChunk];
            load_chunk(x + (m0 + m) * x_stride + k, inner - k, vec_x, xv);
#pragma unroll
            for (int j = 0; j < kChunk; j++) acc[m] = fmaf(xv[j], wv[j], acc[m]);
        }
    }
    float v = 0.0f;
#pragma unroll
    for (int m = 0; m < ROWS; m++) {
        const float s = warp_sum(acc[m]);
        if (lane == m) v = s;
    }
    if (!writes) return;
    v += b;
    if (z) z[(int64_t)mine * outer + n] = from_f32<T>(v);
    y[mine * y_stride + n] = from_f32<T>(activate(v, act) + res);
}
// Rows up to which the row form is taken: one row of 768 x 768 in 4.7 us
// against 10 us by a 128-row tile; each 4 rows read w again, from the cache.
constexpr int64_t kFewRows = 8;

void check_linear(const void* x, int64_t x_stride, const void* w, int64_t w_stride, int32_t dtype, int32_t act,
                  int64_t rows, int32_t inner, int32_t outer) {
    MDH_REQUIRE(dtype == MDH_BF16 || dtype == MDH_F16, MDH_ERR_INVALID_ARG,
                "linear: dtype must be bfloat16 or float16");
    MDH_REQUIRE(act >= MDH_ACT_NONE && act <= MDH_ACT_SILU, MDH_ERR_INVALID_ARG, "linear: unknown activation");
    MDH_REQUIRE(rows >= 0 && inner >= 1 && outer >= 1, MDH_ERR_INVALID_ARG,
                "linear: rows must be >= 0, inner and outer >= 1");
    // Row, column and k indices are 32 bits and run past the size by a tile.
    constexpr int32_t kMost = 1 << 30;
    MDH_REQUIRE(rows <= kMost && inner <= kMost && outer <= kMost, MDH_ERR_UNSUPPORTED,
                "linear: rows, inner and outer are limited to 2^30");
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
    return rows <= kFewRows ? 0 : product_workspace({x, x_stride, true}, {w, w_stride, true}, rows, outer, inner);
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
        if (rows <= kFewRows) {  // no waits
            by_half(dtype, [&](auto zero) {
                using T = decltype(zero);
                auto run = [&](auto group) {
                    const dim3 grid((unsigned)ceil_div(outer, 4), (unsigned)ceil_div(rows, group));
                    k_linear_rows<T, group><<<grid, 128, 0, (cudaStream_t)stream>>>(
                        (const T*)x, x_stride, (const T*)w, w_stride, (const T*)bias, (const T*)residual,
                        residual_stride, activation, (int)rows, inner, outer, (T*)y, y_stride, (T*)z_out,
                        rows_aligned(x, x_stride, 2), rows_aligned(w, w_stride, 2));
                };
                if (rows == 1) run(std::integral_constant<int, 1>{});
                else run(std::integral_constant<int, 4>{});
            });
            check_launch();
            return;
        }
        MDH_REQUIRE(enough(ws, ws_bytes, mdh_linear_forward_workspace(x, x_stride, w, w_stride, rows, inner, outer)),
                    MDH_ERR_INVALID_ARG, "linear: workspace too small or not 16-byte aligned");
        check_product_status();
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

mdh_status mdh_linear_status(void) {
    return guarded([&] { check_product_status(); });
}

mdh_status mdh_linear_set_expired(void) {
    return guarded([&] { set_product_expired(); });
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
        MDH_REQUIRE(ceil_div(outer, 32 * kChunk) <= 65535, MDH_ERR_UNSUPPORTED,
                    "linear: gradients are limited to an outer size of 65,535 x 256");
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
        const BackwardLayout lay = backward_layout(dy, dy_stride, x, x_stride, w, w_stride, activation, rows, inner, outer);
        MDH_REQUIRE(enough(ws, ws_bytes, lay.bytes), MDH_ERR_INVALID_ARG,
                    "linear: workspace too small or not 16-byte aligned");
        check_product_status();
        char* base = static_cast<char*>(ws);
        by_half(dtype, [&](auto zero) {
            using T = decltype(zero);
            T* dz = activation == MDH_ACT_NONE ? nullptr : reinterpret_cast<T*>(base);
            float* part = reinterpret_cast<float*>(base + lay.part);
            const int64_t blocks = ceil_div(rows, kSlopeRows);
            if (dz || db) {
                const dim3 grid((unsigned)blocks, (unsigned)ceil_div(outer, 32 * kChunk));
                k_slope<T><<<grid, 256, 0, st>>>((const T*)dy, dy_stride, (const T*)z, activation, rows, outer, dz,
                                                 lay.dz_stride, db ? part : nullptr, rows_aligned(dy, dy_stride, 2),
                                                 rows_aligned(z, outer, 2));
                check_launch();
            }
            if (db) {
                k_join<T><<<(unsigned)ceil_div(outer, 32), 1024, 0, st>>>(part, blocks, outer, (T*)db);
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
