// Layer norm of rows, forward and backward.
//
// Forward: mean = sum x / W, var = sum (x - mean)^2 / W (the deviations are
// formed from registers, so nothing cancels), y = (x - mean) rstd w + b.
// Backward, with xh = (x - mean) rstd and g = dy w:
//   dx = rstd (g - mean_c(g) - xh mean_c(g xh)),  dw = sum_r dy xh,
//   db = sum_r dy.
// Both are bound by memory: about ten operations an element.
//
// A row belongs to one warp up to 1024 elements (its sums are shuffles), to a
// block beyond; a thread holds 8, 16 or 32 elements of the row in registers,
// in 16-byte vectors where base, stride and width allow, else one by one.
#include "op_common.cuh"

namespace mdh {
namespace {

using namespace op;

constexpr int kWarpsPerBlock = 8;     // rows at a time of a block, warp form
constexpr int kBlockElems = 16;       // elements of a thread, block form
constexpr int kMaxWidth = 16384;

// Sum of `v` over the threads of a row: a warp, or (WIDE) the whole block.
template <bool WIDE>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = warp_sum(v);
    if constexpr (WIDE) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = blockDim.x >> 5;
        __syncthreads();  // the previous sum has been read
        if (lane == 0) red[warp] = v;
        __syncthreads();
        v = lane < n ? red[lane] : 0.0f;
        v = warp_sum(v);
    }
    return v;
}

// Weights are float32 or of the rows' type.
template <class T, int V>
__device__ __forceinline__ void load_weights(const void* w, bool w_f32, int c, float (&out)[V]) {
    if (w_f32) {
        const float* p = static_cast<const float*>(w) + c;
        if constexpr (V >= 4) {
#pragma unroll
            for (int i = 0; i < V / 4; i++) {
                const Pack<float, 4> r = load_pack<float, 4>(p + 4 * i);
#pragma unroll
                for (int j = 0; j < 4; j++) out[4 * i + j] = r.v[j];
            }
        } else {
            out[0] = p[0];
        }
    } else {
        const Pack<T, V> r = load_pack<T, V>(static_cast<const T*>(w) + c);
#pragma unroll
        for (int j = 0; j < V; j++) out[j] = to_f32(r.v[j]);
    }
}

template <class T, int V, int ELEMS, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 1024 : 32 * kWarpsPerBlock)
    k_norm_forward(const T* __restrict__ x, int64_t x_stride, const void* __restrict__ w, const void* __restrict__ b,
                   bool w_f32, int64_t rows, int width, float eps, T* __restrict__ y, int64_t y_stride,
                   float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int NV = ELEMS / V;
    __shared__ float red[32];
    const int64_t row = WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kWarpsPerBlock + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int t = WIDE ? threadIdx.x : threadIdx.x & 31, nt = WIDE ? blockDim.x : 32;
    const T* xr = x + row * x_stride;
    float v[NV][V];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * nt + t) * V;
        if (c < width) {
            const Pack<T, V> p = load_pack<T, V>(xr + c);
#pragma unroll
            for (int j = 0; j < V; j++) sum += v[i][j] = to_f32(p.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) v[i][j] = 0.0f;
        }
    }
    const float mean = row_sum<WIDE>(sum, red) / (float)width;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        if ((i * nt + t) * V < width) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = v[i][j] - mean;
                sq += d * d;
            }
        }
    }
    const float rstd = 1.0f / sqrtf(row_sum<WIDE>(sq, red) / (float)width + eps);
    if (t == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
    T* yr = y + row * y_stride;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * nt + t) * V;
        if (c >= width) continue;
        float ww[V], bb[V];
#pragma unroll
        for (int j = 0; j < V; j++) ww[j] = 1.0f, bb[j] = 0.0f;
        if (w) load_weights<T, V>(w, w_f32, c, ww);
        if (b) load_weights<T, V>(b, w_f32, c, bb);
        Pack<T, V> p;
#pragma unroll
        for (int j = 0; j < V; j++) p.v[j] = from_f32<T>((v[i][j] - mean) * rstd * ww[j] + bb[j]);
        store_pack<T, V>(yr + c, p);
    }
}

// Blocks take rows in turn; each thread sums dw and db of its columns over
// its rows, the warps of a block join theirs in shared memory, and the block
// writes one partial row of part[block][2][width].
template <class T, int V, int ELEMS, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 1024 : 32 * kWarpsPerBlock)
    k_norm_backward(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride,
                    const void* __restrict__ w, bool w_f32, const float* __restrict__ mean_in,
                    const float* __restrict__ rstd_in, int64_t rows, int width, T* __restrict__ dx, int64_t dx_stride,
                    float* __restrict__ part) {
    constexpr int NV = ELEMS / V;
    __shared__ float red[32];
    extern __shared__ float joined[];  // warp form: [2][width]
    const int warp = threadIdx.x >> 5;
    const int t = WIDE ? threadIdx.x : threadIdx.x & 31, nt = WIDE ? blockDim.x : 32;
    float dw[NV][V], db[NV][V];
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < V; j++) dw[i][j] = db[i][j] = 0.0f;
    const int64_t step = WIDE ? gridDim.x : (int64_t)gridDim.x * kWarpsPerBlock;
    for (int64_t row = WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kWarpsPerBlock + warp; row < rows;
         row += step) {
        const float mean = mean_in[row], rstd = rstd_in[row];
        float xh[NV][V], g[NV][V];
        float sg = 0.0f, sgx = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * nt + t) * V;
#pragma unroll
            for (int j = 0; j < V; j++) xh[i][j] = g[i][j] = 0.0f;
            if (c >= width) continue;
            const Pack<T, V> px = load_pack<T, V>(x + row * x_stride + c);
            const Pack<T, V> pd = load_pack<T, V>(dy + row * dy_stride + c);
            float ww[V];
#pragma unroll
            for (int j = 0; j < V; j++) ww[j] = 1.0f;
            if (w) load_weights<T, V>(w, w_f32, c, ww);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = to_f32(pd.v[j]);
                xh[i][j] = (to_f32(px.v[j]) - mean) * rstd;
                g[i][j] = d * ww[j];
                dw[i][j] += d * xh[i][j];
                db[i][j] += d;
                sg += g[i][j];
                sgx += g[i][j] * xh[i][j];
            }
        }
        if (dx) {
            const float mg = row_sum<WIDE>(sg, red) / (float)width;
            const float mgx = row_sum<WIDE>(sgx, red) / (float)width;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = (i * nt + t) * V;
                if (c >= width) continue;
                Pack<T, V> p;
#pragma unroll
                for (int j = 0; j < V; j++) p.v[j] = from_f32<T>(rstd * (g[i][j] - mg - xh[i][j] * mgx));
                store_pack<T, V>(dx + row * dx_stride + c, p);
            }
        }
    }
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * 2 * width;
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * nt + t) * V;
            if (c >= width) continue;
#pragma unroll
            for (int j = 0; j < V; j++) out[c + j] = dw[i][j], out[width + c + j] = db[i][j];
        }
    } else {
        // The warps add theirs one after another: a fixed order.
        for (int k = 0; k < kWarpsPerBlock; k++) {
            if (warp == k) {
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const int c = (i * nt + t) * V;
                    if (c >= width) continue;
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        joined[c + j] = (k ? joined[c + j] : 0.0f) + dw[i][j];
                        joined[width + c + j] = (k ? joined[width + c + j] : 0.0f) + db[i][j];
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * width; c += blockDim.x) out[c] = joined[c];
    }
}

// Column sums of part[n][2][width]: 32 columns of a block, its 8 warps each
// take every eighth partial row, joined in order.
template <class W>
__global__ void __launch_bounds__(256) k_norm_join(const float* __restrict__ part, int n, int width,
                                                   W* __restrict__ dw, W* __restrict__ db) {
    __shared__ float s[8][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (c < 2 * width)
        for (int i = warp; i < n; i += 8) v += part[(int64_t)i * 2 * width + c];
    s[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && c < 2 * width) {
        for (int k = 1; k < 8; k++) v += s[k][lane];
        if (c < width) {
            if (dw) dw[c] = from_f32<W>(v);
        } else if (db) {
            db[c - width] = from_f32<W>(v);
        }
    }
}

int backward_blocks(int64_t rows, int width) {
    const int64_t units = width <= 1024 ? ceil_div(rows, kWarpsPerBlock) : rows;
    return (int)std::min<int64_t>(units, 148 * 2);
}

void check_norm(const void* x, int64_t x_stride, int32_t dtype, int32_t w_dtype, int64_t rows, int32_t width) {
    MDH_REQUIRE(dtype_ok(dtype), MDH_ERR_INVALID_ARG, "layer norm: dtype must be float32, bfloat16 or float16");
    MDH_REQUIRE(w_dtype == MDH_F32 || w_dtype == dtype, MDH_ERR_INVALID_ARG,
                "layer norm: weights must be float32 or of the rows' type");
    MDH_REQUIRE(rows >= 0 && width >= 1, MDH_ERR_INVALID_ARG, "layer norm: rows must be >= 0 and width >= 1");
    MDH_REQUIRE(width <= kMaxWidth, MDH_ERR_UNSUPPORTED, "layer norm: width is limited to 16384");
    MDH_REQUIRE(rows == 0 || x, MDH_ERR_INVALID_ARG, "layer norm: null rows");
    MDH_REQUIRE(rows <= 1 || x_stride >= width, MDH_ERR_INVALID_ARG, "layer norm: row stride below the width");
}

// fn(V, ELEMS, WIDE) as compile-time values.
template <class T, class F>
void by_shape(bool vec, int width, F&& fn) {
    constexpr int V = 16 / sizeof(T);
    auto elems = [&](auto v) {
        if (width <= 256) fn(v, std::integral_constant<int, 8>{}, std::false_type{});
        else if (width <= 512) fn(v, std::integral_constant<int, 16>{}, std::false_type{});
        else if (width <= 1024) fn(v, std::integral_constant<int, 32>{}, std::false_type{});
        else fn(v, std::integral_constant<int, kBlockElems>{}, std::true_type{});
    };
    if (vec) elems(std::integral_constant<int, V>{});
    else elems(std::integral_constant<int, 1>{});
}

}  // namespace
}  // namespace mdh

using namespace mdh;

extern "C" {

mdh_status mdh_layer_norm_forward(const void* x, int64_t x_stride, int32_t dtype, const void* w, const void* b,
                                  int32_t w_dtype, int64_t rows, int32_t width, float eps, void* y, int64_t y_stride,
                                  float* mean, float* rstd, void* stream) {
    return guarded([&] {
        check_norm(x, x_stride, dtype, w_dtype, rows, width);
        MDH_REQUIRE(eps >= 0.0f, MDH_ERR_INVALID_ARG, "layer norm: eps must be >= 0");
        MDH_REQUIRE(rows <= 1 || y_stride >= width, MDH_ERR_INVALID_ARG, "layer norm: row stride below the width");
        current_device();
        if (rows == 0) return;
        MDH_REQUIRE(y, MDH_ERR_INVALID_ARG, "layer norm: null output");
        by_dtype(dtype, [&](auto zero) {
            using T = decltype(zero);
            const bool vec = width % (16 / sizeof(T)) == 0 && rows_aligned(x, x_stride, sizeof(T)) &&
                             rows_aligned(y, y_stride, sizeof(T)) && aligned16(w) && aligned16(b);
            by_shape<T>(vec, width, [&](auto v, auto elems, auto wide) {
                const int threads = wide ? (int)round_up(ceil_div(width, elems), 32) : 32 * kWarpsPerBlock;
                const int64_t blocks = wide ? rows : ceil_div(rows, kWarpsPerBlock);
                MDH_REQUIRE(blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "layer norm: too many rows");
                k_norm_forward<T, v, elems, wide><<<(unsigned)blocks, threads, 0, (cudaStream_t)stream>>>(
                    (const T*)x, x_stride, w, b, w_dtype == MDH_F32, rows, width, eps, (T*)y, y_stride, mean, rstd);
            });
        });
        check_launch();
    });
}

int64_t mdh_layer_norm_backward_workspace(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    return (int64_t)backward_blocks(rows, width) * 2 * width * 4;
}

mdh_status mdh_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, int32_t dtype,
                                   const void* w, int32_t w_dtype, const float* mean, const float* rstd, int64_t rows,
                                   int32_t width, void* dx, int64_t dx_stride, void* dw, void* db, void* ws,
                                   int64_t ws_bytes, void* stream) {
    return guarded([&] {
        check_norm(x, x_stride, dtype, w_dtype, rows, width);
        MDH_REQUIRE(rows <= 1 || dy_stride >= width, MDH_ERR_INVALID_ARG, "layer norm: row stride below the width");
        MDH_REQUIRE(!dx || rows <= 1 || dx_stride >= width, MDH_ERR_INVALID_ARG,
                    "layer norm: row stride below the width");
        MDH_REQUIRE(rows == 0 || (dy && mean && rstd), MDH_ERR_INVALID_ARG, "layer norm: null dy, mean or rstd");
        current_device();
        const cudaStream_t st = (cudaStream_t)stream;
        const size_t wsize = dtype_size(w_dtype);
        if (rows == 0) {
            if (dw) MDH_CUDA(cudaMemsetAsync(dw, 0, width * wsize, st));
            if (db) MDH_CUDA(cudaMemsetAsync(db, 0, width * wsize, st));
            return;
        }
        if (!dx && !dw && !db) return;
        const bool sums = dw || db;
        MDH_REQUIRE(!sums || (ws && aligned16(ws) && ws_bytes >= mdh_layer_norm_backward_workspace(rows, width)),
                    MDH_ERR_INVALID_ARG, "layer norm: workspace too small or not 16-byte aligned");
        const int blocks = backward_blocks(rows, width);
        by_dtype(dtype, [&](auto zero) {
            using T = decltype(zero);
            const bool vec = width % (16 / sizeof(T)) == 0 && rows_aligned(x, x_stride, sizeof(T)) &&
                             rows_aligned(dy, dy_stride, sizeof(T)) && aligned16(w) &&
                             (!dx || rows_aligned(dx, dx_stride, sizeof(T)));
            by_shape<T>(vec, width, [&](auto v, auto elems, auto wide) {
                const int threads = wide ? (int)round_up(ceil_div(width, elems), 32) : 32 * kWarpsPerBlock;
                k_norm_backward<T, v, elems, wide><<<blocks, threads, wide ? 0 : 2 * width * 4, st>>>(
                    (const T*)dy, dy_stride, (const T*)x, x_stride, w, w_dtype == MDH_F32, mean, rstd, rows, width,
                    (T*)dx, dx_stride, sums ? (float*)ws : nullptr);
            });
        });
        check_launch();
        if (!sums) return;
        by_dtype(w_dtype, [&](auto zero) {
            using W = decltype(zero);
            k_norm_join<W><<<(unsigned)ceil_div(2 * (int64_t)width, 32), 256, 0, st>>>((const float*)ws, blocks, width,
                                                                                    (W*)dw, (W*)db);
        });
        check_launch();
    });
}

}  // extern "C"
