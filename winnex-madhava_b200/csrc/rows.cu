// A cache of 8-bit rows: quantised as they are written, read back by id.
//
// int8: a group of elements with largest magnitude a is stored as code =
// round(x (127 / a)) with the scale a / 127; uint8: code = round((x - lo)
// (1 / step)) limited to [0, 255].  Quotients, products and differences are
// each rounded to float32 (no fused multiply-add), so a row's codes are the
// same wherever they are computed.  Both directions are bound by memory.
#include "op_rows.cuh"

namespace mdh {
namespace {

using namespace op;

constexpr int kThreads = 256;

// One warp writes one row, group by group.
template <class T, class I>
__global__ void __launch_bounds__(kThreads)
    k_rows_write(RowsView c, const I* __restrict__ ids, const T* __restrict__ rows, int64_t row_stride, int64_t n) {
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (i >= n) return;
    const int64_t slot = (int64_t)ids[i];
    if (slot < 0 || slot >= c.slots) return;
    const T* x = rows + i * row_stride;
    uint8_t* out = c.codes + slot * c.stride;
    if (c.affine) {
        for (int e = lane; e < c.width; e += 32) out[e] = affine_code(to_f32(x[e]), c.lo, c.inv_step);
        return;
    }
    for (int g = 0; g < c.n_groups; g++) {
        const int e0 = g * c.group, e1 = min(e0 + c.group, c.width);
        float a = 0.0f;
        for (int e = e0 + lane; e < e1; e += 32) a = max_nan(a, fabsf(to_f32(x[e])));
#pragma unroll
        for (int o = 16; o; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        float scale, inv;
        group_scale(a, scale, inv);
        for (int e = e0 + lane; e < e1; e += 32) out[e] = (uint8_t)group_code(to_f32(x[e]), inv);
        if (lane == 0) c.scales[slot * c.n_groups + g] = scale;
    }
}

// A thread reads V consecutive elements of one row.
template <class T, class I, int V>
__global__ void __launch_bounds__(kThreads)
    k_rows_read(RowsView c, const I* __restrict__ ids, int64_t n, int chunks, T* __restrict__ out, int64_t out_stride) {
    const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t i = at / chunks;
    if (i >= n) return;
    const int e = (int)(at - i * chunks) * V;
    const int64_t slot = (int64_t)ids[i];
    Pack<T, V> p;
    if (slot < 0 || slot >= c.slots) {
#pragma unroll
        for (int j = 0; j < V; j++) p.v[j] = from_f32<T>(0.0f);
    } else {
        const uint8_t* src = c.codes + slot * c.stride + e;
        uint8_t code[V];
        if constexpr (V == 8) {
            *reinterpret_cast<uint2*>(code) = __ldg(reinterpret_cast<const uint2*>(src));
        } else if constexpr (V == 4) {
            *reinterpret_cast<uint32_t*>(code) = __ldg(reinterpret_cast<const uint32_t*>(src));
        } else {
            code[0] = src[0];
        }
        if (c.affine) {
#pragma unroll
            for (int j = 0; j < V; j++) p.v[j] = from_f32<T>(affine_value(code[j], c.lo, c.step));
        } else {
            // Groups are multiples of 16 elements: the V share one scale.
            const float scale = c.scales[slot * c.n_groups + e / c.group];
#pragma unroll
            for (int j = 0; j < V; j++) p.v[j] = from_f32<T>((float)(int8_t)code[j] * scale);
        }
    }
    store_pack<T, V>(out + i * out_stride + e, p);
}

template <class F>
void by_id(int32_t bits, F&& fn) {
    if (bits == 32) fn(int32_t{});
    else fn(int64_t{});
}

}  // namespace

namespace op {

RowsView rows_view(const mdh_rows* c) {
    MDH_REQUIRE(c, MDH_ERR_INVALID_ARG, "row cache: null cache");
    MDH_REQUIRE(c->slots >= 0 && c->slots <= INT32_MAX && c->width >= 1, MDH_ERR_INVALID_ARG,
                "row cache: slots must be in [0, 2^31) and width >= 1");
    MDH_REQUIRE(c->width <= 65536, MDH_ERR_UNSUPPORTED, "row cache: width is limited to 65536");
    MDH_REQUIRE(c->stride >= c->width, MDH_ERR_INVALID_ARG, "row cache: stride below the width");
    MDH_REQUIRE(c->code == 0 || c->code == 1, MDH_ERR_INVALID_ARG, "row cache: code must be 0 (int8) or 1 (uint8)");
    MDH_REQUIRE(c->slots == 0 || c->codes, MDH_ERR_INVALID_ARG, "row cache: null codes");
    RowsView v{};
    v.codes = static_cast<uint8_t*>(c->codes);
    v.slots = c->slots;
    v.stride = c->stride;
    v.width = c->width;
    v.affine = c->code == 1;
    if (v.affine) {
        v.lo = (float)c->lo;
        v.step = (float)c->step;
        v.inv_step = (float)(1.0 / c->step);
        MDH_REQUIRE(std::isfinite(v.lo) && v.step > 0.0f && std::isfinite(v.step) && v.inv_step > 0.0f &&
                        std::isfinite(v.inv_step),
                    MDH_ERR_INVALID_ARG, "row cache: lo must be finite and step positive, as float32 and its inverse");
        v.group = c->width;
        v.n_groups = 1;
    } else {
        MDH_REQUIRE(c->group >= 0 && c->group % 16 == 0, MDH_ERR_INVALID_ARG,
                    "row cache: group must be 0 (the whole row) or a multiple of 16");
        MDH_REQUIRE(c->slots == 0 || c->scales, MDH_ERR_INVALID_ARG, "row cache: null scales");
        v.scales = c->scales;
        v.group = c->group ? c->group : (int)round_up(c->width, 16);
        v.n_groups = (int)ceil_div(c->width, v.group);
    }
    return v;
}

}  // namespace op
}  // namespace mdh

using namespace mdh;

extern "C" {

mdh_status mdh_rows_write(const mdh_rows* cache, const void* ids, int32_t id_bits, const void* rows,
                          int64_t row_stride, int32_t dtype, int64_t n, void* stream) {
    return guarded([&] {
        const RowsView c = rows_view(cache);
        MDH_REQUIRE(id_bits == 32 || id_bits == 64, MDH_ERR_INVALID_ARG, "row cache: ids must be int32 or int64");
        MDH_REQUIRE(dtype_ok(dtype), MDH_ERR_INVALID_ARG, "row cache: dtype must be float32, bfloat16 or float16");
        MDH_REQUIRE(n >= 0, MDH_ERR_INVALID_ARG, "row cache: n must be >= 0");
        MDH_REQUIRE(n <= 1 || row_stride >= c.width, MDH_ERR_INVALID_ARG, "row cache: row stride below the width");
        current_device();
        if (n == 0 || c.slots == 0) return;
        MDH_REQUIRE(ids && rows, MDH_ERR_INVALID_ARG, "row cache: null ids or rows");
        const int64_t blocks = ceil_div(n, kThreads / 32);
        MDH_REQUIRE(blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "row cache: too many rows in one call");
        by_dtype(dtype, [&](auto zero) {
            using T = decltype(zero);
            by_id(id_bits, [&](auto id) {
                using I = decltype(id);
                k_rows_write<T, I><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(
                    c, (const I*)ids, (const T*)rows, row_stride, n);
            });
        });
        check_launch();
    });
}

mdh_status mdh_rows_read(const mdh_rows* cache, const void* ids, int32_t id_bits, int64_t n, void* out,
                         int64_t out_stride, int32_t dtype, void* stream) {
    return guarded([&] {
        const RowsView c = rows_view(cache);
        MDH_REQUIRE(id_bits == 32 || id_bits == 64, MDH_ERR_INVALID_ARG, "row cache: ids must be int32 or int64");
        MDH_REQUIRE(dtype_ok(dtype), MDH_ERR_INVALID_ARG, "row cache: dtype must be float32, bfloat16 or float16");
        MDH_REQUIRE(n >= 0, MDH_ERR_INVALID_ARG, "row cache: n must be >= 0");
        MDH_REQUIRE(n <= 1 || out_stride >= c.width, MDH_ERR_INVALID_ARG, "row cache: row stride below the width");
        current_device();
        if (n == 0) return;
        MDH_REQUIRE(ids && out, MDH_ERR_INVALID_ARG, "row cache: null ids or output");
        by_dtype(dtype, [&](auto zero) {
            using T = decltype(zero);
            constexpr int V = 16 / sizeof(T);
            const bool vec = c.width % V == 0 && c.stride % V == 0 &&
                             reinterpret_cast<uintptr_t>(c.codes) % V == 0 && rows_aligned(out, out_stride, sizeof(T));
            const int chunks = vec ? c.width / V : c.width;
            const int64_t blocks = ceil_div(n * chunks, kThreads);
            MDH_REQUIRE(blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "row cache: too many rows in one call");
            by_id(id_bits, [&](auto id) {
                using I = decltype(id);
                if (vec)
                    k_rows_read<T, I, V><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(
                        c, (const I*)ids, n, chunks, (T*)out, out_stride);
                else
                    k_rows_read<T, I, 1><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(
                        c, (const I*)ids, n, chunks, (T*)out, out_stride);
            });
        });
        check_launch();
    });
}

}  // extern "C"
