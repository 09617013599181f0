// A cache of 8-bit rows: quantised as they are written, read back by id.
//
// int8: a group of elements with largest magnitude a is stored as code =
// round(x (127 (1 / a))) with the scale a (1 / 127); uint8: code = round((x -
// lo) (1 / step)) limited to [0, 255].  Inverses, products and differences
// are each rounded to float32 (no fused multiply-add), so a row's codes are
// the same wherever they are computed.  Both directions are bound by memory:
// 1,000,003 float32 rows of 128 are written as u8 to scattered places in 124
// us and read back in 131 us on B200 (5.2 and 4.9 TB/s).
#include "op_rows.cuh"

namespace mdh {
namespace {

using namespace op;

constexpr int kThreads = 256;

// A block is x threads along a row (a power of two) by y rows; no index of
// an element needs a division.
dim3 row_block(int width) {
    int x = 1;
    while (x * kChunk < width && x < kThreads) x *= 2;
    return dim3(x, kThreads / x);
}

__device__ __forceinline__ void store_codes(uint8_t* p, int left, bool vec, const uint32_t (&c)[kChunk]) {
    if (vec && left >= kChunk) {
        uint2 w;
        w.x = (c[0] & 255) | (c[1] & 255) << 8 | (c[2] & 255) << 16 | c[3] << 24;
        w.y = (c[4] & 255) | (c[5] & 255) << 8 | (c[6] & 255) << 16 | c[7] << 24;
        *reinterpret_cast<uint2*>(p) = w;
    } else {
#pragma unroll
        for (int j = 0; j < kChunk; j++)
            if (j < left) p[j] = (uint8_t)c[j];
    }
}
__device__ __forceinline__ float chunk_max(const float (&v)[kChunk], float a) {
#pragma unroll
    for (int j = 0; j < kChunk; j++) a = max_nan(a, fabsf(v[j]));
    return a;
}
__device__ __forceinline__ void encode_group(const float (&v)[kChunk], float inv, uint32_t (&c)[kChunk]) {
#pragma unroll
    for (int j = 0; j < kChunk; j++) c[j] = (uint32_t)group_code(v[j], inv);
}

// uint8, and int8 in groups of `lanes` = 1, 2, 4 .. 32 neighbouring chunks
// (lanes divides the row's threads or the row is one group): the group's
// magnitude is a few shuffles.
template <class T, class I>
__global__ void __launch_bounds__(kThreads)
    k_rows_write(RowsView c, const I* __restrict__ ids, const T* __restrict__ rows, int64_t row_stride, int64_t n,
                 int lanes, bool vec_in, bool vec_out) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    // Every thread of a warp goes through the shuffles; rows that are not written store nothing.
    const int64_t slot = i < n ? (int64_t)ids[i] : -1;
    const bool write = slot >= 0 && slot < c.slots;
    const T* x = rows + (write ? i : 0) * row_stride;
    uint8_t* out = c.codes + (write ? slot : 0) * c.stride;
    for (int e0 = 0; e0 < c.width; e0 += blockDim.x * kChunk) {
        const int e = e0 + threadIdx.x * kChunk, left = write ? c.width - e : 0;
        float v[kChunk];
        load_chunk(x + (left > 0 ? e : 0), left, vec_in, v);
        uint32_t code[kChunk];
        if (c.affine) {
#pragma unroll
            for (int j = 0; j < kChunk; j++) code[j] = affine_code(v[j], c.lo, c.inv_step);
        } else {
            float a = chunk_max(v, 0.0f), scale, inv;
            for (int o = lanes / 2; o; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
            group_scale(a, scale, inv);
            encode_group(v, inv, code);
            if (left > 0 && threadIdx.x % lanes == 0) c.scales[slot * c.n_groups + e / c.group] = scale;
        }
        if (left > 0) store_codes(out + e, left, vec_out, code);
    }
}

// int8 in groups of any other size: a warp writes a row, group by group, and
// reads the group a second time (from the cache) for its codes.
template <class T, class I>
__global__ void __launch_bounds__(kThreads)
    k_rows_write_any(RowsView c, const I* __restrict__ ids, const T* __restrict__ rows, int64_t row_stride, int64_t n,
                     bool vec_in, bool vec_out) {
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (i >= n) return;
    const int64_t slot = (int64_t)ids[i];
    if (slot < 0 || slot >= c.slots) return;
    const T* x = rows + i * row_stride;
    uint8_t* out = c.codes + slot * c.stride;
    for (int g = 0; g < c.n_groups; g++) {
        const int e0 = g * c.group, e1 = min(e0 + c.group, c.width);
        float a = 0.0f, v[kChunk], scale, inv;
        for (int e = e0 + lane * kChunk; e < e1; e += 32 * kChunk) {
            load_chunk(x + e, e1 - e, vec_in, v);
            a = chunk_max(v, a);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        group_scale(a, scale, inv);
        for (int e = e0 + lane * kChunk; e < e1; e += 32 * kChunk) {
            load_chunk(x + e, e1 - e, vec_in, v);
            uint32_t code[kChunk];
            encode_group(v, inv, code);
            store_codes(out + e, e1 - e, vec_out, code);
        }
        if (lane == 0) c.scales[slot * c.n_groups + g] = scale;
    }
}

template <class T, class I>
__global__ void __launch_bounds__(kThreads)
    k_rows_read(RowsView c, const I* __restrict__ ids, int64_t n, bool vec_in, T* __restrict__ out, int64_t out_stride,
                bool vec_out) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (i >= n) return;
    const int64_t slot = (int64_t)ids[i];
    const bool some = slot >= 0 && slot < c.slots;
    for (int e = threadIdx.x * kChunk; e < c.width; e += blockDim.x * kChunk) {
        const int left = c.width - e;
        float v[kChunk] = {};
        if (some) {
            const uint8_t* src = c.codes + slot * c.stride + e;
            uint8_t code[kChunk] = {};
            if (vec_in && left >= kChunk) {
                *reinterpret_cast<uint2*>(code) = __ldg(reinterpret_cast<const uint2*>(src));
            } else {
#pragma unroll
                for (int j = 0; j < kChunk; j++)
                    if (j < left) code[j] = src[j];
            }
            if (c.affine) {
#pragma unroll
                for (int j = 0; j < kChunk; j++) v[j] = affine_value(code[j], c.lo, c.step);
            } else {
                // Groups are multiples of 16 elements: the chunk has one scale.
                const float scale = c.scales[slot * c.n_groups + e / c.group];
#pragma unroll
                for (int j = 0; j < kChunk; j++) v[j] = (float)(int8_t)code[j] * scale;
            }
        }
        store_chunk(out + i * out_stride + e, left, vec_out, v);
    }
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
        // Chunks of a group, where they are neighbouring lanes: a power of two up to 32.
        const int lanes = c.affine ? 1 : c.group % kChunk == 0 ? c.group / kChunk : 0;
        const dim3 block = row_block(c.width);
        const bool shuffled = lanes >= 1 && lanes <= 32 && (lanes & (lanes - 1)) == 0 && lanes <= (int)block.x;
        const int64_t blocks = ceil_div(n, shuffled ? block.y : kThreads / 32);
        MDH_REQUIRE(blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "row cache: too many rows in one call");
        const bool vec_in = rows_aligned(rows, row_stride, dtype_size(dtype)), vec_out = rows_on_8(c);
        by_dtype(dtype, [&](auto zero) {
            using T = decltype(zero);
            by_id(id_bits, [&](auto id) {
                using I = decltype(id);
                if (shuffled)
                    k_rows_write<T, I><<<(unsigned)blocks, block, 0, (cudaStream_t)stream>>>(
                        c, (const I*)ids, (const T*)rows, row_stride, n, lanes, vec_in, vec_out);
                else
                    k_rows_write_any<T, I><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(
                        c, (const I*)ids, (const T*)rows, row_stride, n, vec_in, vec_out);
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
        const dim3 block = row_block(c.width);
        const int64_t blocks = ceil_div(n, block.y);
        MDH_REQUIRE(blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "row cache: too many rows in one call");
        const bool vec_in = rows_on_8(c), vec_out = rows_aligned(out, out_stride, dtype_size(dtype));
        by_dtype(dtype, [&](auto zero) {
            using T = decltype(zero);
            by_id(id_bits, [&](auto id) {
                using I = decltype(id);
                k_rows_read<T, I><<<(unsigned)blocks, block, 0, (cudaStream_t)stream>>>(c, (const I*)ids, n, vec_in, (T*)out,
                                                                                     out_stride, vec_out);
            });
        });
        check_launch();
    });
}

}  // extern "C"
