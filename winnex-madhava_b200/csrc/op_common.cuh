// Shared by the operators around the search (layer_norm.cu, linear.cu,
// rows.cu, attend.cu): element types, vector loads and stores, warp and block
// sums, and the host-side checks of a call.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "internal.h"

namespace mdh {
namespace op {

using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(f16 v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ f16 from_f32<f16>(float v) { return __float2half_rn(v); }

template <class T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
    T v[N];
};

// N consecutive elements; N * sizeof(T) is 16 (one vector access) or N is 1.
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    if constexpr (sizeof(T) * N == 16) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        return *reinterpret_cast<const Pack<T, N>*>(&u);
    } else {
        Pack<T, N> r;
#pragma unroll
        for (int i = 0; i < N; i++) r.v[i] = p[i];
        return r;
    }
}
template <class T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& r) {
    if constexpr (sizeof(T) * N == 16)
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
    else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = r.v[i];
    }
}

constexpr int kChunk = 8;  // elements of a thread
// 8 elements from p, zeros past `left`; vec: one or two 16-byte loads.
template <class T>
__device__ __forceinline__ void load_chunk(const T* p, int left, bool vec, float (&v)[kChunk]) {
    if (vec && left >= kChunk) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < kChunk / N; i++) {
            const Pack<T, N> x = load_pack<T, N>(p + i * N);
#pragma unroll
            for (int j = 0; j < N; j++) v[i * N + j] = to_f32(x.v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kChunk; j++) v[j] = j < left ? to_f32(p[j]) : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store_chunk(T* p, int left, bool vec, const float (&v)[kChunk]) {
    if (vec && left >= kChunk) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < kChunk / N; i++) {
            Pack<T, N> x;
#pragma unroll
            for (int j = 0; j < N; j++) x.v[j] = from_f32<T>(v[i * N + j]);
            store_pack<T, N>(p + i * N, x);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kChunk; j++)
            if (j < left) p[j] = from_f32<T>(v[j]);
    }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Two floats in one register pair: one instruction for two operations.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Starts a copy of BYTES (4, 8 or 16) to shared memory, zeros where `some` is false.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool some = true) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
                 "n"(BYTES), "r"(some ? BYTES : 0)
                 : "memory");
}
// The first `bytes` of BYTES, the rest zeros.
template <int BYTES>
__device__ __forceinline__ void copy_async_part(void* dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
                 "n"(BYTES), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits for this thread's copies, all but those of the last PENDING commits.
template <int PENDING>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// ------------------------------------------------------------ host side
inline size_t dtype_size(int32_t t) { return t == MDH_F32 ? 4 : 2; }
inline bool dtype_ok(int32_t t) { return t == MDH_F32 || t == MDH_BF16 || t == MDH_F16; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Rows of `stride` elements of `size` bytes from p can be read 16 bytes at a time.
inline bool rows_aligned(const void* p, int64_t stride, size_t size) {
    return aligned16(p) && (stride * (int64_t)size) % 16 == 0;
}
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The current device, checked once per device to be an sm_100 GPU.
int current_device();

// fn() under the C ABI's error convention (status code and message).
template <class F>
mdh_status guarded(F&& fn) {
    return run_guarded([](void* p) { (*static_cast<F*>(p))(); }, &fn);
}

inline void check_launch() { MDH_CUDA(cudaPeekAtLastError()); }

// fn with a value of the element type that `t` names.
template <class F>
void by_dtype(int32_t t, F&& fn) {
    switch (t) {
        case MDH_F32: fn(float{}); break;
        case MDH_BF16: fn(bf16{}); break;
        default: fn(f16{}); break;
    }
}

}  // namespace op
}  // namespace mdh
