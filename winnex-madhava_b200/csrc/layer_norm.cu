// Layer norm of rows, forward and backward.
//
// Forward: mean = sum x / W, var = sum (x - mean)^2 / W (the deviations are
// formed from registers, so nothing cancels), y = (x - mean) rstd w + b.
// Backward, with xh = (x - mean) rstd and g = dy w:
//   dx = rstd (g - mean_c(g) - xh mean_c(g xh)),  dw = sum_r dy xh,
//   db = sum_r dy.
// Both are bound by memory: about ten operations an element.
//
// Blocks stay and take rows in turn, so the weights are read once a block.
// What bounds them is the latency of memory: each thread copies its share of
// the next rows, three where they fit, into its own places of a ring in shared
// memory.  Its vectors are of 16 bytes where base, stride and width allow;
// 16-bit rows of any other width go by 4 bytes: such a row may start in the
// middle of a word, and then its pairs begin one element earlier (`shift`).
// Rows an even distance apart start alike, so a warp has one shift.
// A row belongs to one warp up to 1024 elements (its sums are shuffles), to a
// group of warps beyond, 16 elements a thread; weights, and backward the
// running sums of a thread's columns, stay in registers.  65,536 x 768 bf16 on
// B200: forward 35.6 us (5.7 TB/s), backward 60.5 + 3.7 us (5.0 TB/s of dy, x
// and dx); without the ring 55 and 178 us.  x 1,024: 47 us (5.7 TB/s) and 116 +
// 4 us (3.5 TB/s; 32 elements a lane of x, dy and their sums do not fit its
// registers).
#include <algorithm>
#include <atomic>
#include <initializer_list>
#include <utility>

#include "op_common.cuh"

namespace mdh {
namespace {

using namespace op;

constexpr int kWarpsPerBlock = 8;     // rows at a time of a block, warp form
constexpr int kBlockElems = 16;       // elements of a thread, block form
constexpr int kMaxWidth = 16384;

// Sums over the warps of a row: one warp, or all `warps` of the block, which
// share red[warps].
__device__ __forceinline__ float2 row_sums(float2 v, float2* red, int warp, int warps) {
    v.x = warp_sum(v.x);
    v.y = warp_sum(v.y);
    if (warps > 1) {
        const int lane = threadIdx.x & 31;
        __syncthreads();  // the previous sums have been read
        if (lane == 0) red[warp] = v;
        __syncthreads();
        v = lane < warps ? red[lane] : make_float2(0.0f, 0.0f);
        v.x = warp_sum(v.x);
        v.y = warp_sum(v.y);
    }
    return v;
}

// Weight c, float32 or of the rows' type.
template <class T>
__device__ __forceinline__ float weight_at(const void* w, bool w_f32, int c) {
    return w_f32 ? static_cast<const float*>(w)[c] : to_f32(static_cast<const T*>(w)[c]);
}

// A thread's places for its shares of the next rows: elements (i * nt + t) * V
// - shift + 0 .. V - 1 of a row.  Those outside the row are 0.  A shifted row
// takes one place more than it has elements (vector_of sees to it).
// A ring has four stages, fewer where a block's rows are too large for them:
// three small blocks share an SM, larger ones have it for themselves.
constexpr int stages_of(int threads, int bytes) {
    const int most = (threads <= 256 ? 72 : 144) * 1024;
    return threads * bytes * 4 <= most ? 4 : threads * bytes * 2 <= most ? 2 : 1;
}
// Blocks of `smem` bytes that an SM holds.
constexpr int blocks_that_fit(int smem) { return std::max(1, 227 * 1024 / (smem + 1024)); }
template <class T, int V, int NV, int STAGES, int THREADS>
struct Ring {
    Pack<T, V>* at;  // of this thread: place i of stage s at [(s * NV + i) * THREADS]
    int t, nt, width, shift;
    __device__ __forceinline__ Ring(void* smem, int t, int nt, int width, int shift)
        : at(static_cast<Pack<T, V>*>(smem) + threadIdx.x), t(t), nt(nt), width(width), shift(shift) {
        Pack<T, V> zero;
#pragma unroll
        for (int j = 0; j < V; j++) zero.v[j] = from_f32<T>(0.0f);
#pragma unroll
        for (int i = 0; i < NV; i++)
            if ((i * nt + t) * V - shift >= width)
                for (int s = 0; s < STAGES; s++) at[(s * NV + i) * THREADS] = zero;
    }
    __device__ __forceinline__ void fetch(int stage, const T* row) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * nt + t) * V - shift;
            Pack<T, V>* to = at + (stage * NV + i) * THREADS;
            if (c >= width) continue;
            // A last word may hold one element of the row: the copy fills the other with zero.
            if constexpr (V == 2 && sizeof(T) == 2) copy_async_part<4>(to, row + c, c + 1 < width ? 4 : 2);
            else if constexpr (V * sizeof(T) >= 4) copy_async<V * sizeof(T)>(to, row + c);
            else *to = load_pack<T, V>(row + c);
        }
    }
    __device__ __forceinline__ void take(int stage, Pack<T, V> (&raw)[NV]) const {
#pragma unroll
        for (int i = 0; i < NV; i++) raw[i] = at[(stage * NV + i) * THREADS];
        if (V == 2 && shift && t == 0) raw[0].v[0] = from_f32<T>(0.0f);  // the element before the row
    }
};

// Elements 2 p and 2 p + 1 of a thread's share as floats.
template <class T, int V, int NV>
__device__ __forceinline__ f32x2 pair_of(const Pack<T, V> (&raw)[NV], int p) {
    return pair(to_f32(raw[2 * p / V].v[2 * p % V]), to_f32(raw[(2 * p + 1) / V].v[(2 * p + 1) % V]));
}
// Pairs -> the share's vectors in memory (what of them lies in the row).
template <class T, int V, int NV>
__device__ __forceinline__ void store_row(T* row, const f32x2 (&v)[NV * V / 2], int t, int nt, int width, int shift) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * nt + t) * V - shift;
        Pack<T, V> p;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float2 f = unpair(v[(i * V + j) / 2]);
            p.v[j] = from_f32<T>((i * V + j) % 2 ? f.y : f.x);
        }
        if constexpr (V == 2) {
            if (c >= 0 && c + 1 < width) *reinterpret_cast<Pack<T, 2>*>(row + c) = p;
            else if (c >= 0 && c < width) row[c] = p.v[0];
            else if (c == -1) row[0] = p.v[1];
        } else {
            if (c < width) store_pack<T, V>(row + c, p);
        }
    }
}

// A thread's weights, `fallback` where there are none.
template <class T, int V, int NV>
__device__ __forceinline__ void load_share(const void* w, bool w_f32, float fallback, int t, int nt, int width, int shift,
                                           f32x2 (&out)[NV * V / 2]) {
    float f[NV * V];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c0 = (i * nt + t) * V - shift;
        if (V >= 4 && w && c0 < width) {  // whole vectors
            if (w_f32) {
#pragma unroll
                for (int j = 0; j < V / 4; j++) {
                    const Pack<float, 4> r = load_pack<float, 4>(static_cast<const float*>(w) + c0 + 4 * j);
#pragma unroll
                    for (int k = 0; k < 4; k++) f[i * V + 4 * j + k] = r.v[k];
                }
            } else {
                const Pack<T, V> r = load_pack<T, V>(static_cast<const T*>(w) + c0);
#pragma unroll
                for (int j = 0; j < V; j++) f[i * V + j] = to_f32(r.v[j]);
            }
            continue;
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int c = c0 + j;
            f[i * V + j] = w && c >= 0 && c < width ? weight_at<T>(w, w_f32, c) : fallback;
        }
    }
#pragma unroll
    for (int p = 0; p < NV * V / 2; p++) out[p] = pair(f[2 * p], f[2 * p + 1]);
}

// Where this thread's rows start in a word of two elements.
template <class T, int V>
__device__ __forceinline__ int shift_of(int64_t row, int64_t stride) {
    return V == 2 && sizeof(T) == 2 ? (int)((row * stride) & 1) : 0;
}

template <class T, int V, int ELEMS, bool WIDE, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1)
    k_norm_forward(const T* __restrict__ x, int64_t x_stride, const void* __restrict__ w, const void* __restrict__ b,
                   bool w_f32, int64_t rows, int width, float eps, T* __restrict__ y, int64_t y_stride,
                   float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int NV = ELEMS / V, PAIRS = ELEMS / 2, STAGES = stages_of(THREADS, ELEMS * sizeof(T));
    __shared__ float2 red[32];
    extern __shared__ float4 smem4[];  // the ring
    const int t = WIDE ? threadIdx.x : threadIdx.x & 31, nt = WIDE ? blockDim.x : 32;
    int64_t row = WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kWarpsPerBlock + (threadIdx.x >> 5);
    const int64_t step = WIDE ? gridDim.x : (int64_t)gridDim.x * kWarpsPerBlock;
    const int shift = shift_of<T, V>(row, x_stride);
    Ring<T, V, NV, STAGES, THREADS> ring(smem4, t, nt, width, shift);
    for (int k = 0; k < STAGES - 1; k++) {
        if (row + k * step < rows) ring.fetch(k, x + (row + k * step) * x_stride);
        copy_commit();
    }
    f32x2 fw[PAIRS], fb[PAIRS];
    load_share<T, V, NV>(w, w_f32, 1.0f, t, nt, width, shift, fw);
    load_share<T, V, NV>(b, w_f32, 0.0f, t, nt, width, shift, fb);
    for (int stage = 0; row < rows; row += step, stage = (stage + 1) % STAGES) {
        if (STAGES == 1) ring.fetch(0, x + row * x_stride), copy_commit();
        copy_wait<STAGES == 1 ? 0 : STAGES - 2>();
        Pack<T, V> raw[NV];
        ring.take(stage, raw);
        f32x2 v[PAIRS];
#pragma unroll
        for (int p = 0; p < PAIRS; p++) v[p] = pair_of<T, V, NV>(raw, p);
        const int64_t ahead = row + (STAGES - 1) * step;
        if (STAGES > 1 && ahead < rows) ring.fetch((stage + STAGES - 1) % STAGES, x + ahead * x_stride);
        copy_commit();
        f32x2 sum = 0;
#pragma unroll
        for (int p = 0; p < PAIRS; p++) sum = add2(sum, v[p]);
        const float2 s = unpair(sum);
        const float mean =
            row_sums(make_float2(s.x + s.y, 0.0f), red, threadIdx.x >> 5, WIDE ? nt >> 5 : 1).x / (float)width;
        const f32x2 away = pair(-mean, -mean);
        f32x2 sq = 0;
#pragma unroll
        for (int p = 0; p < PAIRS; p++) {
            v[p] = add2(v[p], away);
            // Elements outside the row deviate by 0.  A warp's share is full up to its last 8 elements,
            // but for the element before a shifted row.
            if (WIDE || V == 2 || 2 * p >= ELEMS - 8) {
                const float2 f = unpair(v[p]);
                const int c0 = (2 * p / V * nt + t) * V + 2 * p % V - shift;
                const int c1 = ((2 * p + 1) / V * nt + t) * V + (2 * p + 1) % V - shift;
                v[p] = pair(c0 >= 0 && c0 < width ? f.x : 0.0f, c1 < width ? f.y : 0.0f);
            }
            sq = fma2(v[p], v[p], sq);
        }
        const float2 q = unpair(sq);
        const float var =
            row_sums(make_float2(q.x + q.y, 0.0f), red, threadIdx.x >> 5, WIDE ? nt >> 5 : 1).x / (float)width;
        const float rstd = 1.0f / sqrtf(var + eps);
        if (t == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
        const f32x2 rr = pair(rstd, rstd);
#pragma unroll
        for (int p = 0; p < PAIRS; p++) v[p] = fma2(mul2(v[p], rr), fw[p], fb[p]);
        store_row<T, V, NV>(y + row * y_stride, v, t, nt, width, shift);
    }
}

// Each thread sums dw and db of its columns over its rows, the groups of a
// block join theirs in shared memory in order, and the block writes one
// partial row of part[block][2][width].  `group` threads hold a row.
template <class T, int V, int ELEMS, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 128 ? 3 : 1)
    k_norm_backward(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride,
                    const void* __restrict__ w, bool w_f32, const float* __restrict__ mean_in,
                    const float* __restrict__ rstd_in, int64_t rows, int width, int group, T* __restrict__ dx,
                    int64_t dx_stride, float* __restrict__ part) {
    constexpr int NV = ELEMS / V, PAIRS = ELEMS / 2, STAGES = stages_of(THREADS, 2 * ELEMS * sizeof(T));
    __shared__ float2 red[32];
    extern __shared__ float4 smem4[];  // the rings of x and dy, (mean, rstd); at the end the sums to join
    const int g = threadIdx.x / group, t = threadIdx.x - g * group, groups = blockDim.x / group, warps = group >> 5;
    int64_t row = (int64_t)blockIdx.x * groups + g;
    const int64_t step = (int64_t)gridDim.x * groups;
    constexpr int kRing = STAGES * ELEMS * sizeof(T);  // bytes a thread
    uint8_t* smem = reinterpret_cast<uint8_t*>(smem4);
    const int shift = shift_of<T, V>(row, x_stride);
    Ring<T, V, NV, STAGES, THREADS> ring_x(smem, t, group, width, shift),
        ring_d(smem + kRing * THREADS, t, group, width, shift);
    // (mean, rstd) of each warp's next rows.
    float* stats = reinterpret_cast<float*>(smem + 2 * kRing * THREADS) + (threadIdx.x >> 5) * 2 * STAGES;
    float* joined = reinterpret_cast<float*>(smem);  // [2][width], once the rows are done
    auto fetch = [&](int stage, int64_t r) {
        ring_x.fetch(stage, x + r * x_stride);
        ring_d.fetch(stage, dy + r * dy_stride);
        if ((threadIdx.x & 31) == 0) {
            copy_async<4>(stats + 2 * stage, mean_in + r);
            copy_async<4>(stats + 2 * stage + 1, rstd_in + r);
        }
    };
    for (int k = 0; k < STAGES - 1; k++) {
        if (row + k * step < rows) fetch(k, row + k * step);
        copy_commit();
    }
    f32x2 fw[PAIRS];
    load_share<T, V, NV>(w, w_f32, 1.0f, t, group, width, shift, fw);
    f32x2 dw[PAIRS], db[PAIRS];
#pragma unroll
    for (int p = 0; p < PAIRS; p++) dw[p] = db[p] = 0;
    for (int stage = 0; row < rows; row += step, stage = (stage + 1) % STAGES) {
        if (STAGES == 1) fetch(0, row), copy_commit();
        copy_wait<STAGES == 1 ? 0 : STAGES - 2>();
        __syncwarp();  // lane 0 copied the statistics
        Pack<T, V> px[NV], pd[NV];
        ring_x.take(stage, px);
        ring_d.take(stage, pd);
        f32x2 xh[PAIRS], gy[PAIRS], sg = 0, sgx = 0;
        const f32x2 away = pair(-stats[2 * stage], -stats[2 * stage]), rr = pair(stats[2 * stage + 1], stats[2 * stage + 1]);
#pragma unroll
        for (int p = 0; p < PAIRS; p++) {
            // dy is 0 outside the row, so whatever x and w hold there adds nothing.
            const f32x2 d = pair_of<T, V, NV>(pd, p);
            xh[p] = mul2(add2(pair_of<T, V, NV>(px, p), away), rr);
            gy[p] = mul2(d, fw[p]);
            dw[p] = fma2(d, xh[p], dw[p]);
            db[p] = add2(db[p], d);
            sg = add2(sg, gy[p]);
            sgx = fma2(gy[p], xh[p], sgx);
        }
        __syncwarp();  // the statistics have been read
        const int64_t ahead = row + (STAGES - 1) * step;
        if (STAGES > 1 && ahead < rows) fetch((stage + STAGES - 1) % STAGES, ahead);
        copy_commit();
        if (dx) {
            const float2 a = unpair(sg), b = unpair(sgx);
            const float2 s = row_sums(make_float2(a.x + a.y, b.x + b.y), red, t >> 5, warps);
            const float mg = s.x / (float)width, mgx = s.y / (float)width;
            const f32x2 mg2 = pair(-mg, -mg), mgx2 = pair(-mgx, -mgx);
#pragma unroll
            for (int p = 0; p < PAIRS; p++) gy[p] = mul2(rr, fma2(xh[p], mgx2, add2(gy[p], mg2)));
            store_row<T, V, NV>(dx + row * dx_stride, gy, t, group, width, shift);
        }
    }
    if (!part) return;
    copy_wait<0>();
    __syncthreads();  // the rings are free
    float* out = part + (int64_t)blockIdx.x * 2 * width;
    for (int k = 0; k < groups; k++) {
        float* dst = k + 1 == groups ? out : joined;
        if (g == k) {
#pragma unroll
            for (int e = 0; e < ELEMS; e++) {
                const int c = (e / V * group + t) * V + e % V - shift;
                if (c < 0 || c >= width) continue;
                const float2 fw = unpair(dw[e / 2]), fb = unpair(db[e / 2]);
                dst[c] = (k ? joined[c] : 0.0f) + (e % 2 ? fw.y : fw.x);
                dst[width + c] = (k ? joined[width + c] : 0.0f) + (e % 2 ? fb.y : fb.x);
            }
        }
        __syncthreads();
    }
}

// Column sums of part[n][2][width]: 32 columns of a block, its 32 warps each
// take every 32nd partial row, joined in order.
template <class W>
__global__ void __launch_bounds__(1024) k_norm_join(const float* __restrict__ part, int n, int width,
                                                    W* __restrict__ dw, W* __restrict__ db) {
    __shared__ float s[32][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (c < 2 * width) {
#pragma unroll 4
        for (int i = warp; i < n; i += 32) v += part[(int64_t)i * 2 * width + c];
    }
    s[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && c < 2 * width) {
        for (int k = 1; k < 32; k++) v += s[k][lane];
        if (c < width) {
            if (dw) dw[c] = from_f32<W>(v);
        } else if (db) {
            db[c - width] = from_f32<W>(v);
        }
    }
}

// Backward: threads that hold a row, such groups in a block (of one warp each,
// or one group of several warps), and blocks that stay.
int backward_group(int width) { return width <= 1024 ? 32 : (int)round_up(ceil_div(width, kBlockElems), 32); }
int backward_groups(int width) { return std::max(1, 128 / backward_group(width)); }
int backward_blocks(int64_t rows, int width) {
    const int groups = backward_groups(width), stay = std::max(1, 384 / (backward_group(width) * groups));
    return (int)std::min<int64_t>(ceil_div(rows, groups), 148 * stay);
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

// Lets KERNEL have `BYTES` of dynamic shared memory on the current device.
template <auto KERNEL, size_t BYTES>
void allow_shared() {
    static_assert(BYTES <= 227 * 1024, "shared memory budget");
    static std::atomic<uint64_t> set{0};  // a bit a device
    const uint64_t bit = uint64_t(1) << (current_device() & 63);
    if (BYTES <= 48 * 1024 || (set.load(std::memory_order_relaxed) & bit)) return;
    MDH_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BYTES));
    set.fetch_or(bit, std::memory_order_relaxed);
}

// Elements of a row that its threads have places for: 8, 16, 24 or 32 a lane
// of a warp, kBlockElems a thread of a group of whole warps beyond.
int places_of(int width) { return (int)round_up(width, width <= 1024 ? 256 : 32 * kBlockElems); }

// Elements of a vector: 16 bytes of them, 2 of 16 bits, or 1.  A null
// array does not count.  Rows an odd stride apart begin in the middle of a
// word every other time, so pairs need a place beside the row's; a row that
// fills its places goes by single elements (768 of stride 769, 1,024 of 1,025).
template <class T>
int vector_of(int width, std::initializer_list<std::pair<const void*, int64_t>> arrays, bool weights_aligned) {
    constexpr int V = 16 / sizeof(T);
    bool whole = width % V == 0 && weights_aligned, words = sizeof(T) == 2;
    int64_t parity = -1;
    for (const auto& [p, stride] : arrays) {
        if (!p) continue;
        whole = whole && rows_aligned(p, stride, sizeof(T));
        // Every array's rows start alike in words of 4 bytes.
        words = words && reinterpret_cast<uintptr_t>(p) % 4 == 0 && (parity < 0 || parity == (stride & 1));
        parity = stride & 1;
    }
    words = words && (parity != 1 || width < places_of(width));
    return whole ? V : words ? 2 : 1;
}
template <class T, class F>
void by_vector(int v, F&& fn) {
    if (v == 16 / (int)sizeof(T)) return fn(std::integral_constant<int, 16 / sizeof(T)>{});
    if constexpr (sizeof(T) == 2)
        if (v == 2) return fn(std::integral_constant<int, 2>{});
    fn(std::integral_constant<int, 1>{});
}

// fn(V, ELEMS, WIDE, THREADS) as compile-time values.
template <class T, class F>
void by_shape(int vec, int width, F&& fn) {
    using std::integral_constant;
    const integral_constant<int, 32 * kWarpsPerBlock> small{};
    auto elems = [&](auto v) {
        if (width <= 256) fn(v, integral_constant<int, 8>{}, std::false_type{}, small);
        else if (width <= 512) fn(v, integral_constant<int, 16>{}, std::false_type{}, small);
        else if (width <= 768) fn(v, integral_constant<int, 24>{}, std::false_type{}, small);
        else if (width <= 1024) fn(v, integral_constant<int, 32>{}, std::false_type{}, small);
        else if (width <= 4096) fn(v, integral_constant<int, kBlockElems>{}, std::true_type{}, small);
        else if (width <= 8192) fn(v, integral_constant<int, kBlockElems>{}, std::true_type{}, integral_constant<int, 512>{});
        else fn(v, integral_constant<int, kBlockElems>{}, std::true_type{}, integral_constant<int, 1024>{});
    };
    by_vector<T>(vec, elems);
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
            // One row has no stride of its own.
            const auto at = [&](const void* p, int64_t stride) { return std::make_pair(p, rows > 1 ? stride : (int64_t)width); };
            const int vec = vector_of<T>(width, {at(x, x_stride), at(y, y_stride)}, aligned16(w) && aligned16(b));
            by_shape<T>(vec, width, [&](auto v, auto elems, auto wide, auto most) {
                const int threads = wide ? (int)round_up(ceil_div(width, elems), 32) : 32 * kWarpsPerBlock;
                const int64_t units = wide ? rows : ceil_div(rows, kWarpsPerBlock);
                constexpr int kShare = elems * sizeof(T), kRing = stages_of(most, kShare) * kShare;
                const int smem = kRing * most;
                // Blocks that stay: 512 threads an SM, as far as their rings fit.
                const int64_t stay = 148 * std::min(std::max(1, 512 / threads), blocks_that_fit(smem));
                allow_shared<k_norm_forward<T, v, elems, wide, most>, most * kRing>();
                k_norm_forward<T, v, elems, wide, most>
                    <<<(unsigned)std::min(units, stay), threads, smem, (cudaStream_t)stream>>>((const T*)x, x_stride, w, b, w_dtype == MDH_F32, rows, width, eps, (T*)y,
                                               y_stride, mean, rstd);
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
        const int most_blocks = backward_blocks(rows, width);
        int parts = 0;
        by_dtype(dtype, [&](auto zero) {
            using T = decltype(zero);
            const auto at = [&](const void* p, int64_t stride) { return std::make_pair(p, rows > 1 ? stride : (int64_t)width); };
            const int vec = vector_of<T>(width, {at(x, x_stride), at(dy, dy_stride), at(dx, dx_stride)}, aligned16(w));
            const int group = backward_group(width), groups = backward_groups(width);
            auto launch = [&](auto v, auto elems, auto most) {
                constexpr int kShare = 2 * elems * sizeof(T), kStages = stages_of(most, kShare);
                const int rings = most * kStages * kShare + 8 * kStages * (group * groups / 32);
                const int smem = std::max(rings, groups > 1 ? 2 * width * 4 : 0);
                const int blocks = std::min(most_blocks, 148 * blocks_that_fit(smem));
                if (sums) parts = blocks;
                allow_shared<k_norm_backward<T, v, elems, most>, most * kStages * kShare + 8192>();
                k_norm_backward<T, v, elems, most><<<blocks, group * groups, smem, st>>>(
                    (const T*)dy, dy_stride, (const T*)x, x_stride, w, w_dtype == MDH_F32, mean, rstd, rows, width,
                    group, (T*)dx, dx_stride, sums ? (float*)ws : nullptr);
            };
            using std::integral_constant;
            auto by_elems = [&](auto v) {
                if (width <= 256) launch(v, integral_constant<int, 8>{}, integral_constant<int, 128>{});
                else if (width <= 512) launch(v, integral_constant<int, 16>{}, integral_constant<int, 128>{});
                else if (width <= 768) launch(v, integral_constant<int, 24>{}, integral_constant<int, 128>{});
                else if (width <= 1024) launch(v, integral_constant<int, 32>{}, integral_constant<int, 128>{});
                else if (width <= 4096) launch(v, integral_constant<int, kBlockElems>{}, integral_constant<int, 256>{});
                else if (width <= 8192) launch(v, integral_constant<int, kBlockElems>{}, integral_constant<int, 512>{});
                else launch(v, integral_constant<int, kBlockElems>{}, integral_constant<int, 1024>{});
            };
            by_vector<T>(vec, by_elems);
        });
        check_launch();
        if (!sums) return;
        by_dtype(w_dtype, [&](auto zero) {
            using W = decltype(zero);
            k_norm_join<W><<<(unsigned)ceil_div(2 * (int64_t)width, 32), 1024, 0, st>>>((const float*)ws, parts, width,
                                                                                    (W*)dw, (W*)db);
        });
        check_launch();
    });
}

}  // extern "C"
