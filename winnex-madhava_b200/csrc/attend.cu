// Attention of queries over the rows that a search found for them, keys and
// values from 8-bit row caches.
//
//   s_j = scale q . k_j;  cap > 0: s_j = cap tanh(s_j / cap);  s_j += bias_j
//   out = sum_j p_j v_j,  p = softmax(s) over the entries that are not hidden
// in one pass: a running maximum m, sum l and vector, rescaled when m grows.
// Backward, with dP_j = dout . v_j, D = sum_j p_j dP_j, t_j = tanh(...):
//   dbias_j = sum over heads of p_j (dP_j - D)
//   dq = scale sum_j p_j (dP_j - D) (1 - t_j^2) k_j = scale (A - D B),
//   A = sum_j p_j dP_j (1 - t_j^2) k_j,  B = sum_j p_j (1 - t_j^2) k_j:
// one pass over the rows as well, since p_j follows from lse.  A gradient of
// lse itself adds p_j dlse to each score's: D - dlse stands for D.
//
// A unit is a head of the rows and up to kMaxShared query heads that share it.
// LANES lanes hold a row's head, 8 elements each (an 8-byte load of codes); the
// 32 / LANES lane groups of a warp take units side by side (a row's
// neighbouring heads: nothing to join) and, where a call has too few units,
// entries side by side.  A block takes one query and a range of its list: it
// first lists the range's visible entries in shared memory (ids, documents and
// biases are read once for all units); then its warps share the units and, if
// there are more warps, slices of that list.  Each lane copies the codes and
// scales it will use into its own shared memory (cp.async), STEPS entries a
// stage and some stages ahead: rows lie anywhere in a large cache, and what
// bounds short lists is the latency of reaching them.  The STEPS x heads partial
// products of a lane are summed by halving: each step sends half of the values
// to the partner lane, so a lane ends with one finished score and the softmax
// arithmetic is done once per score.  Entries side by side and slices are
// joined in the block, ranges of other blocks by a second kernel, in a fixed
// order.  On B200: 4,096 queries x 100 entries (a quarter visible) x 12 heads
// of 64 in 82 us, bound by instructions; 2,048 queries x 64 entries x 12 heads
// on 4 in 49 us forward, 67 + 9 us backward; 8 queries x 4,096 entries x 16
// heads of 128 on 2 in 19 + 4 us by the matrix form (36 + 5 us by lanes).
//
// Codes become floats without a conversion instruction: the byte c + 128 in
// the mantissa of 2^23 is the float 8388736 + c, and one subtraction (two
// values at a time) leaves c exactly.  The row's scale multiplies the finished
// 8-term sums; the affine code's offset enters as a constant times the sum of
// the query's elements, or of the weights.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "op_rows.cuh"

namespace mdh {
namespace {

using namespace op;

constexpr int kMaxWarps = 8;          // of a block, forward
constexpr int kMaxWarpsBack = 4;      // backward: its warps hold twice the vectors
constexpr int kRound = 128;           // entries of the list that a warp looks at at a time
constexpr int kMaxHead = 256;
constexpr int kMaxShared = 4;         // query heads of a unit
constexpr int kMaxSharedMma = 8;      // ... in the matrix form
constexpr int kMinSlice = 16;         // entries below which a list is not cut further

struct CodeView {
    const uint8_t* codes;
    const float* scales;  // null: affine
    uint32_t stride;
    int group, n_groups;
    uint32_t flip;        // 0x80808080 for int8: the stored byte becomes c + 128
    float scale, base;    // affine: value = base + scale c
};

// How a call's rows are read: byte by byte, 8 bytes a lane, or by the matrix form.
enum { kFormBytes = 0, kFormLanes = 1, kFormMma = 2 };

struct AttendParams {
    CodeView k, v;
    const void* q;
    const int32_t* ids;
    const float* bias;
    const int32_t *query_docs, *row_docs;
    int64_t q_stride, q_head_stride, ids_stride, bias_stride, slots;
    int64_t queries;
    int found, heads, shared, head, dtype;
    bool q_vec, dout_vec;  // heads start on 16 bytes
    float scale, cap, inv_cap;
    int r_blocks, rb;      // units of a row's head, query heads of each (the last may have fewer)
    int units;             // of a query
    int entries_log;       // log2 of the entries side by side in a warp
    int block_warps;       // warps of a block that take different units
    int unit_blocks;       // blocks that share a query's units
    int slices;            // warps of a block that share their units
    int splits, split_len; // ranges of a list over blocks, entries of each
    int form;              // kForm*
    void* out;
    float* lse;
    float* part;           // splits > 1: vectors [splits][queries][heads][head] (backward: two of them), then float2
                           // [splits][queries][heads] (m, l) or (D, P)
    // backward
    const void* dout;
    const float* lse_in;
    const float* dlse;     // or null
    float2* pd;            // [queries][heads][found] p dP and p, or null
    float2* sum_d;         // [queries][heads] D / P - dlse and 1 / P, or null
};

using u64 = f32x2;
// The codes c as four pairs of floats.
__device__ __forceinline__ void code_pairs(uint2 raw, uint32_t flip, u64 (&c)[4]) {
    const uint32_t w[2] = {raw.x ^ flip, raw.y ^ flip};
    const u64 off = pair(-8388736.0f, -8388736.0f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t x = w[i >> 1], lo = __byte_perm(x, 0x4B000000u, (i & 1) ? 0x7652 : 0x7650),
                       hi = __byte_perm(x, 0x4B000000u, (i & 1) ? 0x7653 : 0x7651);
        c[i] = add2(pair(__uint_as_float(lo), __uint_as_float(hi)), off);
    }
}
__device__ __forceinline__ float dot_pairs(const u64 (&a)[4], const u64 (&b)[4]) {
    u64 s = mul2(a[0], b[0]);
#pragma unroll
    for (int i = 1; i < 4; i++) s = fma2(a[i], b[i], s);
    const float2 f = unpair(s);
    return f.x + f.y;
}

// 8 elements of q's type at p + i; vec: on a 16-byte boundary.
__device__ __forceinline__ void load_elements(const void* p, int64_t i, int dtype, bool vec, float (&v)[8]) {
    if (dtype == MDH_F32) {
        const float* f = static_cast<const float*>(p) + i;
        if (vec) {
            const float4 x = __ldg(reinterpret_cast<const float4*>(f)), y = __ldg(reinterpret_cast<const float4*>(f) + 1);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = f[j];
        }
        return;
    }
    const uint16_t* h = static_cast<const uint16_t*>(p) + i;
    uint32_t w[4];
    if (vec) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(h));
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (dtype == MDH_BF16) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            v[2 * j] = f.x, v[2 * j + 1] = f.y;
        }
    }
}
// 8 elements at place i (a multiple of 8) of an aligned output.
__device__ __forceinline__ void store_elements(void* p, int64_t i, int dtype, const float (&v)[8]) {
    if (dtype == MDH_F32) {
        float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        f[0] = make_float4(v[0], v[1], v[2], v[3]);
        f[1] = make_float4(v[4], v[5], v[6], v[7]);
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (dtype == MDH_BF16) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&x);
        } else {
            const __half2 x = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&x);
        }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
}

// 4 elements of q's type at p + i; vec: on the bytes they take.
__device__ __forceinline__ void load4(const void* p, int64_t i, int dtype, bool vec, float (&v)[4]) {
    if (dtype == MDH_F32) {
        const float* f = static_cast<const float*>(p) + i;
        if (vec) {
            const float4 x = __ldg(reinterpret_cast<const float4*>(f));
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = f[j];
        }
        return;
    }
    const uint16_t* h = static_cast<const uint16_t*>(p) + i;
    uint2 w;
    if (vec) w = __ldg(reinterpret_cast<const uint2*>(h));
    else w = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    if (dtype == MDH_BF16) {
        v[0] = __uint_as_float(w.x << 16), v[1] = __uint_as_float(w.x & 0xffff0000u);
        v[2] = __uint_as_float(w.y << 16), v[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
        v[0] = x.x, v[1] = x.y, v[2] = y.x, v[3] = y.y;
    }
}
// 4 elements at place i (a multiple of 4) of an aligned output.
__device__ __forceinline__ void store4(void* p, int64_t i, int dtype, float4 v) {
    if (dtype == MDH_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = v;
        return;
    }
    uint2 w;
    if (dtype == MDH_BF16) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
        w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    } else {
        const __half2 x = __floats2half2_rn(v.x, v.y), y = __floats2half2_rn(v.z, v.w);
        w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = w;
}

// What a lane works on.
struct Work {
    int64_t i;       // query
    int h0, nr;      // first head, heads (0: an idle lane group)
    int e0;          // this lane's first element of a row
    int d0;          // ... of a head
    bool live;       // the lane holds elements (a head may end inside the lane group)
    int entry;       // of the entries side by side
    int slice;
    bool idle;       // the whole warp has no unit
};
template <int LANES>
__device__ __forceinline__ Work work_of(const AttendParams& a) {
    Work w;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LANES;
    const int side_log = (LANES == 1 ? 5 : LANES == 2 ? 4 : LANES == 4 ? 3 : LANES == 8 ? 2 : LANES == 16 ? 1 : 0) -
                         a.entries_log;  // units side by side
    w.i = blockIdx.x / (unsigned)a.unit_blocks;
    const int wu = (int)(blockIdx.x - w.i * a.unit_blocks) * a.block_warps + warp / a.slices;
    const int unit = (wu << side_log) + (sub >> a.entries_log);
    w.slice = warp % a.slices;
    w.entry = sub & ((1 << a.entries_log) - 1);
    w.idle = wu << side_log >= a.units;
    const int u = min(unit, a.units - 1), g = u / a.r_blocks, r0 = (u - g * a.r_blocks) * a.rb;
    w.h0 = g * a.shared + r0;
    w.nr = unit < a.units ? min(a.rb, a.shared - r0) : 0;
    w.d0 = (lane % LANES) * 8;
    w.live = w.d0 < a.head && w.nr > 0;
    w.e0 = g * a.head + (w.live ? w.d0 : 0);
    return w;
}

// Entry j of the list: its slot, or -1 when it is hidden; its bias.
__device__ __forceinline__ int entry_slot(const AttendParams& a, int64_t i, int j, int32_t doc, float& bias) {
    const int id = __ldg(a.ids + i * a.ids_stride + j);
    bias = a.bias ? __ldg(a.bias + i * a.bias_stride + j) : 0.0f;
    if (id < 0 || id >= a.slots || bias == -INFINITY) return -1;
    if (a.row_docs && __ldg(a.row_docs + id) != doc) return -1;
    return id;
}

// The visible entries of a range, in order (shared memory, kRound a warp).
struct Entries {
    int* slot;
    float* bias;
    int* place;   // in the query's list
    int* count;   // of each warp
};
constexpr int kEntriesBytes = kRound * 12 + 16;  // a warp
__device__ __forceinline__ Entries entries_at(uint8_t* p, int warps) {
    int* q = reinterpret_cast<int*>(p);
    const int n = warps * kRound;
    return {q, reinterpret_cast<float*>(q + n), q + 2 * n, q + 3 * n};
}
// Lists the visible entries of [j0, j1), at most kRound a warp.
__device__ __forceinline__ int list_entries(const AttendParams& a, const Entries& e, int64_t i, int32_t doc, int j0, int j1) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int warps = min((int)blockDim.x >> 5, (j1 - j0 + kRound - 1) / kRound);  // that look at entries
    int slot[kRound / 32], n = 0;
    float bias[kRound / 32];
    uint32_t seen[kRound / 32];
    if (warp < warps) {
#pragma unroll
        for (int c = 0; c < kRound / 32; c++) {
            const int j = j0 + warp * kRound + c * 32 + lane;
            slot[c] = -1;
            if (j < j1) slot[c] = entry_slot(a, i, j, doc, bias[c]);
        }
#pragma unroll
        for (int c = 0; c < kRound / 32; c++) {
            seen[c] = __ballot_sync(0xffffffffu, slot[c] >= 0);
            n += __popc(seen[c]);
        }
    }
    __syncthreads();  // the previous list has been read
    if (lane == 0 && warp < warps) e.count[warp] = n;
    __syncthreads();
    int before = 0, total = 0;
    for (int k = 0; k < warps; k++) {
        const int x = e.count[k];
        if (k < warp) before += x;
        total += x;
    }
    if (warp < warps) {
#pragma unroll
    for (int c = 0; c < kRound / 32; c++) {
        if (slot[c] >= 0) {
            const int at = before + __popc(seen[c] & ((1u << lane) - 1u));
            e.slot[at] = slot[c];
            e.bias[at] = bias[c];
            e.place[at] = j0 + warp * kRound + c * 32 + lane;
        }
        before += __popc(seen[c]);
    }
    }
    __syncthreads();
    return total;
}
// Entries [lo, hi) of n that a slice takes: multiples of `step` but for the end.
__device__ __forceinline__ void slice_of(int n, int slice, int slices, int step, int& lo, int& hi) {
    const int per = ((n + slices - 1) / slices + step - 1) / step * step;
    lo = min(slice * per, n);
    hi = min(lo + per, n);
}

// Sums over LANES lanes by halving.  In: N values a lane (N a power of two).
// Out: KEEP = max(1, N / LANES) finished values a lane, v[x] the sum of the
// values number value_of(lane, x) over the lane group.
template <int LANES, int N>
struct Halving {
    static constexpr int KEEP = N > LANES ? N / LANES : 1;
    static constexpr int BITS = N > LANES ? LANES : N;  // lanes that hold different values
    static constexpr int DUP = LANES / BITS;            // lanes that hold the same
    static __device__ __forceinline__ void sum(float (&v)[N]) {
        const int lane = threadIdx.x & 31;
        int n = N;
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) {
            if (n > KEEP) {
                n >>= 1;
                const bool up = lane & o;
#pragma unroll
                for (int x = 0; x < N / 2; x++) {
                    if (x >= n) break;
                    const float keep = up ? v[n + x] : v[x], send = up ? v[x] : v[n + x];
                    v[x] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                }
            } else {
#pragma unroll
                for (int x = 0; x < KEEP; x++) v[x] += __shfl_xor_sync(0xffffffffu, v[x], o);
            }
        }
    }
    // Number of the lane's value x.
    static __device__ __forceinline__ int value_of(int x) { return (threadIdx.x & 31) % LANES / DUP * KEEP + x; }
    // The lane of this lane's group that holds value number v (in its place v % KEEP).
    static __device__ __forceinline__ int lane_of(int v) { return (threadIdx.x & 31) / LANES * LANES + v / KEEP * DUP; }
    template <class T>
    static __device__ __forceinline__ T get(const T (&v)[KEEP], int number) {
        return __shfl_sync(0xffffffffu, v[number % KEEP], lane_of(number));
    }
};

template <int LANES, int RB>
struct Steps {
    static constexpr int RP = RB == 3 ? 4 : RB;                    // heads, as a power of two
    static constexpr int WANT = RB > 2 ? 2 : 4;
    static constexpr int N = WANT > LANES ? LANES : WANT;          // entries of a stage
    static constexpr int STAGES = N == 4 ? 2 : 4;
    static constexpr int RING = STAGES * N * 768;                  // bytes a warp: codes and scales of its lanes
    using Sums = Halving<LANES, N * RP>;                           // value number step * RP + head
    static_assert(RING >= 576 * 4, "the joined vectors lie in the rings");
    // Over the lanes that hold the same head: the bits of the step and of the entry side by side.
    template <class F>
    static __device__ __forceinline__ void over_entries(int entries_log, F&& f) {
        for (int k = 0; k < entries_log; k++) f(LANES << k);
#pragma unroll
        for (int o = LANES / 2; o >= LANES / N && o > 0; o >>= 1) f(o);
    }
};

// q (times the scale) or dout of a unit's heads as float pairs; sums of each.
template <int RB>
__device__ __forceinline__ void load_heads(const void* p, int64_t at, int64_t stride, int dtype, const Work& w,
                                           bool vec, float scale, u64 (&v)[RB][4], float (&sum)[RB]) {
#pragma unroll
    for (int r = 0; r < RB; r++) {
        float x[8] = {};
        if (w.live && r < w.nr) load_elements(p, at + (w.h0 + r) * stride + w.d0, dtype, vec, x);
        sum[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) sum[r] += x[j] *= scale;
#pragma unroll
        for (int j = 0; j < 4; j++) v[r][j] = pair(x[2 * j], x[2 * j + 1]);
    }
}

// Sums over the entries side by side.
template <int LANES>
__device__ __forceinline__ void join_vectors(u64 (&v)[4], int entries_log, float (&out)[8]) {
    for (int k = 0; k < entries_log; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = add2(v[j], __shfl_xor_sync(0xffffffffu, v[j], LANES << k));
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 f = unpair(v[j]);
        out[2 * j] = f.x, out[2 * j + 1] = f.y;
    }
}
__device__ __forceinline__ void put8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void get8(const float* p, float (&v)[8]) {
    const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
}

// The scaled, capped and biased score of a finished sum; t = tanh of the
// capped one.  The softmax's functions are the accurate ones: lse and dbias
// are float32 results, an error of a score is one of its weight, and a cap
// multiplies the tanh's error (4e-6 under a cap of 20 with the hardware's 2^x
// alone).  They cost nothing measurable: one call a finished score.
__device__ __forceinline__ float score_of(const AttendParams& a, float x, float bias, float& t) {
    t = 0.0f;
    if (a.cap > 0.0f) {
        t = tanhf(x * a.inv_cap);
        x = a.cap * t;
    }
    return x + bias;
}

// Joins two running softmaxes (m, l, vector scaled alike): the factors for
// each side.
__device__ __forceinline__ float join(float m, float mo, float& mine, float& other) {
    const float top = fmaxf(m, mo), ref = top == -INFINITY ? 0.0f : top;
    mine = expf(m - ref);
    other = expf(mo - ref);
    return top;
}

// The 8 elements from d of (query, head) `at`.
__device__ __forceinline__ void finish_forward(const AttendParams& a, int64_t at, int d, float (&v)[8], float m, float l) {
    const float inv = l != 0.0f ? 1.0f / l : 0.0f, base = l != 0.0f ? a.v.base : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = fmaf(v[j], inv, base);
    store_elements(a.out, at * a.head + d, a.dtype, v);
    if (d == 0) a.lse[at] = l != 0.0f ? m + logf(l) : -INFINITY;
}
__device__ __forceinline__ void finish_backward(const AttendParams& a, int64_t at, int d, float (&x)[8],
                                                const float (&y)[8], float sum_d, float sum_p) {
    const float inv = sum_p != 0.0f ? 1.0f / sum_p : 0.0f, f = a.scale * inv;
    sum_d *= inv;
    if (a.dlse && sum_p != 0.0f) sum_d -= __ldg(a.dlse + at);  // a list without entries has no gradient
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = f * (x[j] - sum_d * y[j]);
    store_elements(a.out, at * a.head + d, a.dtype, x);
    if (a.sum_d && d == 0) a.sum_d[at] = make_float2(sum_d, inv);
}

// Where a lane reads rows.
struct Places {
    const uint8_t *k, *v;
    const float *ks, *vs;
    uint32_t k_stride, v_stride, kn, vn;
    float k_scale, v_scale;
};
__device__ __forceinline__ Places places_of(const AttendParams& a, const Work& w) {
    return {a.k.codes + w.e0, a.v.codes + w.e0, a.k.scales ? a.k.scales + w.e0 / a.k.group : nullptr,
            a.v.scales ? a.v.scales + w.e0 / a.v.group : nullptr, a.k.stride, a.v.stride, (uint32_t)a.k.n_groups,
            (uint32_t)a.v.n_groups,
            a.k.scale, a.v.scale};
}
// A lane's place in a stage: codes of key and value (8 bytes), their scales.
struct Slot {
    uint8_t* at;
    __device__ __forceinline__ uint2* codes(int u, int value) const {
        return reinterpret_cast<uint2*>(at + u * 768 + value * 256) + (threadIdx.x & 31);
    }
    __device__ __forceinline__ float* scale(int u, int value) const {
        return reinterpret_cast<float*>(at + u * 768 + 512 + value * 128) + (threadIdx.x & 31);
    }
};
// What a lane uses of one stage's keys or values.
template <int STEPS>
struct Taken {
    uint2 codes[STEPS];
    float scale[STEPS];
    __device__ __forceinline__ void take(const Slot& s, int value, bool scales, float constant) {
#pragma unroll
        for (int u = 0; u < STEPS; u++) {
            codes[u] = *s.codes(u, value);
            scale[u] = scales ? *s.scale(u, value) : constant;
        }
    }
};
template <bool ALIGNED>
__device__ __forceinline__ void fetch_codes(uint2* dst, const uint8_t* src, bool some) {
    if (ALIGNED) return copy_async<8>(dst, src, some);
    uint2 r = make_uint2(0, 0);
    if (some) {
#pragma unroll
        for (int j = 0; j < 4; j++) r.x |= (uint32_t)src[j] << (8 * j), r.y |= (uint32_t)src[4 + j] << (8 * j);
    }
    *dst = r;
}
// Starts the copies of one stage: entries first, first + (1 << entries_log), ...
template <bool ALIGNED, int STEPS>
__device__ __forceinline__ void fetch(Slot to, const Places& p, const int* slots, int first, int entries_log, int hi,
                                      bool live) {
#pragma unroll
    for (int u = 0; u < STEPS; u++) {
        const int e = first + (u << entries_log);
        const bool some = e < hi && live;
        const uint64_t slot = some ? (uint32_t)slots[e] : 0u;  // 32 x 32 bits: rows may lie past 4 GB
        fetch_codes<ALIGNED>(to.codes(u, 0), p.k + slot * p.k_stride, some);
        fetch_codes<ALIGNED>(to.codes(u, 1), p.v + slot * p.v_stride, some);
        if (p.ks) copy_async<4>(to.scale(u, 0), p.ks + slot * p.kn, some);
        if (p.vs) copy_async<4>(to.scale(u, 1), p.vs + slot * p.vn, some);
    }
    copy_commit();
}
template <int LANES, int RB, bool ALIGNED>
__global__ void __launch_bounds__(32 * kMaxWarps, RB == 1 ? 3 : 2) k_attend(const __grid_constant__ AttendParams a) {
    using St = Steps<LANES, RB>;
    using Sums = typename St::Sums;
    constexpr int STEPS = St::N, RP = St::RP, KEEP = Sums::KEEP;
    constexpr int STAGES = St::STAGES;
    extern __shared__ uint8_t sm[];  // the warps' rings, later the vectors to join; then the entries
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, step = STEPS << a.entries_log;
    const Work w = work_of<LANES>(a);
    const int warps = blockDim.x >> 5;
    const Entries list = entries_at(sm + warps * St::RING, warps);
    const Slot ring{sm + warp * St::RING};
    u64 q[RB][4], acc[RB][4];
    float kb[RB];
    load_heads<RB>(a.q, w.i * a.q_stride, a.q_head_stride, a.dtype, w, a.q_vec, a.scale, q, kb);
#pragma unroll
    for (int r = 0; r < RB; r++) {
        kb[r] *= a.k.base;
#pragma unroll
        for (int j = 0; j < 4; j++) acc[r][j] = 0;
    }
    float m[KEEP], l[KEEP];  // of the lane's own values' heads
#pragma unroll
    for (int x = 0; x < KEEP; x++) m[x] = -INFINITY, l[x] = 0.0f;
    const Places places = places_of(a, w);
    const int32_t doc = a.query_docs ? a.query_docs[w.i] : 0;
    const int j0 = (int)min((int64_t)blockIdx.y * a.split_len, (int64_t)a.found);
    const int j1 = (int)min((int64_t)j0 + a.split_len, (int64_t)a.found);
    for (int from = j0; from < j1; from += (blockDim.x >> 5) * kRound) {
        int lo, hi;
        slice_of(list_entries(a, list, w.i, doc, from, j1), w.slice, a.slices, step, lo, hi);
        if (w.idle) hi = lo;
        copy_wait<0>();  // the previous range's last (empty) stages
#pragma unroll
        for (int k = 0; k < STAGES - 1; k++)
            fetch<ALIGNED, STEPS>({ring.at + k * STEPS * 768}, places, list.slot, lo + k * step + w.entry, a.entries_log,
                                  hi, w.live);
        int stage = 0, ahead = STAGES - 1;
        for (int t = lo; t < hi; t += step) {
            copy_wait<STAGES - 2>();
            const Slot now{ring.at + stage * STEPS * 768};
            fetch<ALIGNED, STEPS>({ring.at + ahead * STEPS * 768}, places, list.slot,
                                  t + (STAGES - 1) * step + w.entry, a.entries_log, hi, w.live);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            ahead = ahead + 1 == STAGES ? 0 : ahead + 1;
            Taken<STEPS> key, value;
            key.take(now, 0, places.ks, places.k_scale);
            value.take(now, 1, places.vs, places.v_scale);
            float s[STEPS * RP];
#pragma unroll
            for (int u = 0; u < STEPS; u++) {
                u64 c[4];
                code_pairs(key.codes[u], a.k.flip, c);
#pragma unroll
                for (int r = 0; r < RP; r++) s[u * RP + r] = r < RB ? fmaf(key.scale[u], dot_pairs(q[r < RB ? r : 0], c), kb[r < RB ? r : 0]) : 0.0f;
            }
            Sums::sum(s);
            float p[KEEP], keep[KEEP];
            bool grown = false;
#pragma unroll
            for (int x = 0; x < KEEP; x++) {
                const int e = t + (Sums::value_of(x) / RP << a.entries_log) + w.entry;
                float th;
                p[x] = e < hi ? score_of(a, s[x], list.bias[e], th) : -INFINITY;
                float top = p[x];
                St::over_entries(a.entries_log, [&](int o) { top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o)); });
                top = fmaxf(top, m[x]);
                grown |= top > m[x];
                const float ref = top == -INFINITY ? 0.0f : top;
                keep[x] = expf(m[x] - ref);
                m[x] = top;
                p[x] = expf(p[x] - ref);
                l[x] = l[x] * keep[x] + p[x];
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const float k = Sums::get(keep, r);  // every step's lanes hold the same
                    const u64 kk = pair(k, k);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[r][j] = mul2(acc[r][j], kk);
                }
            }
#pragma unroll
            for (int u = 0; u < STEPS; u++) {
                u64 c[4];
                code_pairs(value.codes[u], a.v.flip, c);
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const float pv = Sums::get(p, u * RP + r) * value.scale[u];
                    const u64 pp = pair(pv, pv);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[r][j] = fma2(pp, c[j], acc[r][j]);
                }
            }
        }
    }
    copy_wait<0>();
#pragma unroll
    for (int x = 0; x < KEEP; x++)
        St::over_entries(a.entries_log, [&](int o) { l[x] += __shfl_xor_sync(0xffffffffu, l[x], o); });
#pragma unroll
    for (int r = 0; r < RB; r++) {
        float v[8], mm = Sums::get(m, r), ll = Sums::get(l, r);
        join_vectors<LANES>(acc[r], a.entries_log, v);
        if (a.slices > 1) {
            __syncthreads();  // the rings, or the previous head's vectors, have been read
            float* mine = reinterpret_cast<float*>(sm) + warp * 320;
            put8(mine + lane * 8, v);
            reinterpret_cast<float2*>(mine + 256)[lane] = make_float2(mm, ll);
            __syncthreads();
            if (w.slice == 0) {
                for (int k = 1; k < a.slices; k++) {
                    const float* src = mine + k * 320;
                    const float2 ml = reinterpret_cast<const float2*>(src + 256)[lane];
                    float o[8], f, g;
                    get8(src + lane * 8, o);
                    mm = join(mm, ml.x, f, g);
                    ll = ll * f + ml.y * g;
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] = v[j] * f + o[j] * g;
                }
            }
        }
        if (r >= w.nr || w.slice != 0 || !w.live || w.entry != 0) continue;
        const int64_t at = w.i * a.heads + w.h0 + r, n = a.queries * a.heads, row = (int64_t)blockIdx.y * n + at;
        if (a.part) {
            put8(a.part + row * a.head + w.d0, v);
            if (w.d0 == 0) reinterpret_cast<float2*>(a.part + a.splits * n * a.head)[row] = make_float2(mm, ll);
        } else {
            finish_forward(a, at, w.d0, v, mm, ll);
        }
    }
}

// ------------------------------------------------------------ matrix form
// Where two or more query heads share a row, the tensor cores take both
// products (mma.sync m16n8k16, float32 sums): a warp holds one unit, up to 8
// heads, and 16 entries at a time.
//
// Scores: A rows 0-7 are the heads' queries and B the key codes, exact in
// float16 (bytes of 1024 + (c + 128) less 1152) and in bfloat16 (a byte's low 7
// bits over 128 less 128 or 256, its top bit).  16-bit queries are taken in
// their own type, float32 ones as three bfloat16 parts (rows 8-15 hold the
// second and, in a product of their own, the third): all their bits at any
// size, since an element may count where larger ones meet keys of 0.  Values: A
// are the value codes with dimensions as rows, in bfloat16, B the weights p
// times the row's scale as three bfloat16 parts: 24 bits at any size, since a
// weight may count where the larger ones' values are 0.  A lane finds its codes
// as 32-bit words: which
// dimension a word's bytes stand for is the same on both sides of a product,
// so no byte moves between lanes.  Each entry's head lies in shared memory
// 16 bytes past a multiple of the bank width, so those words hit all banks.
constexpr int kMmaEntries = 16;
template <int NS>  // of 16 dimensions
struct Mma {
    static constexpr int HEAD = NS * 16;
    static constexpr int ROW = HEAD + 16;                         // bytes of an entry
    static constexpr int STAGE = 2 * kMmaEntries * ROW + 2 * kMmaEntries * 4;
    static constexpr int STAGES = 3;
    static constexpr int RING = STAGES * STAGE;
    static constexpr int JOIN = kMaxSharedMma * (HEAD + 2) * 4;   // vectors, m, l of a warp
    static_assert(JOIN <= RING && STAGE % 16 == 0, "the joined vectors lie in the rings");
};

__device__ __forceinline__ void mma16816_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Bytes c (two's complement) split into low 7 bits and top bit -> the pair of
// bfloat16 c: bytes 0 and 1, or 2 and 3.
__device__ __forceinline__ uint32_t bf16_codes(uint32_t low, uint32_t top, bool high) {
    const uint32_t x = __byte_perm(low, 0x43434343u, high ? 0x4342 : 0x4140), y = __byte_perm(top, 0x43434343u, high ? 0x4342 : 0x4140);
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Two floats as three bfloat16 parts each.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&part)[3]) {
#pragma unroll
    for (int k = 0; k < 3; k++) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        part[k] = *reinterpret_cast<const uint32_t*>(&h);
        x -= __uint_as_float(part[k] << 16);
        y -= __uint_as_float(part[k] & 0xffff0000u);
    }
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Bytes c + 128 -> the pair of float16 c: bytes 0 and 1, or 2 and 3.
__device__ __forceinline__ uint32_t half_codes(uint32_t w, bool high) {
    const uint32_t x = __byte_perm(w, 0x64646464u, high ? 0x4342 : 0x4140);
    const __half2 off = __half2half2(__ushort_as_half(0xE480));  // -1152
    const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&x), off);
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Four elements of a query as A's registers: of its own 16-bit type two, of
// float32 three bfloat16 parts of two each, cut off rather than rounded (no part
// leaves the float range).  An infinity is its first part.
template <class Q>
struct Query {
    static constexpr int REGS = sizeof(Q) == 2 ? 2 : 6;
    static constexpr bool BF16_CODES = !std::is_same<Q, f16>::value;
    static __device__ __forceinline__ void set(const float (&x)[4], uint32_t (&r)[REGS]) {
        if constexpr (std::is_same<Q, f16>::value) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
                r[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
        } else {
            float v[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int k = 0; k < REGS / 2; k++) {
                uint32_t top[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    top[j] = __float_as_uint(v[j]);
                    if (REGS > 2) v[j] = fabsf(v[j]) == INFINITY ? 0.0f : v[j] - __uint_as_float(top[j] & 0xffff0000u);
                }
                r[2 * k] = __byte_perm(top[0], top[1], 0x7632);
                r[2 * k + 1] = __byte_perm(top[2], top[3], 0x7632);
            }
        }
    }
    // d += 16 dimensions' products with the codes of `word` (bytes c + 128, or c for bfloat16).
    static __device__ __forceinline__ void dot(float (&d)[4], const uint32_t (&r)[REGS], uint32_t word) {
        if constexpr (std::is_same<Q, f16>::value) {
            mma16816(d, {r[0], 0u, r[1], 0u}, half_codes(word, false), half_codes(word, true));
        } else {
            const uint32_t low = word & 0x7f7f7f7fu, top = word & 0x80808080u;
            const uint32_t b0 = bf16_codes(low, top, false), b1 = bf16_codes(low, top, true);
            if constexpr (REGS == 2) {
                mma16816_bf16(d, {r[0], 0u, r[1], 0u}, b0, b1);
            } else {
                mma16816_bf16(d, {0u, r[4], 0u, r[5]}, b0, b1);
                mma16816_bf16(d, {r[0], r[2], r[1], r[3]}, b0, b1);
            }
        }
    }
};

template <int NS, class Q>
__global__ void __launch_bounds__(32 * kMaxWarps, NS > 4 ? 1 : 2) k_attend_mma(const __grid_constant__ AttendParams a) {
    using M = Mma<NS>;
    extern __shared__ uint8_t sm[];  // the warps' rings, later the vectors to join; then the entries
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int warps = blockDim.x >> 5;
    const Entries list = entries_at(sm + warps * M::RING, warps);
    uint8_t* ring = sm + warp * M::RING;
    // Lanes of one unit: work_of with a lane group of 32 (its own elements are not used).
    const Work w = work_of<32>(a);
    const int e0 = min(w.h0 / a.shared, a.heads / a.shared - 1) * M::HEAD;
    const bool mine = g < w.nr;  // this lane's score rows are a head

    // Queries: head g, dimensions 16 s + 4 c + 0 .. 3.
    uint32_t q[NS][Query<Q>::REGS];
    float kb = 0.0f;
#pragma unroll
    for (int s = 0; s < NS; s++) {
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (mine) load4(a.q, w.i * a.q_stride + (w.h0 + g) * a.q_head_stride + 16 * s + 4 * c, a.dtype, a.q_vec, x);
#pragma unroll
        for (int j = 0; j < 4; j++) kb += x[j];
        Query<Q>::set(x, q[s]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) kb += __shfl_xor_sync(0xffffffffu, kb, o);
    kb *= a.scale * a.k.base;
    float acc[NS][4];  // dimensions x heads 2 c, 2 c + 1
#pragma unroll
    for (int t = 0; t < NS; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[t][j] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // of head g; l of this lane's entries

    const uint8_t *kp = a.k.codes + e0, *vp = a.v.codes + e0;
    const float* ksp = a.k.scales ? a.k.scales + e0 / a.k.group : nullptr;
    const float* vsp = a.v.scales ? a.v.scales + e0 / a.v.group : nullptr;
    auto fetch = [&](int stage, int first, int hi) {
        uint8_t* to = ring + stage * M::STAGE;
#pragma unroll
        for (int k = 0; k < NS; k++) {
            const int x = lane + 32 * k, value = x / (kMmaEntries * NS), y = x % (kMmaEntries * NS);
            const int e = first + y / NS, at = y % NS * 16;
            const bool some = e < hi;
            const uint64_t slot = some ? (uint32_t)list.slot[e] : 0u;
            copy_async<16>(to + value * kMmaEntries * M::ROW + y / NS * M::ROW + at,
                           (value ? vp + slot * a.v.stride : kp + slot * a.k.stride) + at, some);
        }
        const int e = first + (lane & 15);
        const bool some = e < hi, value = lane >= 16;
        const uint64_t slot = some ? (uint32_t)list.slot[e] : 0u;
        const float* from = value ? vsp : ksp;
        if (from) copy_async<4>(to + 2 * kMmaEntries * M::ROW + lane * 4, from + slot * (uint32_t)(value ? a.v.n_groups : a.k.n_groups), some);
        copy_commit();
    };

    // Bytes c for bfloat16, c + 128 for float16.
    const uint32_t k_flip = Query<Q>::BF16_CODES ? a.k.flip ^ 0x80808080u : a.k.flip, v_flip = a.v.flip ^ 0x80808080u;
    const int32_t doc = a.query_docs ? a.query_docs[w.i] : 0;
    const int j0 = (int)min((int64_t)blockIdx.y * a.split_len, (int64_t)a.found);
    const int j1 = (int)min((int64_t)j0 + a.split_len, (int64_t)a.found);
    for (int from = j0; from < j1; from += warps * kRound) {
        int lo, hi;
        slice_of(list_entries(a, list, w.i, doc, from, j1), w.slice, a.slices, kMmaEntries, lo, hi);
        if (w.idle) hi = lo;
        copy_wait<0>();
        __syncwarp();
#pragma unroll
        for (int k = 0; k < M::STAGES - 1; k++) fetch(k, lo + k * kMmaEntries, hi);
        int stage = 0;
        for (int t = lo; t < hi; t += kMmaEntries) {
            copy_wait<M::STAGES - 2>();
            __syncwarp();  // every lane's copies of this stage are there, and its reads of the one before are done
            fetch(stage == 0 ? M::STAGES - 1 : stage - 1, t + (M::STAGES - 1) * kMmaEntries, hi);
            const uint8_t* at = ring + stage * M::STAGE;
            const float* scales = reinterpret_cast<const float*>(at + 2 * kMmaEntries * M::ROW);
            stage = stage + 1 == M::STAGES ? 0 : stage + 1;
            // Scores of entries 8 n + 2 c, + 1 for head g.
            float p[4];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const uint32_t* row = reinterpret_cast<const uint32_t*>(at + (8 * n + g) * M::ROW);
#pragma unroll
                for (int s = 0; s < NS; s++) Query<Q>::dot(d, q[s], row[4 * s + c] ^ k_flip);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int e = 8 * n + 2 * c + j;
                    const float ks = ksp ? scales[e] : a.k.scale, dot = Query<Q>::REGS > 2 ? d[j] + d[2 + j] : d[j];
                    float th;
                    p[2 * n + j] =
                        t + e < hi ? score_of(a, fmaf(dot * a.scale, ks, kb), list.bias[t + e], th) : -INFINITY;
                }
            }
            float top = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)), m);
            const float ref = top == -INFINITY ? 0.0f : top, keep = m == top ? 1.0f : expf(m - ref);
            m = top;
            if (__any_sync(0xffffffffu, keep != 1.0f)) {
                const float s0 = __shfl_sync(0xffffffffu, keep, 8 * c), s1 = __shfl_sync(0xffffffffu, keep, 8 * c + 4);
#pragma unroll
                for (int k = 0; k < NS; k++) acc[k][0] *= s0, acc[k][1] *= s1, acc[k][2] *= s0, acc[k][3] *= s1;
            }
            l *= keep;
            float weight[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                p[j] = expf(p[j] - ref);
                l += p[j];
                weight[j] = p[j] * (vsp ? scales[kMmaEntries + 8 * (j >> 1) + 2 * c + (j & 1)] : a.v.scale);
            }
            uint32_t w0[3], w1[3];
            split3(weight[0], weight[1], w0);
            split3(weight[2], weight[3], w1);
            // Values: word 8 k + g of an entry holds the rows g and g + 8 of two products.
            const uint8_t* values = at + kMmaEntries * M::ROW + 2 * c * M::ROW;
#pragma unroll
            for (int k = 0; k < NS / 2; k++) {
                const int off = (8 * k + g) * 4;
                uint32_t v[4];
#pragma unroll
                for (int j = 0; j < 4; j++)
                    v[j] = *reinterpret_cast<const uint32_t*>(values + ((j >> 1) * 8 + (j & 1)) * M::ROW + off) ^ v_flip;
                const uint32_t x0 = __byte_perm(v[0], v[1], 0x5140), y0 = __byte_perm(v[0], v[1], 0x7362);
                const uint32_t x1 = __byte_perm(v[2], v[3], 0x5140), y1 = __byte_perm(v[2], v[3], 0x7362);
                constexpr uint32_t kLow = 0x7f7f7f7fu, kTop = 0x80808080u;
                const uint32_t first[4] = {bf16_codes(x0 & kLow, x0 & kTop, false), bf16_codes(x0 & kLow, x0 & kTop, true),
                                           bf16_codes(x1 & kLow, x1 & kTop, false), bf16_codes(x1 & kLow, x1 & kTop, true)};
                const uint32_t second[4] = {bf16_codes(y0 & kLow, y0 & kTop, false), bf16_codes(y0 & kLow, y0 & kTop, true),
                                            bf16_codes(y1 & kLow, y1 & kTop, false), bf16_codes(y1 & kLow, y1 & kTop, true)};
#pragma unroll
                for (int j = 2; j >= 0; j--) {  // the small parts first
                    mma16816_bf16(acc[2 * k], first, w0[j], w1[j]);
                    mma16816_bf16(acc[2 * k + 1], second, w0[j], w1[j]);
                }
            }
        }
    }
    copy_wait<0>();
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    // This lane's vectors: heads 2 c and 2 c + 1, dimensions 32 k + 4 g + 0 .. 3.
    float* mine_at = reinterpret_cast<float*>(sm + warp * M::RING);
    float mm[2], ll[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int from = 8 * c + 4 * h;
        mm[h] = __shfl_sync(0xffffffffu, m, from);
        ll[h] = __shfl_sync(0xffffffffu, l, from);
    }
    if (a.slices > 1) {
        __syncthreads();  // the rings have been read
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float* dst = mine_at + (2 * c + h) * (M::HEAD + 2);
#pragma unroll
            for (int k = 0; k < NS; k++) dst[32 * (k / 2) + 4 * g + 2 * (k & 1)] = acc[k][h], dst[32 * (k / 2) + 4 * g + 2 * (k & 1) + 1] = acc[k][2 + h];
            if (g == 0) dst[M::HEAD] = mm[h], dst[M::HEAD + 1] = ll[h];
        }
        __syncthreads();
        if (w.slice == 0) {
            for (int k2 = 1; k2 < a.slices; k2++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float* src = mine_at + k2 * (M::RING / 4) + (2 * c + h) * (M::HEAD + 2);
                    float f, o;
                    mm[h] = join(mm[h], src[M::HEAD], f, o);
                    ll[h] = ll[h] * f + src[M::HEAD + 1] * o;
#pragma unroll
                    for (int k = 0; k < NS; k++) {
                        const int d = 32 * (k / 2) + 4 * g + 2 * (k & 1);
                        acc[k][h] = acc[k][h] * f + src[d] * o;
                        acc[k][2 + h] = acc[k][2 + h] * f + src[d + 1] * o;
                    }
                }
        }
    }
    if (w.slice != 0) return;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (2 * c + h >= w.nr) continue;
        const int64_t at = w.i * a.heads + w.h0 + 2 * c + h, n = a.queries * a.heads, row = (int64_t)blockIdx.y * n + at;
        const float inv = a.part ? 1.0f : ll[h] != 0.0f ? 1.0f / ll[h] : 0.0f, base = a.part || ll[h] == 0.0f ? 0.0f : a.v.base;
#pragma unroll
        for (int k = 0; k < NS / 2; k++) {
            const float4 v = make_float4(fmaf(acc[2 * k][h], inv, base), fmaf(acc[2 * k][2 + h], inv, base),
                                         fmaf(acc[2 * k + 1][h], inv, base), fmaf(acc[2 * k + 1][2 + h], inv, base));
            const int d = 32 * k + 4 * g;
            if (a.part) *reinterpret_cast<float4*>(a.part + row * a.head + d) = v;
            else store4(a.out, at * a.head + d, a.dtype, v);
        }
        if (g != 0) continue;
        if (a.part) reinterpret_cast<float2*>(a.part + a.splits * n * a.head)[row] = make_float2(mm[h], ll[h]);
        else a.lse[at] = ll[h] != 0.0f ? mm[h] + logf(ll[h]) : -INFINITY;
    }
}

// Joins the ranges of a list: a block for each (query, head), 8 elements a
// lane group of 4 warps, each every fourth range; the warps' sums in order.
__global__ void __launch_bounds__(128) k_attend_join(const __grid_constant__ AttendParams a) {
    __shared__ float joined[4][kMaxHead + 1];
    const int64_t n = a.queries * a.heads, at = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d0 = lane * 8;
    const float2* ml = reinterpret_cast<const float2*>(a.part + a.splits * n * a.head);
    float m = -INFINITY;
    for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, ml[s * n + at].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ref = m == -INFINITY ? 0.0f : m;
    float v[8] = {}, l = 0.0f;
#pragma unroll 4
    for (int s = warp; s < a.splits; s += 4) {
        const float2 x = ml[s * n + at];
        const float f = expf(x.x - ref);
        l += x.y * f;
        if (d0 < a.head) {
            const float4* src = reinterpret_cast<const float4*>(a.part + (s * n + at) * a.head + d0);
            const float4 y = src[0], z = src[1];
            v[0] += y.x * f, v[1] += y.y * f, v[2] += y.z * f, v[3] += y.w * f;
            v[4] += z.x * f, v[5] += z.y * f, v[6] += z.z * f, v[7] += z.w * f;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) joined[warp][d0 + j] = v[j];
    if (lane == 0) joined[warp][kMaxHead] = l;
    __syncthreads();
    if (warp != 0) return;
    for (int k = 1; k < 4; k++) {
        l += joined[k][kMaxHead];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] += joined[k][d0 + j];
    }
    if (d0 < a.head) finish_forward(a, at, d0, v, m, l);
}

// A, B, D and the weights' own sum P of the lists' slices; dq = scale (A - (D / P) B) / P.
// P is 1 up to rounding, except where lse cannot hold its own digits beside
// scores of 1e9 and more (a mask of the type's lowest value throughout).
template <int LANES, int RB, bool ALIGNED>
__global__ void __launch_bounds__(32 * kMaxWarpsBack, RB == 1 ? 3 : 2) k_attend_backward(const __grid_constant__ AttendParams a) {
    using St = Steps<LANES, RB>;
    using Sums = typename St::Sums;
    constexpr int STEPS = St::N, RP = St::RP, KEEP = Sums::KEEP;
    constexpr int STAGES = St::STAGES;
    extern __shared__ uint8_t sm[];  // the warps' rings, later the vectors to join; then the entries
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, step = STEPS << a.entries_log;
    const Work w = work_of<LANES>(a);
    const int warps = blockDim.x >> 5;
    const Entries list = entries_at(sm + warps * St::RING, warps);
    const Slot ring{sm + warp * St::RING};
    u64 q[RB][4], g[RB][4], va[RB][4], vb[RB][4];
    float kb[RB], gb[RB];
    load_heads<RB>(a.q, w.i * a.q_stride, a.q_head_stride, a.dtype, w, a.q_vec, a.scale, q, kb);
    load_heads<RB>(a.dout, w.i * a.heads * a.head, a.head, a.dtype, w, a.dout_vec, 1.0f, g, gb);
#pragma unroll
    for (int r = 0; r < RB; r++) {
        kb[r] *= a.k.base;
        gb[r] *= a.v.base;
#pragma unroll
        for (int j = 0; j < 4; j++) va[r][j] = vb[r][j] = 0;
    }
    float z[KEEP], dsum[KEEP], psum[KEEP];  // of the lane's own values' heads
#pragma unroll
    for (int x = 0; x < KEEP; x++) {
        const int r = Sums::value_of(x) % RP;
        z[x] = r < w.nr ? a.lse_in[w.i * a.heads + w.h0 + r] : 0.0f;
        dsum[x] = psum[x] = 0.0f;
    }
    const Places places = places_of(a, w);
    const int32_t doc = a.query_docs ? a.query_docs[w.i] : 0;
    const u64 kbase = pair(a.k.base, a.k.base);
    const int j0 = (int)min((int64_t)blockIdx.y * a.split_len, (int64_t)a.found);
    const int j1 = (int)min((int64_t)j0 + a.split_len, (int64_t)a.found);
    for (int from = j0; from < j1; from += (blockDim.x >> 5) * kRound) {
        int lo, hi;
        slice_of(list_entries(a, list, w.i, doc, from, j1), w.slice, a.slices, step, lo, hi);
        if (w.idle) hi = lo;
        copy_wait<0>();  // the previous range's last (empty) stages
#pragma unroll
        for (int k = 0; k < STAGES - 1; k++)
            fetch<ALIGNED, STEPS>({ring.at + k * STEPS * 768}, places, list.slot, lo + k * step + w.entry, a.entries_log,
                                  hi, w.live);
        int stage = 0, ahead = STAGES - 1;
        for (int t = lo; t < hi; t += step) {
            copy_wait<STAGES - 2>();
            const Slot now{ring.at + stage * STEPS * 768};
            fetch<ALIGNED, STEPS>({ring.at + ahead * STEPS * 768}, places, list.slot,
                                  t + (STAGES - 1) * step + w.entry, a.entries_log, hi, w.live);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            ahead = ahead + 1 == STAGES ? 0 : ahead + 1;
            Taken<STEPS> key, value;
            key.take(now, 0, places.ks, places.k_scale);
            value.take(now, 1, places.vs, places.v_scale);
            float s[STEPS * RP], dp[STEPS * RP];
#pragma unroll
            for (int u = 0; u < STEPS; u++) {
                u64 c[4];
                code_pairs(key.codes[u], a.k.flip, c);
#pragma unroll
                for (int r = 0; r < RP; r++) s[u * RP + r] = r < RB ? fmaf(key.scale[u], dot_pairs(q[r < RB ? r : 0], c), kb[r < RB ? r : 0]) : 0.0f;
                code_pairs(value.codes[u], a.v.flip, c);
#pragma unroll
                for (int r = 0; r < RP; r++) dp[u * RP + r] = r < RB ? fmaf(value.scale[u], dot_pairs(g[r < RB ? r : 0], c), gb[r < RB ? r : 0]) : 0.0f;
            }
            Sums::sum(s);
            Sums::sum(dp);
            float fa[KEEP], fb[KEEP];
#pragma unroll
            for (int x = 0; x < KEEP; x++) {
                const int v = Sums::value_of(x), r = v % RP, e = t + (v / RP << a.entries_log) + w.entry;
                fa[x] = fb[x] = 0.0f;
                if (e < hi && r < w.nr) {
                    float th;
                    const float sc = score_of(a, s[x], list.bias[e], th);
                    const float p = expf(sc - z[x]), pdp = p * dp[x], slope = 1.0f - th * th;
                    dsum[x] += pdp;
                    psum[x] += p;
                    fa[x] = pdp * slope;
                    fb[x] = p * slope;
                    if (a.pd && lane % Sums::DUP == 0)
                        a.pd[(w.i * a.heads + w.h0 + r) * a.found + list.place[e]] = make_float2(pdp, p);
                }
            }
#pragma unroll
            for (int u = 0; u < STEPS; u++) {
                u64 c[4];
                code_pairs(key.codes[u], a.k.flip, c);
                const u64 kss = pair(key.scale[u], key.scale[u]);
#pragma unroll
                for (int j = 0; j < 4; j++) c[j] = fma2(kss, c[j], kbase);  // the key's values
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const float xa = Sums::get(fa, u * RP + r), xb = Sums::get(fb, u * RP + r);
                    const u64 pa = pair(xa, xa), pb = pair(xb, xb);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        va[r][j] = fma2(pa, c[j], va[r][j]);
                        vb[r][j] = fma2(pb, c[j], vb[r][j]);
                    }
                }
            }
        }
    }
    copy_wait<0>();
#pragma unroll
    for (int x = 0; x < KEEP; x++)
        St::over_entries(a.entries_log, [&](int o) {
            dsum[x] += __shfl_xor_sync(0xffffffffu, dsum[x], o);
            psum[x] += __shfl_xor_sync(0xffffffffu, psum[x], o);
        });
#pragma unroll
    for (int r = 0; r < RB; r++) {
        float x[8], y[8], sd = Sums::get(dsum, r), sp = Sums::get(psum, r);
        join_vectors<LANES>(va[r], a.entries_log, x);
        join_vectors<LANES>(vb[r], a.entries_log, y);
        if (a.slices > 1) {
            __syncthreads();  // the rings, or the previous head's vectors, have been read
            float* mine = reinterpret_cast<float*>(sm) + warp * 576;
            put8(mine + lane * 8, x);
            put8(mine + 256 + lane * 8, y);
            reinterpret_cast<float2*>(mine + 512)[lane] = make_float2(sd, sp);
            __syncthreads();
            if (w.slice == 0) {
                for (int k = 1; k < a.slices; k++) {
                    const float* src = mine + k * 576;
                    const float2 dp = reinterpret_cast<const float2*>(src + 512)[lane];
                    float o[8], h[8];
                    get8(src + lane * 8, o);
                    get8(src + 256 + lane * 8, h);
                    sd += dp.x;
                    sp += dp.y;
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] += o[j], y[j] += h[j];
                }
            }
        }
        if (r >= w.nr || w.slice != 0 || !w.live || w.entry != 0) continue;
        const int64_t at = w.i * a.heads + w.h0 + r, n = a.queries * a.heads, row = (int64_t)blockIdx.y * n + at;
        if (a.part) {
            put8(a.part + row * 2 * a.head + w.d0, x);
            put8(a.part + (row * 2 + 1) * a.head + w.d0, y);
            if (w.d0 == 0) reinterpret_cast<float2*>(a.part + a.splits * n * 2 * a.head)[row] = make_float2(sd, sp);
        } else {
            finish_backward(a, at, w.d0, x, y, sd, sp);
        }
    }
}

// Joins the ranges of a list, as k_attend_join: plain sums.
__global__ void __launch_bounds__(128) k_attend_backward_join(const __grid_constant__ AttendParams a) {
    __shared__ float joined[4][2 * kMaxHead + 2];
    const int64_t n = a.queries * a.heads, at = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d0 = lane * 8;
    const float2* dp = reinterpret_cast<const float2*>(a.part + a.splits * n * 2 * a.head);
    float x[8] = {}, y[8] = {}, d = 0.0f, p = 0.0f;
#pragma unroll 4
    for (int s = warp; s < a.splits; s += 4) {
        const float2 f = dp[s * n + at];
        d += f.x;
        p += f.y;
        if (d0 < a.head) {
            const float* src = a.part + (s * n + at) * 2 * a.head + d0;
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] += src[j], y[j] += src[a.head + j];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) joined[warp][d0 + j] = x[j], joined[warp][kMaxHead + d0 + j] = y[j];
    if (lane == 0) joined[warp][2 * kMaxHead] = d, joined[warp][2 * kMaxHead + 1] = p;
    __syncthreads();
    if (warp != 0) return;
    for (int k = 1; k < 4; k++) {
        d += joined[k][2 * kMaxHead];
        p += joined[k][2 * kMaxHead + 1];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] += joined[k][d0 + j], y[j] += joined[k][kMaxHead + d0 + j];
    }
    if (d0 < a.head) finish_backward(a, at, d0, x, y, d, p);
}

// dbias[i][j] = sum over heads of (p dP - p (D / P - dlse)) / P, in head order; 0 at hidden entries.
__global__ void __launch_bounds__(256) k_attend_dbias(const __grid_constant__ AttendParams a, float* __restrict__ dbias) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= a.queries * a.found) return;
    const int64_t i = at / a.found;
    const int j = (int)(at - i * a.found);
    float v = 0.0f, bias;
    if (entry_slot(a, i, j, a.query_docs ? a.query_docs[i] : 0, bias) >= 0) {
#pragma unroll 4
        for (int h = 0; h < a.heads; h++) {
            const float2 x = __ldg(a.pd + (i * a.heads + h) * a.found + j), d = __ldg(a.sum_d + i * a.heads + h);
            v += (x.x - x.y * d.x) * d.y;
        }
    }
    dbias[at] = v;
}

CodeView code_view(const RowsView& r) {
    CodeView c{};
    c.codes = r.codes;
    c.scales = r.affine ? nullptr : r.scales;
    MDH_REQUIRE(r.stride <= INT32_MAX, MDH_ERR_UNSUPPORTED, "attend: the caches' row stride is limited to 2^31 - 1 bytes");
    c.stride = (uint32_t)r.stride;
    c.group = r.group;
    c.n_groups = r.n_groups;
    c.flip = r.affine ? 0u : 0x80808080u;
    c.scale = r.step;
    c.base = r.affine ? r.lo + 128.0f * r.step : 0.0f;
    return c;
}

// Lanes that hold a head; rows off 8 bytes take the widest form alone, the
// matrix form a warp.
int lanes_of(const AttendParams& p) {
    int lanes = 1;
    while (lanes * 8 < p.head) lanes *= 2;
    return p.form == kFormLanes ? lanes : 32;
}

// How a call is laid out over warps and blocks.  Units side by side in a warp
// need no join, so lane groups take entries of one unit only where fewer than
// kEnough warps would have work (2,048 queries x 4 units: 48 us with four
// units side by side, 58 us with two and twice the warps); then several warps
// of a block share units' lists, and then blocks take ranges of a list, up to
// kFill warps; no slice is below kMinSlice entries.
void lay_out(AttendParams& p, int max_warps) {
    // The matrix form of heads past 64 has room for 8 warps an SM.
    const int64_t kEnough = 148 * 8, kFill = p.form == kFormMma && p.head > 64 ? 148 * 8 : 148 * 16;
    p.r_blocks = (int)ceil_div(p.shared, p.form == kFormMma ? kMaxSharedMma : kMaxShared);
    p.rb = (int)ceil_div(p.shared, p.r_blocks);
    p.units = p.heads / p.shared * p.r_blocks;
    int side = 32 / lanes_of(p);
    p.entries_log = 0;
    while (side > 1 && (side / 2 >= p.units || p.queries * ceil_div(p.units, side) < kEnough))
        side /= 2, p.entries_log++;
    const int64_t unit_warps = ceil_div(p.units, side);
    p.unit_blocks = (int)ceil_div(unit_warps, max_warps);
    p.block_warps = (int)ceil_div(unit_warps, p.unit_blocks);
    const int64_t warps = std::max<int64_t>(1, p.queries * p.unit_blocks * p.block_warps);
    p.slices = (int)std::max<int64_t>(
        1, std::min({(int64_t)max_warps / p.block_warps, ceil_div(p.found, kMinSlice), kFill / warps}));
    const int64_t splits = std::min(ceil_div(p.found, p.slices * kMinSlice), kFill / (warps * p.slices));
    p.split_len = (int)std::max<int64_t>(1, ceil_div(p.found, std::max<int64_t>(1, splits)));
    p.splits = (int)std::max<int64_t>(1, ceil_div(p.found, p.split_len));
}

AttendParams check_attend(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values, bool forward) {
    MDH_REQUIRE(a, MDH_ERR_INVALID_ARG, "attend: null arguments");
    AttendParams p{};
    const RowsView k = rows_view(keys), v = rows_view(values);
    MDH_REQUIRE(dtype_ok(a->dtype), MDH_ERR_INVALID_ARG, "attend: dtype must be float32, bfloat16 or float16");
    MDH_REQUIRE(a->queries >= 0 && a->found >= 0, MDH_ERR_INVALID_ARG, "attend: queries and found must be >= 0");
    // Places in a list are 32 bits and run past its end by what a block looks at.
    MDH_REQUIRE(a->found <= INT32_MAX - kMaxWarps * kRound, MDH_ERR_UNSUPPORTED, "attend: found is limited to 2^31 - 1025");
    MDH_REQUIRE(a->heads >= 1 && a->shared >= 1 && a->heads % a->shared == 0, MDH_ERR_INVALID_ARG,
                "attend: heads must be a positive multiple of shared");
    MDH_REQUIRE(a->head >= 8 && a->head % 8 == 0 && a->head <= kMaxHead, MDH_ERR_UNSUPPORTED,
                "attend: the head size must be a multiple of 8 up to 256");
    MDH_REQUIRE(k.slots == v.slots, MDH_ERR_INVALID_ARG, "attend: key and value caches differ in slots");
    const int64_t width = (int64_t)(a->heads / a->shared) * a->head;
    MDH_REQUIRE(k.width == width && v.width == width, MDH_ERR_INVALID_ARG,
                "attend: cache rows must hold heads / shared heads");
    MDH_REQUIRE((a->query_docs == nullptr) == (a->row_docs == nullptr), MDH_ERR_INVALID_ARG,
                "attend: query_docs and row_docs go together");
    MDH_REQUIRE(std::isfinite(a->scale), MDH_ERR_INVALID_ARG, "attend: scale must be finite");
    MDH_REQUIRE(a->cap >= 0.0f && std::isfinite(a->cap), MDH_ERR_INVALID_ARG, "attend: cap must be finite and >= 0");
    MDH_REQUIRE(a->queries == 0 || a->q, MDH_ERR_INVALID_ARG, "attend: null queries");
    MDH_REQUIRE(a->queries == 0 || a->found == 0 || a->ids, MDH_ERR_INVALID_ARG, "attend: null ids");
    auto lists = [&](int64_t stride) { return a->queries <= 1 || stride >= a->found || stride == 0; };
    MDH_REQUIRE(lists(a->ids_stride) && (!a->bias || lists(a->bias_stride)), MDH_ERR_INVALID_ARG,
                "attend: list stride below its length (0: one list for every query)");
    p.k = code_view(k);
    p.v = code_view(v);
    // The matrix form takes heads of 32 .. 128 that start on 16 bytes and have one scale each.  Its time hardly
    // depends on how many heads share a row (256 queries x 1,000 x 4 heads of 64, shared by 2, 3, 4, 8: 58 us in
    // float16, 62 in bfloat16, 66 in float32; by lanes 81, 96, 112 and 206).  Short lists of many queries are bound by what comes before and after the entries, which the
    // lanes do for several units at once (2,048 queries x 64 entries, shared by 2, 3, 4, 8: 43 us against 34, 46, 54
    // and 99); a head of its own gains nothing.
    auto one_scale = [&](const RowsView& c) { return c.affine || c.n_groups == 1 || c.group % a->head == 0; };
    auto on_16 = [](const RowsView& c) { return aligned16(c.codes) && c.stride % 16 == 0; };
    const bool pays = a->shared >= 4 || a->found >= 128 || a->queries * (a->heads / a->shared) < 148 * 8;
    const bool matrix = forward && a->shared >= 2 && pays && a->head % 32 == 0 && a->head <= 128 && one_scale(k) && one_scale(v) &&
                        on_16(k) && on_16(v);
    p.form = matrix ? kFormMma : rows_on_8(k) && rows_on_8(v) ? kFormLanes : kFormBytes;
    const size_t size = dtype_size(a->dtype);
    p.q_vec = rows_aligned(a->q, a->q_stride, size) && rows_aligned(a->q, a->q_head_stride, size) &&
              a->head * size % 16 == 0;
    p.q = a->q;
    p.ids = a->ids;
    p.bias = a->bias;
    p.query_docs = a->query_docs;
    p.row_docs = a->row_docs;
    p.q_stride = a->q_stride;
    p.q_head_stride = a->q_head_stride;
    p.ids_stride = a->ids_stride;
    p.bias_stride = a->bias_stride;
    p.slots = k.slots;
    p.queries = a->queries;
    p.found = a->found;
    p.heads = a->heads;
    p.shared = a->shared;
    p.head = a->head;
    p.dtype = a->dtype;
    p.scale = a->scale;
    p.cap = a->cap;
    p.inv_cap = a->cap > 0.0f ? 1.0f / a->cap : 0.0f;
    lay_out(p, forward ? kMaxWarps : kMaxWarpsBack);
    MDH_REQUIRE(p.queries * p.unit_blocks <= INT32_MAX && p.queries * p.heads <= INT32_MAX, MDH_ERR_UNSUPPORTED, "attend: too many queries");
    return p;
}

// The layout of a call from its sizes alone, for the workspace.
AttendParams layout_of(const mdh_attend_args* a, int form, int max_warps) {
    AttendParams p{};
    p.queries = a->queries;
    p.found = a->found;
    p.heads = a->heads;
    p.shared = a->shared;
    p.head = a->head;
    p.form = form;
    lay_out(p, max_warps);
    return p;
}
bool has_sizes(const mdh_attend_args* a) {
    return a && a->queries > 0 && a->found >= 0 && a->heads > 0 && a->shared > 0 && a->heads % a->shared == 0 &&
           a->head > 0 && a->head <= kMaxHead;
}
int64_t forward_part(const AttendParams& p) {
    return p.splits > 1 ? p.splits * p.queries * p.heads * ((int64_t)p.head + 2) * 4 : 0;
}
int64_t backward_part(const AttendParams& p) {
    return p.splits > 1 ? round_up(p.splits * p.queries * p.heads * (2 * (int64_t)p.head + 2) * 4, 16) : 0;
}

// fn(LANES, RB, ALIGNED): lanes that hold a head, query heads of a unit.  Rows
// off 8 bytes are read byte by byte, by the widest form alone.
template <class F>
void by_shape(const AttendParams& p, F&& fn) {
    using std::integral_constant;
    if (p.form == kFormBytes) return fn(integral_constant<int, 32>{}, integral_constant<int, 4>{}, std::false_type{});
    auto heads = [&](auto lanes) {
        if (p.rb == 1) fn(lanes, integral_constant<int, 1>{}, std::true_type{});
        else if (p.rb == 2) fn(lanes, integral_constant<int, 2>{}, std::true_type{});
        else if (p.rb == 3) fn(lanes, integral_constant<int, 3>{}, std::true_type{});
        else fn(lanes, integral_constant<int, 4>{}, std::true_type{});
    };
    switch (lanes_of(p)) {
        case 1: heads(integral_constant<int, 1>{}); break;
        case 2: heads(integral_constant<int, 2>{}); break;
        case 4: heads(integral_constant<int, 4>{}); break;
        case 8: heads(integral_constant<int, 8>{}); break;
        case 16: heads(integral_constant<int, 16>{}); break;
        default: heads(integral_constant<int, 32>{}); break;
    }
}
dim3 attend_grid(const AttendParams& p) {
    return dim3((unsigned)(p.queries * p.unit_blocks), (unsigned)p.splits);
}
// Launches KERNEL with `WARP_BYTES` of shared memory for each of its warps.
template <auto KERNEL, int WARP_BYTES, int MAX_WARPS>
void launch_warps(const AttendParams& p, cudaStream_t st) {
    static std::atomic<uint64_t> set{0};  // a bit a device
    const int dev = current_device(), warps = p.block_warps * p.slices;
    if (!(set.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
        MDH_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_WARPS * WARP_BYTES));
        set.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_relaxed);
    }
    KERNEL<<<attend_grid(p), 32 * warps, warps * WARP_BYTES, st>>>(p);
    check_launch();
}
template <int LANES, int RB, bool ALIGNED, bool BACKWARD>
void launch_lanes(const AttendParams& p, cudaStream_t st) {
    constexpr int kWarpBytes = Steps<LANES, RB>::RING + kEntriesBytes;
    if constexpr (BACKWARD) launch_warps<k_attend_backward<LANES, RB, ALIGNED>, kWarpBytes, kMaxWarpsBack>(p, st);
    else launch_warps<k_attend<LANES, RB, ALIGNED>, kWarpBytes, kMaxWarps>(p, st);
}
void launch_mma(const AttendParams& p, cudaStream_t st) {
    by_dtype(p.dtype, [&](auto zero) {
        using Q = decltype(zero);
        switch (p.head) {
            case 32: launch_warps<k_attend_mma<2, Q>, Mma<2>::RING + kEntriesBytes, kMaxWarps>(p, st); break;
            case 64: launch_warps<k_attend_mma<4, Q>, Mma<4>::RING + kEntriesBytes, kMaxWarps>(p, st); break;
            case 96: launch_warps<k_attend_mma<6, Q>, Mma<6>::RING + kEntriesBytes, kMaxWarps>(p, st); break;
            default: launch_warps<k_attend_mma<8, Q>, Mma<8>::RING + kEntriesBytes, kMaxWarps>(p, st); break;
        }
    });
}

}  // namespace
}  // namespace mdh

using namespace mdh;

extern "C" {

int64_t mdh_attend_workspace(const mdh_attend_args* a) {
    if (!has_sizes(a)) return 0;
    return std::max({forward_part(layout_of(a, kFormBytes, kMaxWarps)), forward_part(layout_of(a, kFormLanes, kMaxWarps)),
                     forward_part(layout_of(a, kFormMma, kMaxWarps))});
}

mdh_status mdh_attend(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values, void* out, float* lse,
                      void* ws, int64_t ws_bytes, void* stream) {
    return guarded([&] {
        AttendParams p = check_attend(a, keys, values, true);
        current_device();
        if (p.queries == 0) return;
        MDH_REQUIRE(out && lse && aligned16(out), MDH_ERR_INVALID_ARG, "attend: output null or not 16-byte aligned");
        const int64_t need = mdh_attend_workspace(a);
        MDH_REQUIRE(need == 0 || (ws && aligned16(ws) && ws_bytes >= need), MDH_ERR_INVALID_ARG,
                    "attend: workspace too small or not 16-byte aligned");
        const cudaStream_t st = (cudaStream_t)stream;
        p.out = out;
        p.lse = lse;
        p.part = p.splits > 1 ? (float*)ws : nullptr;
        if (p.form == kFormMma) launch_mma(p, st);
        else by_shape(p, [&](auto lanes, auto rb, auto aligned) { launch_lanes<lanes, rb, aligned, false>(p, st); });
        if (p.splits > 1) {
            k_attend_join<<<(unsigned)(p.queries * p.heads), 128, 0, st>>>(p);
            check_launch();
        }
    });
}

int64_t mdh_attend_backward_workspace(const mdh_attend_args* a, int32_t want_dbias) {
    if (!has_sizes(a)) return 0;
    int64_t need = std::max(backward_part(layout_of(a, kFormBytes, kMaxWarpsBack)),
                            backward_part(layout_of(a, kFormLanes, kMaxWarpsBack)));
    if (want_dbias) need += a->queries * a->heads * 8 + a->queries * a->heads * (int64_t)a->found * 8;
    return need;
}

mdh_status mdh_attend_backward(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values,
                               const void* dout, const float* lse, void* dq, float* dbias, void* ws, int64_t ws_bytes,
                               void* stream) {
    return mdh_attend_backward_lse(a, keys, values, dout, lse, nullptr, dq, dbias, ws, ws_bytes, stream);
}

mdh_status mdh_attend_backward_lse(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values,
                                   const void* dout, const float* lse, const float* dlse, void* dq, float* dbias,
                                   void* ws, int64_t ws_bytes, void* stream) {
    return guarded([&] {
        AttendParams p = check_attend(a, keys, values, false);
        current_device();
        if (p.queries == 0) return;
        MDH_REQUIRE(dout && lse && dq && aligned16(dq), MDH_ERR_INVALID_ARG,
                    "attend: null dout, lse or dq, or dq not 16-byte aligned");
        const int64_t need = mdh_attend_backward_workspace(a, dbias != nullptr);
        MDH_REQUIRE(need == 0 || (ws && aligned16(ws) && ws_bytes >= need), MDH_ERR_INVALID_ARG,
                    "attend: workspace too small or not 16-byte aligned");
        const cudaStream_t st = (cudaStream_t)stream;
        const int64_t bias_blocks = ceil_div(p.queries * p.found, 256);
        MDH_REQUIRE(bias_blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "attend: too many queries");
        char* at = (char*)ws;
        if (p.splits > 1) p.part = (float*)at;
        at += backward_part(p);
        if (dbias) {
            p.sum_d = (float2*)at;
            p.pd = p.sum_d + p.queries * p.heads;
        }
        p.out = dq;
        p.dout = dout;
        p.dout_vec = aligned16(dout) && a->head * dtype_size(a->dtype) % 16 == 0;
        p.lse_in = lse;
        p.dlse = dlse;
        by_shape(p, [&](auto lanes, auto rb, auto aligned) {
            launch_lanes<lanes, rb, aligned, true>(p, st);
        });
        if (p.splits > 1) {
            k_attend_backward_join<<<(unsigned)(p.queries * p.heads), 128, 0, st>>>(p);
            check_launch();
        }
        if (dbias && p.found) {
            k_attend_dbias<<<(unsigned)bias_blocks, 256, 0, st>>>(p, dbias);
            check_launch();
        }
    });
}

}  // extern "C"
