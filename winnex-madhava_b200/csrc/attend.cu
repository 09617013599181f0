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
// one pass over the rows as well, since p_j follows from lse.
//
// Bound by memory: a key and a value code are read once and meet one multiply
// each for every head that shares them.  A warp takes one (query, group of
// heads that share a row's head, slice of the list).  LANES lanes hold one
// entry, 8 elements each (an 8-byte load of codes); 32 / LANES entries go side
// by side and STEPS of them are loaded before the first is used.  Each lane
// group keeps its own maximum, sum and vector, joined at the end: first
// inside the warp, then over the block's slices in shared memory, then over
// blocks by a second kernel where a list is cut across blocks.
//
// Codes become floats without a conversion instruction: the byte c + 128 in
// the mantissa of 2^23 is the float 8388736 + c, and one subtraction (two
// values at a time) leaves c exactly.  The row's scale multiplies the finished
// 8-term sums; the affine code's offset enters as a constant times the sum of
// the query's elements, or of the weights.
#include <algorithm>

#include "op_rows.cuh"

namespace mdh {
namespace {

using namespace op;

constexpr int kWarps = 8;             // of a block
constexpr int kMaxHead = 256;
constexpr int kMaxShared = 4;         // query heads a warp takes at a time
constexpr int kMinSlice = 16;         // entries below which a list is not cut further

struct CodeView {
    const uint8_t* codes;
    const float* scales;  // null: affine
    int64_t stride;
    int group, n_groups;
    uint32_t flip;        // 0x80808080 for int8: the stored byte becomes c + 128
    float scale, base;    // affine: value = base + scale c
    bool vec;             // 8-byte loads of codes are aligned
};

struct AttendParams {
    CodeView k, v;
    const void* q;
    const int32_t* ids;
    const float* bias;
    const int32_t *query_docs, *row_docs;
    int64_t q_stride, q_head_stride, ids_stride, bias_stride, slots;
    int64_t queries;
    int found, heads, shared, head, dtype;
    float scale, cap, inv_cap;
    int r_blocks;          // blocks of kMaxShared heads of a group
    int units;             // (group, block of heads) pairs of a query
    int slices;            // of a list, over the warps of a block
    int splits;            // of a list, over blocks
    int slice_len;         // entries of a slice
    void* out;
    float* lse;
    float* part;           // splits > 1
    // backward
    const void* dout;
    const float* lse_in;
    float2* pd;            // [queries][heads][found] p dP and p, or null
    float2* sum_d;         // [queries][heads] D / P and 1 / P, or null
};

using u64 = unsigned long long;
__device__ __forceinline__ u64 pair(float a, float b) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(u64 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
    u64 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
    u64 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
    u64 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
constexpr float kLog2e = 1.44269504088896341f;
// e^x for x <= 0, by the hardware's 2^x (relative error about 2^-22).
__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * kLog2e); }
// tanh x = 1 - 2 / (e^2x + 1): absolute error below 2^-21, what a capped score needs.
__device__ __forceinline__ float tanh_fast(float x) {
    return 1.0f - __fdividef(2.0f, exp2_fast(fminf(x * (2.0f * kLog2e), 126.0f)) + 1.0f);
}

// 8 codes of a row.
__device__ __forceinline__ uint2 load_codes(const CodeView& c, int64_t slot, int e) {
    const uint8_t* p = c.codes + slot * c.stride + e;
    if (c.vec) return __ldg(reinterpret_cast<const uint2*>(p));
    uint2 r = make_uint2(0, 0);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        r.x |= (uint32_t)p[j] << (8 * j);
        r.y |= (uint32_t)p[4 + j] << (8 * j);
    }
    return r;
}
__device__ __forceinline__ float load_scale(const CodeView& c, int64_t slot, int group) {
    return c.scales ? __ldg(c.scales + slot * c.n_groups + group) : c.scale;
}
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

// 8 elements of q's type at p + i.
__device__ __forceinline__ void load_elements(const void* p, int64_t i, int dtype, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++)
        v[j] = dtype == MDH_F32    ? static_cast<const float*>(p)[i + j]
               : dtype == MDH_BF16 ? to_f32(static_cast<const bf16*>(p)[i + j])
                                   : to_f32(static_cast<const f16*>(p)[i + j]);
}
__device__ __forceinline__ void store_elements(void* p, int64_t i, int dtype, const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (dtype == MDH_F32) static_cast<float*>(p)[i + j] = v[j];
        else if (dtype == MDH_BF16) static_cast<bf16*>(p)[i + j] = from_f32<bf16>(v[j]);
        else static_cast<f16*>(p)[i + j] = from_f32<f16>(v[j]);
    }
}

// What a warp works on.
struct Work {
    int64_t i;       // query
    int h0, nr;      // first head, heads
    int e0;          // this lane's first element of a row
    int d0;          // ... of a head
    bool live;       // the lane holds elements (a head may end inside the lane group)
    int j0, j1;      // entries
    int slice;       // within the block
};
template <int LANES, int RB>
__device__ __forceinline__ bool work_of(const AttendParams& a, Work& w) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * (kWarps / a.slices) + warp / a.slices;
    w.i = at / a.units;
    w.slice = warp % a.slices;
    if (w.i >= a.queries) return false;
    const int unit = (int)(at - w.i * a.units);
    const int g = unit / a.r_blocks, rb = unit - g * a.r_blocks;
    w.h0 = g * a.shared + rb * RB;
    w.nr = min(RB, a.shared - rb * RB);
    w.d0 = (lane % LANES) * 8;
    w.live = w.d0 < a.head;
    w.e0 = g * a.head + (w.live ? w.d0 : 0);
    const int64_t s = (int64_t)(blockIdx.y * a.slices + w.slice) * a.slice_len;
    w.j0 = (int)min(s, (int64_t)a.found);
    w.j1 = (int)min(s + a.slice_len, (int64_t)a.found);
    return true;
}

// Entry j of the list: its slot, or -1 when it is hidden; its bias.
__device__ __forceinline__ int entry_slot(const AttendParams& a, int64_t i, int j, int32_t doc, float& bias) {
    const int id = __ldg(a.ids + i * a.ids_stride + j);
    bias = 0.0f;
    if (id < 0 || id >= a.slots) return -1;
    if (a.bias) {
        bias = __ldg(a.bias + i * a.bias_stride + j);
        if (bias == -INFINITY) return -1;
    }
    if (a.row_docs && __ldg(a.row_docs + id) != doc) return -1;
    return id;
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Joins two running softmaxes (m, l, vector scaled alike): the factors for
// each side.
__device__ __forceinline__ float join(float m, float mo, float& mine, float& other) {
    const float top = fmaxf(m, mo), ref = top == -INFINITY ? 0.0f : top;
    mine = exp_fast(m - ref);
    other = exp_fast(mo - ref);
    return top;
}

template <int LANES, int RB>
__global__ void __launch_bounds__(32 * kWarps) k_attend(const __grid_constant__ AttendParams a) {
    constexpr int ENTRIES = 32 / LANES;               // side by side
    constexpr int STEPS = RB == 4 ? 2 : 4;            // loaded at a time
    constexpr int ROW = LANES * 8 + 2;                // vector, m, l
    __shared__ float joined[kWarps][ROW];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LANES;
    Work w;
    const bool some = work_of<LANES, RB>(a, w);
    if (!some) w.nr = 0;
    u64 q[RB][4], acc[RB][4];
    float m[RB], l[RB], kb[RB];
    if (some) {
#pragma unroll
        for (int r = 0; r < RB; r++) {
            float v[8] = {};
            if (w.live && r < w.nr) load_elements(a.q, w.i * a.q_stride + (w.h0 + r) * a.q_head_stride + w.d0, a.dtype, v);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) sum += v[j] *= a.scale;
#pragma unroll
            for (int j = 0; j < 4; j++) q[r][j] = pair(v[2 * j], v[2 * j + 1]), acc[r][j] = 0;
            kb[r] = a.k.base * sum;
            m[r] = -INFINITY;
            l[r] = 0.0f;
        }
        const int kg = w.e0 / a.k.group, vg = w.e0 / a.v.group;
        const int32_t doc = a.query_docs ? a.query_docs[w.i] : 0;
        for (int j0 = w.j0; j0 < w.j1; j0 += 32) {
            float my_bias = 0.0f;
            const int my_slot = j0 + lane < w.j1 ? entry_slot(a, w.i, j0 + lane, doc, my_bias) : -1;
            const int n = min(32, w.j1 - j0);
            for (int t = 0; t < n; t += STEPS * ENTRIES) {
                uint2 kraw[STEPS], vraw[STEPS];
                float ks[STEPS], vs[STEPS], bias[STEPS];
                bool seen[STEPS];
#pragma unroll
                for (int u = 0; u < STEPS; u++) {
                    const int e = t + u * ENTRIES + sub;  // past the list: lane e & 31 holds -1 or e wraps
                    const int slot = __shfl_sync(0xffffffffu, my_slot, e & 31);
                    bias[u] = __shfl_sync(0xffffffffu, my_bias, e & 31);
                    seen[u] = e < n && slot >= 0;
                    kraw[u] = vraw[u] = make_uint2(0, 0);
                    ks[u] = vs[u] = 0.0f;
                    if (seen[u] && w.live) {
                        kraw[u] = load_codes(a.k, slot, w.e0);
                        vraw[u] = load_codes(a.v, slot, w.e0);
                        ks[u] = load_scale(a.k, slot, kg);
                        vs[u] = load_scale(a.v, slot, vg);
                    }
                }
                float s[STEPS][RB];
#pragma unroll
                for (int u = 0; u < STEPS; u++) {
                    u64 c[4];
                    code_pairs(kraw[u], a.k.flip, c);
#pragma unroll
                    for (int r = 0; r < RB; r++) {
                        if (r >= w.nr) continue;
                        float x = group_sum<LANES>(fmaf(ks[u], dot_pairs(q[r], c), kb[r]));
                        if (a.cap > 0.0f) x = a.cap * tanh_fast(x * a.inv_cap);
                        s[u][r] = seen[u] ? x + bias[u] : -INFINITY;
                    }
                }
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    if (r >= w.nr) continue;
                    float top = m[r];
#pragma unroll
                    for (int u = 0; u < STEPS; u++) top = fmaxf(top, s[u][r]);
                    const float ref = top == -INFINITY ? 0.0f : top, keep = exp_fast(m[r] - ref);
                    m[r] = top;
                    l[r] *= keep;
                    const u64 kk = pair(keep, keep);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[r][j] = mul2(acc[r][j], kk);
#pragma unroll
                    for (int u = 0; u < STEPS; u++) {
                        s[u][r] = exp_fast(s[u][r] - ref);  // now the weight
                        l[r] += s[u][r];
                    }
                }
#pragma unroll
                for (int u = 0; u < STEPS; u++) {
                    u64 c[4];
                    code_pairs(vraw[u], a.v.flip, c);
#pragma unroll
                    for (int r = 0; r < RB; r++) {
                        if (r >= w.nr) continue;
                        const float p = s[u][r] * vs[u];
                        const u64 pp = pair(p, p);
#pragma unroll
                        for (int j = 0; j < 4; j++) acc[r][j] = fma2(pp, c[j], acc[r][j]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < RB; r++) {
        // The lane groups of the warp, then the block's slices.
        if (r < w.nr) {
#pragma unroll
            for (int o = LANES; o < 32; o <<= 1) {
                const float mo = __shfl_xor_sync(0xffffffffu, m[r], o), lo = __shfl_xor_sync(0xffffffffu, l[r], o);
                float mine, other;
                m[r] = join(m[r], mo, mine, other);
                l[r] = l[r] * mine + lo * other;
                const u64 mm = pair(mine, mine), oo = pair(other, other);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const u64 x = __shfl_xor_sync(0xffffffffu, acc[r][j], o);
                    acc[r][j] = fma2(acc[r][j], mm, mul2(x, oo));
                }
            }
            if (a.slices > 1 && lane < LANES) {
                float* dst = joined[warp];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = unpair(acc[r][j]);
                    dst[w.d0 + 2 * j] = f.x;
                    dst[w.d0 + 2 * j + 1] = f.y;
                }
                if (lane == 0) dst[LANES * 8] = m[r], dst[LANES * 8 + 1] = l[r];
            }
        }
        if (a.slices > 1) __syncthreads();
        if (r < w.nr && w.slice == 0 && lane < LANES && w.live) {
            float v[8], mm = m[r], ll = l[r];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = unpair(acc[r][j]);
                v[2 * j] = f.x, v[2 * j + 1] = f.y;
            }
            for (int k = 1; k < a.slices; k++) {
                const float* src = joined[warp + k];
                float mine, other;
                mm = join(mm, src[LANES * 8], mine, other);
                ll = ll * mine + src[LANES * 8 + 1] * other;
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = v[j] * mine + src[w.d0 + j] * other;
            }
            const int64_t at = w.i * a.heads + w.h0 + r;
            if (a.part) {
                float* dst = a.part + ((int64_t)blockIdx.y * a.queries * a.heads + at) * (a.head + 2);
#pragma unroll
                for (int j = 0; j < 8; j++) dst[w.d0 + j] = v[j];
                if (lane == 0) dst[a.head] = mm, dst[a.head + 1] = ll;
            } else {
                const float inv = ll != 0.0f ? 1.0f / ll : 0.0f, base = ll != 0.0f ? a.v.base : 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = fmaf(v[j], inv, base);
                store_elements(a.out, at * a.head + w.d0, a.dtype, v);
                if (lane == 0) a.lse[at] = ll != 0.0f ? mm + logf(ll) : -INFINITY;
            }
        }
        if (a.slices > 1) __syncthreads();  // `joined` has been read
    }
}

// Joins the blocks' parts of a list in order: a warp for each (query, head).
__global__ void __launch_bounds__(128) k_attend_join(const __grid_constant__ AttendParams a) {
    const int64_t n = a.queries * a.heads, at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, d0 = lane * 8;
    if (at >= n) return;
    float v[8] = {}, m = -INFINITY, l = 0.0f;
    for (int s = 0; s < a.splits; s++) {
        const float* src = a.part + (s * n + at) * (a.head + 2);
        float mine, other;
        m = join(m, src[a.head], mine, other);
        l = l * mine + src[a.head + 1] * other;
        if (d0 < a.head)
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = v[j] * mine + src[d0 + j] * other;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f, base = l != 0.0f ? a.v.base : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = fmaf(v[j], inv, base);
    if (d0 < a.head) store_elements(a.out, at * a.head + d0, a.dtype, v);
    if (lane == 0) a.lse[at] = l != 0.0f ? m + logf(l) : -INFINITY;
}

__device__ __forceinline__ void finish_backward(const AttendParams& a, int64_t at, int d0, bool first, float (&x)[8],
                                                const float (&y)[8], float d, float p) {
    const float inv = p != 0.0f ? 1.0f / p : 0.0f;
    d *= inv;
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = a.scale * inv * (x[j] - d * y[j]);
    store_elements(a.out, at * a.head + d0, a.dtype, x);
    if (a.sum_d && first) a.sum_d[at] = make_float2(d, inv);
}

// A, B, D and the weights' own sum P of the lists' slices; dq = scale (A - (D / P) B) / P.
// P is 1 up to rounding, except where lse cannot hold its own digits beside
// scores of 1e9 and more (a mask of the type's lowest value throughout).
template <int LANES, int RB>
__global__ void __launch_bounds__(32 * kWarps) k_attend_backward(const __grid_constant__ AttendParams a) {
    constexpr int ENTRIES = 32 / LANES;
    constexpr int STEPS = 2;
    constexpr int ROW = LANES * 16 + 2;               // A, B, D, P
    __shared__ float joined[kWarps][ROW];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LANES;
    Work w;
    const bool some = work_of<LANES, RB>(a, w);
    if (!some) w.nr = 0;
    u64 q[RB][4], g[RB][4], va[RB][4], vb[RB][4];
    float kb[RB], gb[RB], z[RB], dsum[RB], psum[RB];
    if (some) {
#pragma unroll
        for (int r = 0; r < RB; r++) {
            float v[8] = {}, d[8] = {};
            const int64_t at = w.i * a.heads + w.h0 + r;
            z[r] = 0.0f;
            if (r < w.nr) {
                z[r] = a.lse_in[at];
                if (w.live) {
                    load_elements(a.q, w.i * a.q_stride + (w.h0 + r) * a.q_head_stride + w.d0, a.dtype, v);
                    load_elements(a.dout, at * a.head + w.d0, a.dtype, d);
                }
            }
            float sq = 0.0f, sg = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) sq += v[j] *= a.scale, sg += d[j];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                q[r][j] = pair(v[2 * j], v[2 * j + 1]);
                g[r][j] = pair(d[2 * j], d[2 * j + 1]);
                va[r][j] = vb[r][j] = 0;
            }
            kb[r] = a.k.base * sq;
            gb[r] = a.v.base * sg;
            dsum[r] = psum[r] = 0.0f;
        }
        const int kg = w.e0 / a.k.group, vg = w.e0 / a.v.group;
        const int32_t doc = a.query_docs ? a.query_docs[w.i] : 0;
        const u64 kbase = pair(a.k.base, a.k.base);
        for (int j0 = w.j0; j0 < w.j1; j0 += 32) {
            float my_bias = 0.0f;
            const int my_slot = j0 + lane < w.j1 ? entry_slot(a, w.i, j0 + lane, doc, my_bias) : -1;
            const int n = min(32, w.j1 - j0);
            for (int t = 0; t < n; t += STEPS * ENTRIES) {
                uint2 kraw[STEPS], vraw[STEPS];
                float ks[STEPS], vs[STEPS], bias[STEPS];
                bool seen[STEPS];
#pragma unroll
                for (int u = 0; u < STEPS; u++) {
                    const int e = t + u * ENTRIES + sub;
                    const int slot = __shfl_sync(0xffffffffu, my_slot, e & 31);
                    bias[u] = __shfl_sync(0xffffffffu, my_bias, e & 31);
                    seen[u] = e < n && slot >= 0;
                    kraw[u] = vraw[u] = make_uint2(0, 0);
                    ks[u] = vs[u] = 0.0f;
                    if (seen[u] && w.live) {
                        kraw[u] = load_codes(a.k, slot, w.e0);
                        vraw[u] = load_codes(a.v, slot, w.e0);
                        ks[u] = load_scale(a.k, slot, kg);
                        vs[u] = load_scale(a.v, slot, vg);
                    }
                }
#pragma unroll
                for (int u = 0; u < STEPS; u++) {
                    const int e = t + u * ENTRIES + sub;
                    u64 kc[4], vc[4];
                    code_pairs(kraw[u], a.k.flip, kc);
                    code_pairs(vraw[u], a.v.flip, vc);
                    const u64 kss = pair(ks[u], ks[u]);
#pragma unroll
                    for (int r = 0; r < RB; r++) {
                        if (r >= w.nr) continue;
                        float x = group_sum<LANES>(fmaf(ks[u], dot_pairs(q[r], kc), kb[r]));
                        const float dp = group_sum<LANES>(fmaf(vs[u], dot_pairs(g[r], vc), gb[r]));
                        float slope = 1.0f;
                        if (a.cap > 0.0f) {
                            const float th = tanh_fast(x * a.inv_cap);
                            x = a.cap * th;
                            slope = 1.0f - th * th;
                        }
                        const float p = seen[u] ? exp_fast(x + bias[u] - z[r]) : 0.0f;
                        const float pdp = seen[u] ? p * dp : 0.0f;
                        dsum[r] += pdp;
                        psum[r] += p;
                        if (a.pd && lane % LANES == 0 && e < n)
                            a.pd[(w.i * a.heads + w.h0 + r) * a.found + j0 + e] = make_float2(pdp, p);
                        const float fa = pdp * slope, fb = p * slope;
                        const u64 pa = pair(fa, fa), pb = pair(fb, fb);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const u64 kv = fma2(kss, kc[j], kbase);  // the key's values (an unseen entry: pa = pb = 0)
                            va[r][j] = fma2(pa, kv, va[r][j]);
                            vb[r][j] = fma2(pb, kv, vb[r][j]);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < RB; r++) {
        if (r < w.nr) {
#pragma unroll
            for (int o = LANES; o < 32; o <<= 1) {
                dsum[r] += __shfl_xor_sync(0xffffffffu, dsum[r], o);
                psum[r] += __shfl_xor_sync(0xffffffffu, psum[r], o);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    va[r][j] = add2(va[r][j], __shfl_xor_sync(0xffffffffu, va[r][j], o));
                    vb[r][j] = add2(vb[r][j], __shfl_xor_sync(0xffffffffu, vb[r][j], o));
                }
            }
            if (a.slices > 1 && lane < LANES) {
                float* dst = joined[warp];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 x = unpair(va[r][j]), y = unpair(vb[r][j]);
                    dst[w.d0 + 2 * j] = x.x, dst[w.d0 + 2 * j + 1] = x.y;
                    dst[LANES * 8 + w.d0 + 2 * j] = y.x, dst[LANES * 8 + w.d0 + 2 * j + 1] = y.y;
                }
                if (lane == 0) dst[LANES * 16] = dsum[r], dst[LANES * 16 + 1] = psum[r];
            }
        }
        if (a.slices > 1) __syncthreads();
        if (r < w.nr && w.slice == 0 && lane < LANES && w.live) {
            float x[8], y[8], d = dsum[r], p = psum[r];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 fa = unpair(va[r][j]), fb = unpair(vb[r][j]);
                x[2 * j] = fa.x, x[2 * j + 1] = fa.y, y[2 * j] = fb.x, y[2 * j + 1] = fb.y;
            }
            for (int k = 1; k < a.slices; k++) {
                const float* src = joined[warp + k];
                d += src[LANES * 16];
                p += src[LANES * 16 + 1];
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] += src[w.d0 + j], y[j] += src[LANES * 8 + w.d0 + j];
            }
            const int64_t at = w.i * a.heads + w.h0 + r;
            if (a.part) {
                float* dst = a.part + ((int64_t)blockIdx.y * a.queries * a.heads + at) * (2 * a.head + 2);
#pragma unroll
                for (int j = 0; j < 8; j++) dst[w.d0 + j] = x[j], dst[a.head + w.d0 + j] = y[j];
                if (lane == 0) dst[2 * a.head] = d, dst[2 * a.head + 1] = p;
            } else {
                finish_backward(a, at, w.d0, lane == 0, x, y, d, p);
            }
        }
        if (a.slices > 1) __syncthreads();  // `joined` has been read
    }
}

__global__ void __launch_bounds__(128) k_attend_backward_join(const __grid_constant__ AttendParams a) {
    const int64_t n = a.queries * a.heads, at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, d0 = lane * 8;
    if (at >= n) return;
    float x[8] = {}, y[8] = {}, d = 0.0f, p = 0.0f;
    for (int s = 0; s < a.splits; s++) {
        const float* src = a.part + (s * n + at) * (2 * a.head + 2);
        d += src[2 * a.head];
        p += src[2 * a.head + 1];
        if (d0 < a.head)
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] += src[d0 + j], y[j] += src[a.head + d0 + j];
    }
    if (d0 < a.head) finish_backward(a, at, d0, lane == 0, x, y, d, p);
}

// dbias[i][j] = sum over heads of (p dP - p D / P) / P, in head order.
__global__ void __launch_bounds__(256) k_attend_dbias(const float2* __restrict__ pd, const float2* __restrict__ sum_d,
                                                      int64_t queries, int heads, int found,
                                                      float* __restrict__ dbias) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= queries * found) return;
    const int64_t i = at / found;
    const int j = (int)(at - i * found);
    float v = 0.0f;
    for (int h = 0; h < heads; h++) {
        const float2 x = pd[(i * heads + h) * found + j];
        const float2 d = __ldg(sum_d + i * heads + h);
        v += (x.x - x.y * d.x) * d.y;
    }
    dbias[at] = v;
}

CodeView code_view(const RowsView& r) {
    CodeView c{};
    c.codes = r.codes;
    c.scales = r.affine ? nullptr : r.scales;
    c.stride = r.stride;
    c.group = r.group;
    c.n_groups = r.n_groups;
    c.flip = r.affine ? 0u : 0x80808080u;
    c.scale = r.step;
    c.base = r.affine ? r.lo + 128.0f * r.step : 0.0f;
    c.vec = reinterpret_cast<uintptr_t>(r.codes) % 8 == 0 && r.stride % 8 == 0;
    return c;
}

// How a call's lists are cut: enough warps to fill the GPU, no slice below
// kMinSlice entries; over a block's warps first (joined in shared memory),
// then over blocks.
void cut_lists(AttendParams& p) {
    p.r_blocks = (int)ceil_div(p.shared, kMaxShared);
    p.units = p.heads / p.shared * p.r_blocks;
    const int64_t want = 148 * 24;
    const int64_t most = std::max<int64_t>(1, ceil_div(p.found, kMinSlice));
    const int64_t cuts = std::max<int64_t>(1, std::min(most, want / std::max<int64_t>(1, p.queries * p.units)));
    p.slices = 1;
    while (p.slices * 2 <= std::min<int64_t>(cuts, kWarps)) p.slices *= 2;
    p.splits = (int)std::min<int64_t>(ceil_div(cuts, p.slices), 65535);
    p.slice_len = (int)std::max<int64_t>(1, ceil_div(p.found, (int64_t)p.slices * p.splits));
}

AttendParams check_attend(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values) {
    MDH_REQUIRE(a, MDH_ERR_INVALID_ARG, "attend: null arguments");
    AttendParams p{};
    const RowsView k = rows_view(keys), v = rows_view(values);
    MDH_REQUIRE(dtype_ok(a->dtype), MDH_ERR_INVALID_ARG, "attend: dtype must be float32, bfloat16 or float16");
    MDH_REQUIRE(a->queries >= 0 && a->found >= 0, MDH_ERR_INVALID_ARG, "attend: queries and found must be >= 0");
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
    cut_lists(p);
    MDH_REQUIRE(p.queries * p.units <= INT32_MAX, MDH_ERR_UNSUPPORTED, "attend: too many queries");
    return p;
}

// The cut of a call from its sizes alone, for the workspace.
AttendParams cut_of(const mdh_attend_args* a) {
    AttendParams p{};
    p.queries = a->queries;
    p.found = a->found;
    p.heads = a->heads;
    p.shared = a->shared;
    p.head = a->head;
    cut_lists(p);
    return p;
}
bool has_sizes(const mdh_attend_args* a) {
    return a && a->queries > 0 && a->found >= 0 && a->heads > 0 && a->shared > 0 && a->heads % a->shared == 0 &&
           a->head > 0;
}
int64_t backward_part(const AttendParams& p) {
    return p.splits > 1 ? round_up(p.splits * p.queries * p.heads * (2 * (int64_t)p.head + 2) * 4, 16) : 0;
}

// fn(LANES, RB): lanes that hold a head, and heads of a warp.
template <class F>
void by_shape(int head, int shared, F&& fn) {
    auto heads = [&](auto lanes) {
        if (shared == 1) fn(lanes, std::integral_constant<int, 1>{});
        else if (shared == 2) fn(lanes, std::integral_constant<int, 2>{});
        else fn(lanes, std::integral_constant<int, kMaxShared>{});
    };
    if (head <= 8) heads(std::integral_constant<int, 1>{});
    else if (head <= 16) heads(std::integral_constant<int, 2>{});
    else if (head <= 32) heads(std::integral_constant<int, 4>{});
    else if (head <= 64) heads(std::integral_constant<int, 8>{});
    else if (head <= 128) heads(std::integral_constant<int, 16>{});
    else heads(std::integral_constant<int, 32>{});
}
dim3 attend_grid(const AttendParams& p) {
    return dim3((unsigned)ceil_div(p.queries * p.units, kWarps / p.slices), (unsigned)p.splits);
}

}  // namespace
}  // namespace mdh

using namespace mdh;

extern "C" {

int64_t mdh_attend_workspace(const mdh_attend_args* a) {
    if (!has_sizes(a)) return 0;
    const AttendParams p = cut_of(a);
    return p.splits > 1 ? p.splits * p.queries * p.heads * ((int64_t)p.head + 2) * 4 : 0;
}

mdh_status mdh_attend(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values, void* out, float* lse,
                      void* ws, int64_t ws_bytes, void* stream) {
    return guarded([&] {
        AttendParams p = check_attend(a, keys, values);
        current_device();
        if (p.queries == 0) return;
        MDH_REQUIRE(out && lse, MDH_ERR_INVALID_ARG, "attend: null output");
        const int64_t need = mdh_attend_workspace(a);
        MDH_REQUIRE(need == 0 || (ws && aligned16(ws) && ws_bytes >= need), MDH_ERR_INVALID_ARG,
                    "attend: workspace too small or not 16-byte aligned");
        const cudaStream_t st = (cudaStream_t)stream;
        p.out = out;
        p.lse = lse;
        p.part = need ? (float*)ws : nullptr;
        by_shape(p.head, p.shared, [&](auto lanes, auto rb) { k_attend<lanes, rb><<<attend_grid(p), 32 * kWarps, 0, st>>>(p); });
        check_launch();
        if (p.splits > 1) {
            k_attend_join<<<(unsigned)ceil_div(p.queries * p.heads, 4), 128, 0, st>>>(p);
            check_launch();
        }
    });
}

int64_t mdh_attend_backward_workspace(const mdh_attend_args* a, int32_t want_dbias) {
    if (!has_sizes(a)) return 0;
    int64_t need = backward_part(cut_of(a));
    if (want_dbias) need += a->queries * a->heads * 8 + a->queries * a->heads * (int64_t)a->found * 8;
    return need;
}

mdh_status mdh_attend_backward(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values,
                               const void* dout, const float* lse, void* dq, float* dbias, void* ws, int64_t ws_bytes,
                               void* stream) {
    return guarded([&] {
        AttendParams p = check_attend(a, keys, values);
        current_device();
        if (p.queries == 0) return;
        MDH_REQUIRE(dout && lse && dq, MDH_ERR_INVALID_ARG, "attend: null dout, lse or dq");
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
        p.lse_in = lse;
        by_shape(p.head, p.shared,
                 [&](auto lanes, auto rb) { k_attend_backward<lanes, rb><<<attend_grid(p), 32 * kWarps, 0, st>>>(p); });
        check_launch();
        if (p.splits > 1) {
            k_attend_backward_join<<<(unsigned)ceil_div(p.queries * p.heads, 4), 128, 0, st>>>(p);
            check_launch();
        }
        if (dbias && p.found) {
            k_attend_dbias<<<(unsigned)bias_blocks, 256, 0, st>>>(p.pd, p.sum_d, p.queries, p.heads, p.found, dbias);
            check_launch();
        }
    });
}

}  // extern "C"
