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
#include "op_rows.cuh"

namespace mdh {
namespace {

using namespace op;

constexpr int kThreads = 128;
constexpr int kMaxHead = 256;
constexpr int kPer = kMaxHead / 32;  // elements of a head a lane holds

struct AttendParams {
    RowsView k, v;
    const int32_t* ids;
    const float* bias;
    const int32_t *query_docs, *row_docs;
    int64_t q_stride, q_head_stride, ids_stride, bias_stride;
    int64_t queries;
    int found, heads, shared, head;
    float scale, cap;
};

// Slot of entry j of query i, or -1 when it is hidden; its bias.
__device__ __forceinline__ int entry_slot(const AttendParams& a, int64_t i, int j, float& bias) {
    const int id = a.ids[i * a.ids_stride + j];
    bias = 0.0f;
    if (id < 0 || id >= a.k.slots) return -1;
    if (a.bias) {
        bias = a.bias[i * a.bias_stride + j];
        if (bias == -INFINITY) return -1;
    }
    if (a.row_docs && a.row_docs[id] != a.query_docs[i]) return -1;
    return id;
}

__device__ __forceinline__ float row_value(const RowsView& c, int64_t slot, int e) {
    const uint8_t code = c.codes[slot * c.stride + e];
    return c.affine ? affine_value(code, c.lo, c.step)
                    : (float)(int8_t)code * c.scales[slot * c.n_groups + e / c.group];
}

// One warp for one (query, head).
template <class T>
__global__ void __launch_bounds__(kThreads)
    k_attend(AttendParams a, const T* __restrict__ q, T* __restrict__ out, float* __restrict__ lse) {
    const int lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (at >= a.queries * a.heads) return;
    const int64_t i = at / a.heads;
    const int h = (int)(at - i * a.heads), base = h / a.shared * a.head;
    float qv[kPer], acc[kPer], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int d = lane + 32 * e;
        qv[e] = d < a.head ? to_f32(q[i * a.q_stride + h * a.q_head_stride + d]) : 0.0f;
        acc[e] = 0.0f;
    }
    for (int j = 0; j < a.found; j++) {
        float bias;
        const int slot = entry_slot(a, i, j, bias);
        if (slot < 0) continue;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const int d = lane + 32 * e;
            if (d < a.head) s += qv[e] * row_value(a.k, slot, base + d);
        }
        s = warp_sum(s) * a.scale;
        if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
        s += bias;
        const float top = fmaxf(m, s);
        const float keep = m == -INFINITY ? 0.0f : expf(m - top), p = top == -INFINITY ? 0.0f : expf(s - top);
        l = l * keep + p;
        m = top;
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const int d = lane + 32 * e;
            if (d < a.head) acc[e] = acc[e] * keep + p * row_value(a.v, slot, base + d);
        }
    }
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int d = lane + 32 * e;
        if (d < a.head) out[at * a.head + d] = from_f32<T>(l != 0.0f ? acc[e] / l : 0.0f);
    }
    if (lane == 0) lse[at] = l != 0.0f ? m + logf(l) : -INFINITY;
}

// As above.  pd[2][queries][heads][found] (or null) keeps p_j dP_j and p_j of
// every entry for dbias, sum_d[queries][heads] keeps D.
template <class T>
__global__ void __launch_bounds__(kThreads)
    k_attend_backward(AttendParams a, const T* __restrict__ q, const T* __restrict__ dout,
                      const float* __restrict__ lse, T* __restrict__ dq, float2* __restrict__ pd,
                      float* __restrict__ sum_d) {
    const int lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (at >= a.queries * a.heads) return;
    const int64_t i = at / a.heads;
    const int h = (int)(at - i * a.heads), base = h / a.shared * a.head;
    float qv[kPer], ov[kPer], va[kPer], vb[kPer], dsum = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int d = lane + 32 * e;
        qv[e] = d < a.head ? to_f32(q[i * a.q_stride + h * a.q_head_stride + d]) : 0.0f;
        ov[e] = d < a.head ? to_f32(dout[at * a.head + d]) : 0.0f;
        va[e] = vb[e] = 0.0f;
    }
    const float z = lse[at];
    for (int j = 0; j < a.found; j++) {
        float bias;
        const int slot = entry_slot(a, i, j, bias);
        float p = 0.0f, pdp = 0.0f;
        if (slot >= 0) {
            float s = 0.0f, dp = 0.0f, kv[kPer];
#pragma unroll
            for (int e = 0; e < kPer; e++) {
                const int d = lane + 32 * e;
                kv[e] = d < a.head ? row_value(a.k, slot, base + d) : 0.0f;
                s += qv[e] * kv[e];
                if (d < a.head) dp += ov[e] * row_value(a.v, slot, base + d);
            }
            s = warp_sum(s) * a.scale;
            dp = warp_sum(dp);
            float slope = 1.0f;
            if (a.cap > 0.0f) {
                const float t = tanhf(s / a.cap);
                s = a.cap * t;
                slope = 1.0f - t * t;
            }
            p = expf(s + bias - z);
            pdp = p * dp;
            dsum += pdp;
#pragma unroll
            for (int e = 0; e < kPer; e++) {
                va[e] += pdp * slope * kv[e];
                vb[e] += p * slope * kv[e];
            }
        }
        if (pd && lane == 0) pd[at * a.found + j] = make_float2(pdp, p);
    }
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int d = lane + 32 * e;
        if (d < a.head) dq[at * a.head + d] = from_f32<T>(a.scale * (va[e] - dsum * vb[e]));
    }
    if (sum_d && lane == 0) sum_d[at] = dsum;
}

// dbias[i][j] = sum over heads of p dP - p D, in head order.
__global__ void __launch_bounds__(256) k_attend_dbias(const float2* __restrict__ pd, const float* __restrict__ sum_d,
                                                      int64_t queries, int heads, int found,
                                                      float* __restrict__ dbias) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= queries * found) return;
    const int64_t i = at / found;
    const int j = (int)(at - i * found);
    float v = 0.0f;
    for (int h = 0; h < heads; h++) {
        const float2 x = pd[(i * heads + h) * found + j];
        v += x.x - x.y * sum_d[i * heads + h];
    }
    dbias[at] = v;
}

AttendParams check_attend(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values) {
    MDH_REQUIRE(a, MDH_ERR_INVALID_ARG, "attend: null arguments");
    AttendParams p{};
    p.k = rows_view(keys);
    p.v = rows_view(values);
    MDH_REQUIRE(dtype_ok(a->dtype), MDH_ERR_INVALID_ARG, "attend: dtype must be float32, bfloat16 or float16");
    MDH_REQUIRE(a->queries >= 0 && a->found >= 0, MDH_ERR_INVALID_ARG, "attend: queries and found must be >= 0");
    MDH_REQUIRE(a->heads >= 1 && a->shared >= 1 && a->heads % a->shared == 0, MDH_ERR_INVALID_ARG,
                "attend: heads must be a positive multiple of shared");
    MDH_REQUIRE(a->head >= 8 && a->head % 8 == 0 && a->head <= kMaxHead, MDH_ERR_UNSUPPORTED,
                "attend: the head size must be a multiple of 8 up to 256");
    MDH_REQUIRE(p.k.slots == p.v.slots, MDH_ERR_INVALID_ARG, "attend: key and value caches differ in slots");
    const int64_t width = (int64_t)(a->heads / a->shared) * a->head;
    MDH_REQUIRE(p.k.width == width && p.v.width == width, MDH_ERR_INVALID_ARG,
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
    p.ids = a->ids;
    p.bias = a->bias;
    p.query_docs = a->query_docs;
    p.row_docs = a->row_docs;
    p.q_stride = a->q_stride;
    p.q_head_stride = a->q_head_stride;
    p.ids_stride = a->ids_stride;
    p.bias_stride = a->bias_stride;
    p.queries = a->queries;
    p.found = a->found;
    p.heads = a->heads;
    p.shared = a->shared;
    p.head = a->head;
    p.scale = a->scale;
    p.cap = a->cap;
    return p;
}

}  // namespace
}  // namespace mdh

using namespace mdh;

extern "C" {

int64_t mdh_attend_workspace(const mdh_attend_args* a) {
    (void)a;
    return 0;
}

mdh_status mdh_attend(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values, void* out, float* lse,
                      void* ws, int64_t ws_bytes, void* stream) {
    (void)ws;
    (void)ws_bytes;
    return guarded([&] {
        const AttendParams p = check_attend(a, keys, values);
        current_device();
        if (p.queries == 0) return;
        MDH_REQUIRE(out && lse, MDH_ERR_INVALID_ARG, "attend: null output");
        const int64_t blocks = ceil_div(p.queries * p.heads, kThreads / 32);
        MDH_REQUIRE(blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "attend: too many queries");
        by_dtype(a->dtype, [&](auto zero) {
            using T = decltype(zero);
            k_attend<T><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(p, (const T*)a->q, (T*)out, lse);
        });
        check_launch();
    });
}

int64_t mdh_attend_backward_workspace(const mdh_attend_args* a, int32_t want_dbias) {
    if (!a || !want_dbias || a->queries <= 0 || a->heads <= 0 || a->found < 0) return 0;
    return round_up(a->queries * a->heads * 4, 16) + a->queries * a->heads * (int64_t)a->found * 8;
}

mdh_status mdh_attend_backward(const mdh_attend_args* a, const mdh_rows* keys, const mdh_rows* values,
                               const void* dout, const float* lse, void* dq, float* dbias, void* ws, int64_t ws_bytes,
                               void* stream) {
    return guarded([&] {
        const AttendParams p = check_attend(a, keys, values);
        current_device();
        if (p.queries == 0) return;
        MDH_REQUIRE(dout && lse && dq, MDH_ERR_INVALID_ARG, "attend: null dout, lse or dq");
        MDH_REQUIRE(!dbias || (ws && aligned16(ws) && ws_bytes >= mdh_attend_backward_workspace(a, 1)),
                    MDH_ERR_INVALID_ARG, "attend: workspace too small or not 16-byte aligned");
        const cudaStream_t st = (cudaStream_t)stream;
        const int64_t blocks = ceil_div(p.queries * p.heads, kThreads / 32);
        const int64_t bias_blocks = ceil_div(p.queries * p.found, 256);
        MDH_REQUIRE(blocks <= INT32_MAX && bias_blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "attend: too many queries");
        float* sum_d = dbias ? (float*)ws : nullptr;
        float2* pd = dbias ? (float2*)((char*)ws + round_up(p.queries * p.heads * 4, 16)) : nullptr;
        by_dtype(a->dtype, [&](auto zero) {
            using T = decltype(zero);
            k_attend_backward<T><<<(unsigned)blocks, kThreads, 0, st>>>(p, (const T*)a->q, (const T*)dout, lse, (T*)dq,
                                                                      pd, sum_d);
        });
        check_launch();
        if (dbias && p.found) {
            k_attend_dbias<<<(unsigned)bias_blocks, 256, 0, st>>>(pd, sum_d, p.queries, p.heads, p.found, dbias);
            check_launch();
        }
    });
}

}  // extern "C"
