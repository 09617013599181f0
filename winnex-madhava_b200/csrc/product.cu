// C[m][n] = sum_k a(m, k) b(n, k) for bfloat16 or float16 operands on tcgen05
// (kind::f16, float32 accumulators in tensor memory), with the bias, the
// activation and the residual of a linear layer in the epilogue.
//
// Tile: 128 rows x BN columns, k in blocks of 64.  Either operand may be
// k-major (k contiguous: rows of 128 bytes in shared memory) or row-major in
// its other index (64 x 64 boxes whose 128-byte rows run along m or n), so
// the layer's product and both of its gradients read x, w and dy as they lie
// in memory.  Warps 0-15 are the epilogue (tensor-memory lane quarter w % 4,
// columns by w / 4), warp 16 issues the TMA loads, warp 17 the MMAs; two
// accumulators let an epilogue overlap the next tile's products.  A product
// with few tiles and a long k is split over k: the parts are written in float32
// and joined in order by a second kernel.  Every mbarrier wait is bounded; one
// that gives up is reported once, by the device's next product or by
// mdh_linear_status.  16,384 x 768 x 2,048 bf16 on B200: 48 and 50 us
// for the gradients' products (1.04-1.07 PFLOP/s; their 384 tiles fill 148 SMs
// to 86%, and 48 KB of operands a block of k come from L2), 65 us for the
// forward one with GELU, z and y in its epilogue.
#include <algorithm>
#include <atomic>
#include <mutex>

#include "product.h"
#include "tc_ptx.cuh"

namespace mdh {
namespace {

using namespace op;
using namespace tc;

constexpr int BM = 128, KB = 64;
constexpr int EPI_WARPS = 16;
constexpr int PRODUCER_WARP = EPI_WARPS, MMA_WARP = EPI_WARPS + 1;
constexpr int NUM_THREADS = 32 * (EPI_WARPS + 2);
constexpr uint32_t A_BYTES = BM * KB * 2;
constexpr uint32_t WARP_SMEM = 32 * 64;  // a warp's 32 x 32 chunk of 16-bit values

template <int BN>
struct Shape {
    static constexpr uint32_t B_BYTES = BN * KB * 2;
    static constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr uint32_t OFF_EPI = STAGES * STAGE_BYTES;
    static constexpr uint32_t OFF_BAR = OFF_EPI + EPI_WARPS * WARP_SMEM;
    static constexpr uint32_t BAR_FULL = 0, BAR_EMPTY = STAGES, BAR_ACC_FULL = 2 * STAGES, BAR_ACC_EMPTY = 2 * STAGES + 2,
                              BAR_DRAIN = 2 * STAGES + 4, NUM_BARS = BAR_DRAIN + 1;
    static constexpr uint32_t OFF_SLOT = OFF_BAR + NUM_BARS * 8;
    static constexpr uint32_t SMEM = OFF_SLOT + 8 + 1024;
    static constexpr int TMEM_COLS = 2 * BN;  // 128, 256 or 512
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

struct ProductParams {
    int m, n, nkb;          // nkb: blocks of 64 of k
    int m_tiles, n_tiles, splits;
    int units;
    uint32_t idesc;
    bool f16;
    int act;
    const void *bias, *residual;
    int64_t residual_stride;
    void* y;
    int64_t y_stride;
    void* z;
    float* part;            // splits > 1: [splits][m][pitch]
    int64_t pitch;
    int y_width, z_width, r_width;  // bytes that every row starts on: 16, 8, 4 or 2
    bool b_vec;                     // the bias starts on 16 bytes
    int32_t* status;
};

struct Unit {
    int m0, n0, kb0, kb1, split;
};
template <int BN>
__device__ __forceinline__ Unit unit_at(const ProductParams& p, int u) {
    const int tiles = p.m_tiles * p.n_tiles;
    const int s = u / tiles, t = u - s * tiles, mt = t / p.n_tiles;
    return {mt * BM, (t - mt * p.n_tiles) * BN, (int)((int64_t)s * p.nkb / p.splits),
            (int)((int64_t)(s + 1) * p.nkb / p.splits), s};
}

// Descriptor of an operand whose 128-byte rows run along m or n (128-byte
// swizzle): 8 k-rows are 1024 bytes, a further 64 elements of m or n are one
// box (64 k-rows x 128 bytes) away.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(KB * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ uint32_t pack2(float a, float b, bool f16) {
    uint32_t r;
    if (f16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint32_t v, bool f16) {
    if (f16) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ float half_at(const void* p, int64_t i, bool f16) {
    return f16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Offset of 16-byte piece `piece` of row `row` in a warp's staging chunk.
__device__ __forceinline__ uint32_t staged(int row, int piece) { return row * 64 + ((piece ^ (row >> 1)) & 3) * 16; }

// The forms of the two below for rows that start on fewer than 8 bytes.
__device__ __forceinline__ void chunk_out_any(const uint8_t* stage, uint16_t* out, int64_t stride, int width, int row0,
                                           int col0, int m, int n, int lane) {
    // Rows that start anywhere: lanes side by side, a row (or two, by words) at a time.
    const int per = width == 4 ? 2 : 1, sub = width == 4 ? lane >> 4 : 0, e = width == 4 ? (lane & 15) * 2 : lane;
    const int col = col0 + e;
#pragma unroll 8
    for (int r = sub; r < 32; r += per) {
        if (row0 + r >= m || col >= n) continue;
        const uint8_t* src = stage + staged(r, e >> 3) + (e & 7) * 2;
        uint16_t* dst = out + (int64_t)(row0 + r) * stride + col;
        if (width == 4 && col + 1 < n) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
        else *dst = *reinterpret_cast<const uint16_t*>(src);
    }
}
__device__ __forceinline__ void chunk_in_any(uint8_t* stage, const uint16_t* in, int64_t stride, int row0, int col0, int m,
                                          int n, int lane) {
    // Lanes side by side; eight rows are in flight before the first is stored (more would cost the other forms
    // registers).
    const int col = col0 + lane;
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 8) {
        uint16_t v[8];
#pragma unroll
        for (int r = 0; r < 8; r++)
            v[r] = row0 + r0 + r < m && col < n ? __ldg(in + (int64_t)(row0 + r0 + r) * stride + col) : (uint16_t)0;
#pragma unroll
        for (int r = 0; r < 8; r++)
            *reinterpret_cast<uint16_t*>(stage + staged(r0 + r, lane >> 3) + (lane & 7) * 2) = v[r];
    }
}

// Staging chunk -> 32 rows x 32 columns of p at (row0, col0), clipped to m x
// n; rows start on `width` bytes (16, 8, 4 or 2).
__device__ __forceinline__ void chunk_out(const uint8_t* stage, void* p, int64_t stride, int width, int row0, int col0,
                                          int m, int n, int lane) {
    uint16_t* out = static_cast<uint16_t*>(p);
    if (width < 8) return chunk_out_any(stage, out, stride, width, row0, col0, m, n, lane);
#pragma unroll
    for (int it = 0; it < 4; it++) {
        const int r = it * 8 + (lane >> 2), piece = lane & 3, col = col0 + piece * 8;
        if (row0 + r >= m || col >= n) continue;
        uint16_t* dst = out + (int64_t)(row0 + r) * stride + col;
        const uint4 v = *reinterpret_cast<const uint4*>(stage + staged(r, piece));
        if (width == 16 && col + 8 <= n) {
            *reinterpret_cast<uint4*>(dst) = v;
        } else if (width == 8 && col + 8 <= n) {
            reinterpret_cast<uint2*>(dst)[0] = make_uint2(v.x, v.y);
            reinterpret_cast<uint2*>(dst)[1] = make_uint2(v.z, v.w);
        } else {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(&v);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (col + j < n) dst[j] = e[j];
        }
    }
}
// The reverse: zeros outside m x n.
__device__ __forceinline__ void chunk_in(uint8_t* stage, const void* p, int64_t stride, int width, int row0, int col0,
                                         int m, int n, int lane) {
    const uint16_t* in = static_cast<const uint16_t*>(p);
    if (width < 8) return chunk_in_any(stage, in, stride, row0, col0, m, n, lane);
#pragma unroll
    for (int it = 0; it < 4; it++) {
        const int r = it * 8 + (lane >> 2), piece = lane & 3, col = col0 + piece * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row0 + r < m && col < n) {
            const uint16_t* src = in + (int64_t)(row0 + r) * stride + col;
            if (width == 16 && col + 8 <= n) {
                v = __ldg(reinterpret_cast<const uint4*>(src));
            } else if (width == 8 && col + 8 <= n) {
                const uint2 a = __ldg(reinterpret_cast<const uint2*>(src)), b = __ldg(reinterpret_cast<const uint2*>(src) + 1);
                v = make_uint4(a.x, a.y, b.x, b.y);
            } else {
                uint16_t e[8];
#pragma unroll
                for (int j = 0; j < 8; j++) e[j] = col + j < n ? src[j] : 0;
                v = *reinterpret_cast<const uint4*>(e);
            }
        }
        *reinterpret_cast<uint4*>(stage + staged(r, piece)) = v;
    }
}
__device__ __forceinline__ void stage_row(uint8_t* stage, const f32x2 (&v)[16], bool f16, int lane) {
#pragma unroll
    for (int piece = 0; piece < 4; piece++) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = unpair(v[piece * 4 + j]);
            w[j] = pack2(f.x, f.y, f16);
        }
        *reinterpret_cast<uint4*>(stage + staged(lane, piece)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int ACT>
__device__ __forceinline__ void activate32(f32x2 (&v)[16]) {
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = activate(v[j], ACT);
}

// Adds 8 16-bit values to four pairs.
__device__ __forceinline__ void add8(f32x2* v, uint4 x, bool f16) {
    const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 f = unpack2(e[j], f16);
        v[j] = add2(v[j], pair(f.x, f.y));
    }
}

// One 32 x 32 chunk of sums, a row a lane: bias, z, activation, residual, y.
__device__ __forceinline__ void finish_chunk(const ProductParams& p, f32x2 (&v)[16], int row0, int col0, uint8_t* stage,
                                             int lane) {
    if (p.bias) {
        // The same 32 values for every lane.
        const uint16_t* b = static_cast<const uint16_t*>(p.bias) + col0;
        if (p.b_vec && col0 + 32 <= p.n) {
#pragma unroll
            for (int piece = 0; piece < 4; piece++) add8(v + 4 * piece, __ldg(reinterpret_cast<const uint4*>(b) + piece), p.f16);
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int c = col0 + 2 * j;
                v[j] = add2(v[j], pair(c < p.n ? half_at(b, 2 * j, p.f16) : 0.0f,
                                       c + 1 < p.n ? half_at(b, 2 * j + 1, p.f16) : 0.0f));
            }
        }
    }
    if (p.z) {
        stage_row(stage, v, p.f16, lane);
        __syncwarp();
        chunk_out(stage, p.z, p.n, p.z_width, row0, col0, p.m, p.n, lane);
        __syncwarp();
    }
    if (p.act == MDH_ACT_RELU) activate32<MDH_ACT_RELU>(v);
    else if (p.act == MDH_ACT_GELU) activate32<MDH_ACT_GELU>(v);
    else if (p.act == MDH_ACT_SILU) activate32<MDH_ACT_SILU>(v);
    if (p.residual) {
        chunk_in(stage, p.residual, p.residual_stride, p.r_width, row0, col0, p.m, p.n, lane);
        __syncwarp();
#pragma unroll
        for (int piece = 0; piece < 4; piece++)
            add8(v + 4 * piece, *reinterpret_cast<const uint4*>(stage + staged(lane, piece)), p.f16);
        __syncwarp();
    }
    stage_row(stage, v, p.f16, lane);
    __syncwarp();
    chunk_out(stage, p.y, p.y_stride, p.y_width, row0, col0, p.m, p.n, lane);
    __syncwarp();
}

// Offset of an operand's next 16 of k within a block of 64, in descriptor units of 16 bytes.
template <bool MN>
__device__ __forceinline__ uint64_t k_step(int kk) {
    return MN ? (uint64_t)(kk * 2048 >> 4) : (uint64_t)(kk * 32 >> 4);
}

template <int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    k_product(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
              const __grid_constant__ ProductParams p) {
    using S = Shape<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bars = sbase + S::OFF_BAR;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::OFF_SLOT);
    volatile int32_t* abort_flag = reinterpret_cast<volatile int32_t*>(smem + S::OFF_SLOT + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; s++) {
            mbar_init(bars + 8 * (S::BAR_FULL + s), 1);
            mbar_init(bars + 8 * (S::BAR_EMPTY + s), 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(bars + 8 * (S::BAR_ACC_FULL + s), 1);
            mbar_init(bars + 8 * (S::BAR_ACC_EMPTY + s), EPI_WARPS);
        }
        mbar_init(bars + 8 * S::BAR_DRAIN, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == MMA_WARP) tmem_alloc<1>(smem_u32(tmem_slot), S::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == PRODUCER_WARP) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_a) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_b) : "memory");
            int stage = 0;
            uint32_t phase = 0, issued_mask = 0, last_parity = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
                const Unit t = unit_at<BN>(p, u);
                for (int kb = t.kb0; kb < t.kb1; kb++) {
                    ok = mbar_wait<false>(bars + 8 * (S::BAR_EMPTY + stage), phase ^ 1, abort_flag, p.status);
                    if (!ok) break;
                    const uint32_t full = bars + 8 * (S::BAR_FULL + stage);
                    const uint32_t sa = sbase + stage * S::STAGE_BYTES, sb = sa + A_BYTES;
                    mbar_expect_tx(full, S::STAGE_BYTES);
                    if (A_MN) {
#pragma unroll
                        for (int i = 0; i < BM / 64; i++)
                            tma_load_2d(sa + i * KB * 128, &tmap_a, full, t.m0 + 64 * i, kb * KB);
                    } else {
                        tma_load_2d(sa, &tmap_a, full, kb * KB, t.m0);
                    }
                    if (B_MN) {
#pragma unroll
                        for (int i = 0; i < BN / 64; i++)
                            tma_load_2d(sb + i * KB * 128, &tmap_b, full, t.n0 + 64 * i, kb * KB);
                    } else {
                        tma_load_2d(sb, &tmap_b, full, kb * KB, t.n0);
                    }
                    issued_mask |= 1u << stage;
                    last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == S::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok)
                for (int s = 0; s < S::STAGES; s++)
                    if (issued_mask & (1u << s))
                        mbar_drain_wait<false>(bars + 8 * (S::BAR_FULL + s), (last_parity >> s) & 1);
        }
    } else if (warp == MMA_WARP) {
        if (lane == 0) {
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true, issued = false, full_ready = false;
            for (int u = blockIdx.x; u < p.units && ok; u += gridDim.x) {
                const Unit t = unit_at<BN>(p, u);
                ok = mbar_wait_inl<false>(bars + 8 * (S::BAR_ACC_EMPTY + acc), acc_phase ^ 1, abort_flag, p.status);
                if (!ok) break;
                const uint32_t d = tmem_base + (uint32_t)(acc * BN);
                for (int kb = t.kb0; kb < t.kb1; kb++) {
                    if (!full_ready) {
                        ok = mbar_wait_inl<false>(bars + 8 * (S::BAR_FULL + stage), phase, abort_flag, p.status);
                        if (!ok) break;
                    }
                    tc_fence_after();
                    const int nstage = stage + 1 == S::STAGES ? 0 : stage + 1;
                    const uint32_t nphase = stage + 1 == S::STAGES ? phase ^ 1 : phase;
                    const uint32_t sa = sbase + stage * S::STAGE_BYTES, sb = sa + A_BYTES;
                    const uint64_t ad = A_MN ? mn_desc(sa) : sw128_desc(sa), bd = B_MN ? mn_desc(sb) : sw128_desc(sb);
                    bool pf = false;
#pragma unroll
                    for (int kk = 0; kk < KB / 16; kk++) {
                        umma_f16(d, ad + k_step<A_MN>(kk), bd + k_step<B_MN>(kk), p.idesc,
                                 (kb > t.kb0 || kk > 0) ? 1u : 0u);
                        if (kk == 1) pf = mbar_test_wait(bars + 8 * (S::BAR_FULL + nstage), nphase);
                    }
                    issued = true;
                    umma_commit(bars + 8 * (S::BAR_EMPTY + stage));
                    full_ready = pf;
                    stage = nstage;
                    phase = nphase;
                }
                if (!ok) break;
                umma_commit(bars + 8 * (S::BAR_ACC_FULL + acc));
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
            if (!ok && issued) {
                umma_commit(bars + 8 * S::BAR_DRAIN);
                mbar_drain_wait<false>(bars + 8 * S::BAR_DRAIN, 0);
            }
        }
    } else {
        const int quarter = warp & 3, part = warp >> 2;
        // Chunks of 32 columns of this warp; a tile of 64 columns has none for the last 8 warps.
        constexpr int CHUNKS = BN >= 128 ? BN / 128 : 1;
        const bool works = part * 32 < BN;
        uint8_t* stage = smem + S::OFF_EPI + warp * WARP_SMEM;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int u = blockIdx.x; u < p.units; u += gridDim.x) {
            const Unit t = unit_at<BN>(p, u);
            if (!mbar_wait_inl<false>(bars + 8 * (S::BAR_ACC_FULL + acc), acc_phase, abort_flag, p.status)) break;
            tc_fence_after();
            const int row0 = t.m0 + quarter * 32;
#pragma unroll 1
            for (int c = 0; c < CHUNKS; c++) {
                const int off = (part * CHUNKS + c) * 32;
                uint32_t raw[32];
                __syncwarp();
                if (works) {
                    tmem_ld32_issue(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * BN + off), raw);
                    tmem_ld_wait(raw);
                }
                if (c == CHUNKS - 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bars + 8 * (S::BAR_ACC_EMPTY + acc));
                }
                const int col0 = t.n0 + off;
                if (!works || row0 >= p.m || col0 >= p.n) continue;
                if (p.part) {
                    if (row0 + lane < p.m) {
                        float* dst = p.part + ((int64_t)t.split * p.m + row0 + lane) * p.pitch + col0;
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (col0 + 4 * j < p.n)  // the pitch is a multiple of 4
                                *reinterpret_cast<float4*>(dst + 4 * j) =
                                    make_float4(__uint_as_float(raw[4 * j]), __uint_as_float(raw[4 * j + 1]),
                                                __uint_as_float(raw[4 * j + 2]), __uint_as_float(raw[4 * j + 3]));
                    }
                } else {
                    f32x2 v[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] = pair(__uint_as_float(raw[2 * j]), __uint_as_float(raw[2 * j + 1]));
                    finish_chunk(p, v, row0, col0, stage, lane);
                }
            }
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1;
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, S::TMEM_COLS);
    }
}

// Joins the parts of a split k in order and finishes: 4 columns a thread.
__global__ void __launch_bounds__(256) k_product_join(const __grid_constant__ ProductParams p) {
    const int groups = (int)(p.pitch / 4);
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = at / groups;
    if (row >= p.m) return;
    const int col = (int)(at - row * groups) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    const int64_t step = (int64_t)p.m * p.pitch;
    const float* src = p.part + row * p.pitch + col;
    for (int s = 0; s < p.splits; s++) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(src + s * step));
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int c = col + j;
        if (c >= p.n) break;
        float f = e[j] + (p.bias ? half_at(p.bias, c, p.f16) : 0.0f);
        if (p.z) static_cast<uint16_t*>(p.z)[row * p.n + c] = (uint16_t)pack2(f, 0.0f, p.f16);
        f = activate(f, p.act);
        if (p.residual) f += half_at(p.residual, row * p.residual_stride + c, p.f16);
        static_cast<uint16_t*>(p.y)[row * p.y_stride + c] = (uint16_t)pack2(f, 0.0f, p.f16);
    }
}

// Rows of 16-bit elements -> rows of `pitch` elements (what follows the row is
// not read); one operand for each blockIdx.y.
struct PackJob {
    const uint16_t* src;
    uint16_t* dst;
    int64_t stride, rows, width, pitch;
};
struct PackJobs {
    PackJob job[2];
};
__global__ void __launch_bounds__(256) k_pack_rows(const __grid_constant__ PackJobs jobs) {
    const PackJob& p = jobs.job[blockIdx.y];
    const int64_t pieces = p.pitch / 8, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t r = at / pieces;
    if (r >= p.rows) return;
    const int64_t c = (at - r * pieces) * 8;
    uint16_t e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = c + j < p.width ? p.src[r * p.stride + c + j] : (uint16_t)0;
    *reinterpret_cast<uint4*>(p.dst + r * p.pitch + c) = *reinterpret_cast<const uint4*>(e);
}

// ------------------------------------------------------------ host
// The words that products which gave up a wait write, one a device: pinned
// host memory.
constexpr int kDevices = 64;
int32_t* status_word(int dev) {
    static std::once_flag once;
    static int32_t* words = nullptr;
    std::call_once(once, [] {
        int32_t* w = nullptr;
        MDH_CUDA(cudaHostAlloc((void**)&w, kDevices * sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped));
        std::fill_n(w, kDevices, 0);
        words = w;
    });
    return words + dev % kDevices;
}

struct Plan {
    int bn, splits;
};

// Tile width and parts of k: the choice whose slowest SM finishes first.  In
// units of one 128 x 256 x 64 block: a narrower tile's block costs more per
// column (its operands are read from shared memory more often), a tile costs
// its fill and its epilogue, and a split costs a second kernel.
Plan plan_product(int64_t m, int64_t n, int64_t nkb) {
    Plan best{256, 1};
    double best_cost = 1e300;
    for (int bn : {256, 128, 64}) {
        const double block = bn == 256 ? 1.0 : bn == 128 ? 0.55 : 0.35;
        const int64_t tiles = ceil_div(m, BM) * ceil_div(n, bn);
        // Unsplit, or the fewest parts that bring a part down to what 1, 2 or 3 rounds of the SMs allow.
        for (int rounds = 0; rounds <= 3; rounds++) {
            int64_t s = rounds ? std::min<int64_t>({64, nkb, 148 * rounds / tiles}) : 1;
            if (rounds && s < 2) continue;
            s = ceil_div(nkb, ceil_div(nkb, s));
            const double waves = (double)ceil_div(tiles * s, 148);
            double cost = waves * ((double)ceil_div(nkb, s) * block + 3.0);
            if (s > 1) cost += 10.0 + (double)(s + 1) * m * n * 4 / 3.0e6;
            if (cost < best_cost) best_cost = cost, best = {bn, (int)s};
        }
    }
    return best;
}

// The bytes, 16 at most, that every row of 16-bit elements starts on.
int row_width(const void* p, int64_t stride) {
    const uint64_t bits = reinterpret_cast<uintptr_t>(p) | (uint64_t)stride * 2 | 16;
    return (int)(bits & (~bits + 1));
}

// Whether TMA reads the operand in place.
bool readable(const ProductOperand& o) { return rows_aligned(o.p, o.stride, 2); }
int64_t lines(const ProductOperand& o, int64_t rows, int64_t k) { return o.k_major ? rows : k; }
int64_t line(const ProductOperand& o, int64_t rows, int64_t k) { return o.k_major ? k : rows; }
int64_t packed_bytes(const ProductOperand& o, int64_t rows, int64_t k) {
    return readable(o) ? 0 : lines(o, rows, k) * round_up(line(o, rows, k), 8) * 2;
}

// The operand itself, or where its packed copy will be and the job that makes it.
ProductOperand packed(const ProductOperand& o, int64_t rows, int64_t k, void* to, PackJobs& jobs, int& n) {
    if (readable(o)) return o;
    const int64_t width = line(o, rows, k), pitch = round_up(width, 8);
    jobs.job[n++] = {(const uint16_t*)o.p, (uint16_t*)to, o.stride, lines(o, rows, k), width, pitch};
    return {to, pitch, o.k_major};
}
void pack(const PackJobs& jobs, int n, cudaStream_t st) {
    if (n == 0) return;
    int64_t blocks = 0;
    for (int i = 0; i < n; i++) blocks = std::max(blocks, ceil_div(jobs.job[i].rows * (jobs.job[i].pitch / 8), 256));
    MDH_REQUIRE(blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "linear: operand too large");
    k_pack_rows<<<dim3((unsigned)blocks, (unsigned)n), 256, 0, st>>>(jobs);
    check_launch();
}

void tensor_map(CUtensorMap* map, const ProductOperand& o, int64_t rows, int64_t k, int tile_rows) {
    const int64_t width = line(o, rows, k);
    // One line needs no stride of its own; TMA asks for one that holds it.
    const int64_t stride = lines(o, rows, k) == 1 ? round_up(width, 8) : o.stride;
    encode_tmap_2d_sw128(map, 1, o.p, width, lines(o, rows, k), stride * 2, 64, o.k_major ? tile_rows : KB);
}

template <int BN, bool A_MN, bool B_MN>
void launch(const CUtensorMap& ta, const CUtensorMap& tb, const ProductParams& p, int sms, cudaStream_t st) {
    static std::atomic<uint64_t> set{0};
    int dev = 0;
    MDH_CUDA(cudaGetDevice(&dev));
    if (!(set.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
        MDH_CUDA(cudaFuncSetAttribute(k_product<BN, A_MN, B_MN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      Shape<BN>::SMEM));
        set.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_relaxed);
    }
    k_product<BN, A_MN, B_MN><<<std::min(p.units, sms), NUM_THREADS, Shape<BN>::SMEM, st>>>(ta, tb, p);
    check_launch();
}

}  // namespace

namespace op {

int64_t product_workspace(const ProductOperand& a, const ProductOperand& b, int64_t m, int64_t n, int64_t k) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    const Plan plan = plan_product(m, n, ceil_div(k, KB));
    const int64_t parts = plan.splits > 1 ? plan.splits * m * round_up(n, 4) * 4 : 0;
    return round_up(packed_bytes(a, m, k), 128) + round_up(packed_bytes(b, n, k), 128) + parts;
}

void product(const ProductOperand& a0, const ProductOperand& b0, int64_t m, int64_t n, int64_t k, int32_t dtype,
             const ProductEpilogue& ep, void* ws, cudaStream_t st) {
    const int dev = current_device(), sms = device_sm_count(dev);
    char* at = static_cast<char*>(ws);
    PackJobs jobs{};
    int n_jobs = 0;
    const ProductOperand a = packed(a0, m, k, at, jobs, n_jobs);
    at += round_up(packed_bytes(a0, m, k), 128);
    const ProductOperand b = packed(b0, n, k, at, jobs, n_jobs);
    at += round_up(packed_bytes(b0, n, k), 128);
    pack(jobs, n_jobs, st);
    const Plan plan = plan_product(m, n, ceil_div(k, KB));
    ProductParams p{};
    p.m = (int)m;
    p.n = (int)n;
    p.nkb = (int)ceil_div(k, KB);
    p.m_tiles = (int)ceil_div(m, BM);
    p.n_tiles = (int)ceil_div(n, plan.bn);
    p.splits = plan.splits;
    const int64_t units = (int64_t)p.m_tiles * p.n_tiles * p.splits;
    MDH_REQUIRE(units <= INT32_MAX / 2, MDH_ERR_UNSUPPORTED, "linear: product too large");
    p.units = (int)units;
    p.f16 = dtype == MDH_F16;
    const uint32_t type = p.f16 ? 0u : 1u;
    p.idesc = (1u << 4) | (type << 7) | (type << 10) | (a.k_major ? 0u : 1u << 15) | (b.k_major ? 0u : 1u << 16) |
              ((uint32_t)(plan.bn >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
    p.act = ep.act;
    p.bias = ep.bias;
    p.residual = ep.residual;
    p.residual_stride = ep.residual_stride;
    p.y = ep.y;
    p.y_stride = ep.y_stride;
    p.z = ep.z;
    p.y_width = row_width(ep.y, ep.y_stride);
    p.z_width = row_width(ep.z, n);
    p.r_width = row_width(ep.residual, ep.residual_stride);
    p.b_vec = aligned16(ep.bias);
    p.pitch = round_up(n, 4);
    p.part = p.splits > 1 ? reinterpret_cast<float*>(at) : nullptr;
    p.status = status_word(dev);
    CUtensorMap ta, tb;
    tensor_map(&ta, a, m, k, BM);
    tensor_map(&tb, b, n, k, plan.bn);
    auto by_bn = [&](auto bn) {
        if (a.k_major && b.k_major) launch<bn, false, false>(ta, tb, p, sms, st);
        else if (a.k_major) launch<bn, false, true>(ta, tb, p, sms, st);
        else launch<bn, true, true>(ta, tb, p, sms, st);
    };
    MDH_REQUIRE(a.k_major || !b.k_major, MDH_ERR_INTERNAL, "linear: operand order");
    if (plan.bn == 256) by_bn(std::integral_constant<int, 256>{});
    else if (plan.bn == 128) by_bn(std::integral_constant<int, 128>{});
    else by_bn(std::integral_constant<int, 64>{});
    if (p.splits > 1) {
        const int64_t blocks = ceil_div(m * (p.pitch / 4), 256);
        MDH_REQUIRE(blocks <= INT32_MAX, MDH_ERR_UNSUPPORTED, "linear: product too large");
        k_product_join<<<(unsigned)blocks, 256, 0, st>>>(p);
        check_launch();
    }
}

void check_product_status() {
    const int32_t s = __atomic_exchange_n(status_word(current_device()), 0, __ATOMIC_ACQ_REL);
    MDH_REQUIRE(s == 0, MDH_ERR_TIMEOUT,
                "linear: a device-side wait of an earlier call expired; the results since the last check are void");
}

void set_product_expired() { __atomic_store_n(status_word(current_device()), (int32_t)kDevTimeout, __ATOMIC_RELEASE); }

}  // namespace op
}  // namespace mdh
