// Attention over the 8-bit KV cache for many queries a kv head (prompt chunks, drafts): the formulas of kv8_attn.cu on
// the 5th-generation tensor cores. What bounds it is the tensor pipe (4 D flops a query and row), so tiles are
// 128 queries x 128 rows:
//   S = Q . K^T      tcgen05 kind::f16, Q and the decoded codes of K from shared memory, S in tensor memory
//   O += P . V       P (fp16, written over S) from tensor memory, the decoded codes of V from shared memory
// The codes become fp16 exactly (|c| <= 127); K's scales multiply the finished scores, V's the weights, as in the
// kernel for few queries, and so do its choices: q as fp16 scaled by a power of two to [256, 512) (bf16: exact but
// for values 2^-22 below the row's largest; fp32: two parts, 22 bits), weights w = 2^(x - m) s_v c as fp16 (fp32
// calls: two parts), m raised only when a score passes it by 2^6 (e^4 with a mask, scores then in natural units).
//
// One CTA per SM walks its part of the list of units (128 rows of one tile and kv head; Walk). Warp roles:
//  * softmax warps (four per query tile; a thread is a query): stage the tile's queries, then per row tile read S,
//    form the weights, write P; at a segment's end scale O and store it (or a partial). S is read twice, for the
//    largest score and for the weights, 32 columns at a time: holding the weights back instead, until the reference is
//    known to stand, spilled, and its unrolled code missed the instruction cache (412 -> XXX us).
//  * four decode warps: 128 rows of codes, K and V in turn, from memory (the next tile's loads in flight) to fp16 in
//    the 128-byte-swizzled layout, two stages each. K is read K-major, V (rows are K of the product) MN-major.
//  * one warp issues the products and owns tensor memory.
// QT = 2 query tiles share a decoded row tile and alternate: one's softmax runs beside the other's products. QT = 1
// (at most 128 queries, or fp32) alternates two S buffers instead.
// Every wait is bounded (2 s) and reports through the error word.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.h"
#include "kv8.cuh"
#include "ptx.cuh"
#include "tc.cuh"

namespace onpu_b200 {
namespace {

constexpr int kRows = 128;                               // rows of a tile, queries of a tile
constexpr int kSub = kRows * 128;                        // bytes of 128 rows x 64 fp16
constexpr int kBars = 20;
constexpr int kDec = 4;                                  // decode warps

template <int DP, int QT, int PARTS>
struct TileSizes {
    static constexpr int tile = kRows * DP * 2;          // 128 rows of DP fp16: DP / 64 sub-tiles of 64
    static constexpr int smem = 1024 + (QT * PARTS + 4) * tile + kBars * 8 + 16;
    static constexpr int soft = 4 * QT, threads = (soft + kDec + 1) * 32;
};

// byte offset of 16-byte chunk c (8 fp16) of row r in a tile
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
    return static_cast<uint32_t>((c >> 3) * kSub + r * 128 + (((c ^ r) & 7) << 4));
}
__device__ __forceinline__ void sts_v4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// pairs of fp32 in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// instruction descriptor: fp32 accumulator, fp16 A and B, B MN-major or K-major, N x 128
template <int N, bool BMN>
constexpr uint32_t kIdesc = (1u << 4) | (BMN ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
                            (static_cast<uint32_t>(kRows >> 4) << 24);

template <int DP, int QT, int PARTS, bool BF16, bool MASK>
__global__ void __launch_bounds__(TileSizes<DP, QT, PARTS>::threads, 1) kv8_attn_tile_kernel(const Kv8AttnParams p) {
    using Z = TileSizes<DP, QT, PARTS>;
    constexpr int CH = DP / 16;                          // 16-code chunks of a row
    constexpr float U = MASK ? kLog2e : 1.f, RAISE = MASK ? 4.f : 6.f;
    constexpr int kO = 256, kP2 = kO + 128;              // tensor-memory columns of O, of the weights' second parts; S at 0, 128
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t qs = base, ks = qs + QT * PARTS * Z::tile, vs = ks + 2 * Z::tile, bars = vs + 2 * Z::tile;
    const uint32_t q_full = bars, s_full = q_full + 16, p_full = s_full + 16, o_full = p_full + 16, k_full = o_full + 16,
                   k_empty = k_full + 16, v_full = k_empty + 16, v_empty = v_full + 16, drain = v_empty + 16;
    const uint32_t slot_addr = bars + kBars * 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = gridDim.x, D = p.c.D;
    const Kv8Cache &c = p.c;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + 8 * i, 4);                // a query tile's softmax warps
            mbar_init(s_full + 8 * i, 1);                // commits
            mbar_init(p_full + 8 * i, 4);
            mbar_init(o_full + 8 * i, 1);
            mbar_init(k_full + 8 * i, kDec);             // decode warps
            mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_full + 8 * i, kDec);
            mbar_init(v_empty + 8 * i, 1);
        }
        mbar_init(drain, 1);
        mbar_init_fence();
    }
    pdl_wait_prerequisites();
    pdl_launch_dependents();                             // after the wait: the join may read pos and cnt as it starts
    if (warp == Z::soft + kDec) {
        tmem_alloc(slot_addr, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot_addr));

    const Plan pl(p, QT * kRows, kRows);
    Walk wk;
    const bool any = wk.start(p, pl, lane, blockIdx.x, G);
    bool failed = false;
    int jt = 0;                                          // row tiles so far, over all segments
    if (!any) {
        // nothing for this CTA
    } else if (warp < Z::soft) {
        // ============================================================ softmax
        const int qt = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t otm = tmem + lanes + kO + qt * DP;
        int pv = 0;                                      // products of this query tile with V so far
        int ns = 0;                                      // its S tiles so far
        for (; wk.segment(p, pl); wk.next()) {
            const int row0 = wk.ua * kRows, row1 = min(wk.len, wk.ub * kRows), n = wk.ub - wk.ua;
            const int qi = qt * kRows + row;
            if (qt * kRows >= wk.nq) continue;
            const bool ok = qi < wk.nq;
            const int b = wk.b, h = wk.h;
            const int tok = static_cast<int>(div64(wk.q0 + (ok ? qi : 0), pl.rep));
            const int hq = h * pl.rep + static_cast<int>(wk.q0 + (ok ? qi : 0) - static_cast<int64_t>(tok) * pl.rep);
            const int64_t qo = (static_cast<int64_t>(b) * p.r.T + tok) * p.ldq + static_cast<int64_t>(hq) * D;
            const float *ksb = c.ks + b * c.sbs + h * c.shs, *vsb = c.vs + b * c.sbs + h * c.shs;
            // lane i: K's (i < 8) or V's scale of the i % 8-th 16 rows of a tile
            auto load_scale = [&](int r0) {
                const int r = r0 + 16 * (lane & 7);
                return lane < 16 && r < row1 ? (lane < 8 ? ksb : vsb)[r >> c.blk_log2] : 0.f;
            };
            float sc = load_scale(row0);

            // the query, scaled to [256, 512) and rounded to fp16, into its row of the tile
            auto load8 = [&](int d, float (&x)[8]) {
                if (!ok || d >= D) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = 0.f;
                } else if constexpr (BF16) {
                    const uint4 v = ld_nc_v4(static_cast<const uint16_t *>(p.q) + qo + d);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[2 * e] = __uint_as_float(w[e] << 16);
                        x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint4 v = ld_nc_v4(static_cast<const float *>(p.q) + qo + d + 4 * k);
                        x[4 * k] = __uint_as_float(v.x);
                        x[4 * k + 1] = __uint_as_float(v.y);
                        x[4 * k + 2] = __uint_as_float(v.z);
                        x[4 * k + 3] = __uint_as_float(v.w);
                    }
                }
            };
            float mx = 0.f;
#pragma unroll 4
            for (int d = 0; d < DP; d += 8) {
                float x[8];
                load8(d, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) mx = max_nan(mx, fabsf(x[e]));
            }
            const float fq = pow2_to(mx, 8), fs = p.scale < 0.f ? -fq : fq;     // a negative scale: on the query
#pragma unroll 4
            for (int d = 0; d < DP; d += 8) {
                float x[8];
                load8(d, x);
                uint32_t w[4], w2[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = x[2 * e] * fs, bb = x[2 * e + 1] * fs;
                    w[e] = pack_h2(a, bb);
                    if constexpr (PARTS == 2) {
                        const float2 r = unpack_h2(w[e]);
                        w2[e] = pack_h2(a - r.x, bb - r.y);
                    }
                }
                sts_v4(qs + qt * PARTS * Z::tile + tile_off(row, d >> 3), make_uint4(w[0], w[1], w[2], w[3]));
                if constexpr (PARTS == 2)
                    sts_v4(qs + (qt * PARTS + 1) * Z::tile + tile_off(row, d >> 3), make_uint4(w2[0], w2[1], w2[2], w2[3]));
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + 8 * qt);
            // a query that is not finite has NaN scores
            const float rs = mx < INFINITY ? fabsf(p.scale) * (MASK ? 1.f : kLog2e) / fq : __uint_as_float(0x7fc00000u);
            const int lim = ok ? wk.pos + tok : -1;              // the last row it sees
            const int edge = __shfl_sync(0xffffffffu, lim, 0) + 1;   // lane 0's is the warp's smallest, or -1: nothing valid
            const float *mrow = MASK ? p.mask + b * p.mbs + tok * p.mts : nullptr;

            float m = 0.f, l = 0.f, cv = 0.f;
            bool have = false;                                   // m is a score's
            for (int j = 0; j < n; ++j) {
                const int r0 = row0 + j * kRows, buf = QT == 2 ? qt : ns & 1;
                const uint32_t stm = tmem + lanes + buf * kRows;
                const float scj = sc;
                if (j + 1 < n) sc = load_scale(r0 + kRows);
                const uint32_t sphase = QT == 2 ? ns & 1 : ns >> 1 & 1;
                if (!failed) failed = __any_sync(0xffffffffu, !mbar_wait_bounded(s_full + 8 * buf, sphase, kWaitNs));
                ++ns;
                tc_fence_after();
                if (edge > 0) {                                  // a warp without a valid query leaves its lanes of P as they are
                    // V's largest scale (bits: NaN does not count) against the weights' power of two
                    uint32_t vb = lane >= 8 && lane < 16 ? __float_as_uint(scj) : 0u;
                    vb = __reduce_max_sync(0xffffffffu, vb <= 0x7f800000u ? vb : 0u);
                    const float vmax = __uint_as_float(vb);
                    float fix = 1.f;                             // of O, for a new power of two and a new reference
                    if (vmax * cv > 512.f || (cv == 0.f && vmax > 0.f)) {
                        const float cn = pow2_to(vmax, 7);
                        if (cv != 0.f) fix = cn / cv;
                        cv = cn;
                    }
                    bool touch = fix != 1.f;                     // uniform
                    const bool edged = MASK || r0 + kRows > edge;
                    // a score of the tile's column, -inf where it is not seen
                    auto score = [&](uint32_t s, float f, int col) {
                        float x = __uint_as_float(s) * f;
                        if (col > lim) return -INFINITY;
                        if constexpr (MASK) {
                            const float mk = mrow[col];
                            x = mk == -INFINITY ? -INFINITY : x + mk;
                        }
                        return x;
                    };
                    // the tile's largest score against the reference
                    float top = -INFINITY;
#pragma unroll 1
                    for (int ch = 0; ch < 4; ++ch) {
                        uint32_t s[32];
                        tc_ld_32x32b_x32(stm + 32 * ch, s);
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const float f = rs * __shfl_sync(0xffffffffu, scj, 2 * ch + g);
                            if (!edged) {                        // scales are not negative
                                float t = __uint_as_float(s[16 * g]);
#pragma unroll
                                for (int k = 1; k < 16; ++k) t = fmaxf(t, __uint_as_float(s[16 * g + k]));
                                top = fmaxf(top, t * f);
                            } else {
#pragma unroll
                                for (int k = 0; k < 16; ++k) top = fmaxf(top, score(s[16 * g + k], f, r0 + 32 * ch + 16 * g + k));
                            }
                        }
                    }
                    const bool raise = top > m + RAISE || (!have && top > -INFINITY);
                    if (__any_sync(0xffffffffu, raise)) {
                        if (raise) {
                            const float a = have ? ex2((m - top) * U) : 0.f;
                            m = top;
                            l *= a;
                            fix *= a;
                            have = true;
                        }
                        touch = true;
                    }
                    if (touch && j > 0) {                        // O onto the new reference, once its last product is done
                        if (!failed)
                            failed = __any_sync(0xffffffffu, !mbar_wait_bounded(o_full + 8 * qt, (pv - 1) & 1, kWaitNs));
                        tc_fence_after();
#pragma unroll 1
                        for (int ch = 0; ch < DP / 32; ++ch) {
                            uint32_t v[32];
                            tc_ld_32x32b_x32(otm + 32 * ch, v);
#pragma unroll
                            for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * fix);
                            tc_st_32x32b_x32(otm + 32 * ch, v);
                        }
                    }
                    // weights: 32 scores at a time, their pairs over the first half of the columns read so far (the second
                    // parts of fp32 calls in a buffer of their own)
                    const float2 mm = make_float2(-m, -m);
                    float2 lt = make_float2(0.f, 0.f);
#pragma unroll 1
                    for (int ch = 0; ch < 4; ++ch) {
                        uint32_t s[32], ph[16], pw[16];
                        tc_ld_32x32b_x32(stm + 32 * ch, s);
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const float f = rs * __shfl_sync(0xffffffffu, scj, 2 * ch + g);
                            const float wv = cv * __shfl_sync(0xffffffffu, scj, 8 + 2 * ch + g);
                            auto keep = [&](int k, float2 w) {
                                ph[8 * g + k / 2] = pack_h2(w.x, w.y);
                                if constexpr (PARTS == 2) {
                                    const float2 r = unpack_h2(ph[8 * g + k / 2]);
                                    pw[8 * g + k / 2] = pack_h2(w.x - r.x, w.y - r.y);
                                }
                            };
                            if (!edged) {
#pragma unroll
                                for (int k = 0; k < 16; k += 2) {
                                    const float2 a = fma2(make_float2(__uint_as_float(s[16 * g + k]), __uint_as_float(s[16 * g + k + 1])),
                                                          make_float2(f, f), mm);
                                    const float2 e = make_float2(ex2(a.x * U), ex2(a.y * U));
                                    lt = add2(lt, e);
                                    keep(k, mul2(e, make_float2(wv, wv)));
                                }
                            } else {
#pragma unroll
                                for (int k = 0; k < 16; k += 2) {
                                    const int col = r0 + 32 * ch + 16 * g + k;
                                    const float x0 = score(s[16 * g + k], f, col), x1 = score(s[16 * g + k + 1], f, col + 1);
                                    const float2 e = make_float2(ex2((x0 - m) * U), ex2((x1 - m) * U));
                                    lt = add2(lt, e);
                                    // a row that is not seen weighs nothing, even where its scale is NaN
                                    keep(k, make_float2(x0 == -INFINITY ? 0.f : e.x * wv, x1 == -INFINITY ? 0.f : e.y * wv));
                                }
                            }
                        }
                        tc_st_32x32b_x16(stm + 16 * ch, ph);
                        if constexpr (PARTS == 2) tc_st_32x32b_x16(tmem + lanes + kP2 + 64 * buf + 16 * ch, pw);
                    }
                    l += lt.x + lt.y;
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * buf);
                ++pv;
            }
            if (!failed) failed = __any_sync(0xffffffffu, !mbar_wait_bounded(o_full + 8 * qt, (pv - 1) & 1, kWaitNs));
            tc_fence_after();
            // O c^-1 relative to m: the output, or a partial
            const float M = have ? m : -INFINITY, inv = cv == 0.f ? 1.f : 1.f / cv;
            float so, f = inv;
            if (wk.whole()) f = out_factor<MASK>(M, l, p.sinks, hq, so) * so * inv;
            const int64_t oo = (static_cast<int64_t>(b) * p.r.T + tok) * p.ldo + static_cast<int64_t>(hq) * D;
            float *po = slot_o<DP>(p.ws, QT * kRows, wk.slot(blockIdx.x)) + static_cast<int64_t>(qi) * DP;
#pragma unroll 1
            for (int ch = 0; ch < DP / 32; ++ch) {
                uint32_t v[32];
                __syncwarp();
                tc_ld_32x32b_x32(otm + 32 * ch, v);
                if (!ok) continue;
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    const int d = 32 * ch + k;
                    const float4 y = make_float4(__uint_as_float(v[k]) * f, __uint_as_float(v[k + 1]) * f,
                                                 __uint_as_float(v[k + 2]) * f, __uint_as_float(v[k + 3]) * f);
                    if (d < D) {
                        if (wk.whole()) store4<BF16>(p.out, oo + d, y);
                        else *reinterpret_cast<float4 *>(po + d) = y;
                    }
                }
            }
            if (ok && !wk.whole()) slot_ml<DP>(p.ws, QT * kRows, G, wk.slot(blockIdx.x))[qi] = make_float2(M, l);
            tc_fence_before();
            __syncwarp();
        }
    } else if (warp < Z::soft + kDec) {
        // ============================================================ decode
        const int dt = threadIdx.x - Z::soft * 32;
        for (; wk.segment(p, pl); wk.next()) {
            const int row0 = wk.ua * kRows, row1 = min(wk.len, wk.ub * kRows), n = wk.ub - wk.ua;
            const int8_t *kb = c.k + wk.b * c.bs + wk.h * c.hs, *vb = c.v + wk.b * c.bs + wk.h * c.hs;
            // a thread's chunks of a tile: every (32 kDec)-th, CH chunks to a row
            constexpr int IT = (kRows * CH + 32 * kDec - 1) / (32 * kDec);
            auto load = [&](const int8_t *src, int r0, uint4 (&x)[IT]) {
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    const int idx = dt + i * 32 * kDec, r = r0 + idx / CH, ch = idx % CH;
                    x[i] = r < row1 && idx < kRows * CH && ch * 16 < D
                               ? ld_nc_v4(src + static_cast<int64_t>(r) * c.rs + ch * 16) : make_uint4(0, 0, 0, 0);
                }
            };
            auto store = [&](uint32_t dst, const uint4 (&x)[IT]) {
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    const int idx = dt + i * 32 * kDec, r = idx / CH, ch = idx % CH;
                    if (idx >= kRows * CH) break;
                    const uint32_t w[4] = {x[i].x ^ 0x80808080u, x[i].y ^ 0x80808080u, x[i].z ^ 0x80808080u, x[i].w ^ 0x80808080u};
                    const uint4 lo = make_uint4(h2_lo(w[0]), h2_hi(w[0]), h2_lo(w[1]), h2_hi(w[1]));
                    const uint4 hi = make_uint4(h2_lo(w[2]), h2_hi(w[2]), h2_lo(w[3]), h2_hi(w[3]));
                    const int odd = ch >> 2 & 1;                 // the second sub-tile's halves the other way round: no bank twice
                    sts_v4(dst + tile_off(r, 2 * ch + odd), odd ? hi : lo);
                    sts_v4(dst + tile_off(r, 2 * ch + 1 - odd), odd ? lo : hi);
                }
            };
            uint4 xk[IT], xv[IT];
            load(kb, row0, xk);
            for (int j = 0; j < n; ++j, ++jt) {
                const int st = jt & 1, use = jt >> 1;
                load(vb, row0 + j * kRows, xv);
                if (!failed && use > 0) failed = __any_sync(0xffffffffu, !mbar_wait_bounded(k_empty + 8 * st, (use - 1) & 1, kWaitNs));
                store(ks + st * Z::tile, xk);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full + 8 * st);
                if (j + 1 < n) load(kb, row0 + (j + 1) * kRows, xk);
                if (!failed && use > 0) failed = __any_sync(0xffffffffu, !mbar_wait_bounded(v_empty + 8 * st, (use - 1) & 1, kWaitNs));
                store(vs + st * Z::tile, xv);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full + 8 * st);
            }
        }
    } else if (lane == 0) {
        // ============================================================ products
        auto wait = [&](uint32_t bar, uint32_t parity) {
            if (!failed && !mbar_wait_bounded(bar, parity & 1, kWaitNs)) failed = true;
            tc_fence_after();
        };
        auto qk = [&](int qt, int tile, int buf) {               // S[buf] = Q . K^T of row tile `tile`
            if (!failed) {
#pragma unroll
                for (int pt = 0; pt < PARTS; ++pt)
#pragma unroll
                    for (int kk = 0; kk < DP / 16; ++kk) {
                        const uint32_t off = (kk >> 2) * kSub + (kk & 3) * 32;
                        tc_mma_f16(tmem + buf * kRows, sw128_desc(qs + (qt * PARTS + pt) * Z::tile + off),
                                   sw128_desc(ks + (tile & 1) * Z::tile + off), kIdesc<kRows, false>, (pt | kk) != 0);
                    }
            }
            tc_commit(s_full + 8 * buf);                         // also after a failure: keeps the others moving
        };
        auto pvp = [&](int qt, int tile, int buf, bool more) {   // O[qt] (+)= P[buf] . V of row tile `tile`
            if (!failed) {
#pragma unroll
                for (int pt = 0; pt < PARTS; ++pt)
#pragma unroll
                    for (int kk = 0; kk < kRows / 16; ++kk)
                        tc_mma_f16_ta(tmem + kO + qt * DP, tmem + (pt ? kP2 + buf * 64 : buf * kRows) + kk * 8,
                                      sw128_desc_mn(vs + (tile & 1) * Z::tile + kk * 2048, kSub), kIdesc<DP, true>,
                                      more || (pt | kk) != 0);
            }
            tc_commit(o_full + 8 * qt);
        };
        int nq[2] = {0, 0}, np[2] = {0, 0};                      // phases of q_full and p_full waited for
        for (; wk.segment(p, pl); wk.next()) {
            const int n = wk.ub - wk.ua, nqt = QT == 2 && wk.nq > kRows ? 2 : 1;
            wait(k_full + 8 * (jt & 1), jt >> 1);
            for (int qt = 0; qt < nqt; ++qt) {
                wait(q_full + 8 * qt, nq[qt]++);
                qk(qt, jt, QT == 2 ? qt : jt & 1);
            }
            tc_commit(k_empty + 8 * (jt & 1));
            for (int j = 0; j < n; ++j, ++jt) {
                const bool more = j + 1 < n;
                const int nx = jt + 1;
                if (more) wait(k_full + 8 * (nx & 1), nx >> 1);
                if (QT == 1 && more) {
                    qk(0, nx, nx & 1);
                    tc_commit(k_empty + 8 * (nx & 1));
                }
                for (int qt = 0; qt < nqt; ++qt) {
                    const int buf = QT == 2 ? qt : jt & 1;
                    wait(p_full + 8 * buf, np[buf]++);
                    if (qt == 0) wait(v_full + 8 * (jt & 1), jt >> 1);
                    pvp(qt, jt, buf, j > 0);
                    if (QT == 2 && more) qk(qt, nx, qt);
                }
                tc_commit(v_empty + 8 * (jt & 1));
                if (QT == 2 && more) tc_commit(k_empty + 8 * (nx & 1));
            }
        }
        // tensor memory is idle before it is freed
        tc_commit(drain);
        if (!mbar_wait_bounded(drain, 0, kWaitNs)) failed = true;
    }
    if (failed && lane == 0) atomicOr(p.r.err, 64);
    tc_fence_before();
    __syncthreads();
    if (warp == Z::soft + kDec) tmem_dealloc(tmem, 512);
}

int sms() {
    static const int n = [] {
        int dev = 0, v = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
        return v > 0 ? v : 1;
    }();
    return n;
}

template <int DP, int QT, bool BF16, bool MASK>
cudaError_t launch_t(const Kv8AttnParams &p, cudaStream_t s) {
    constexpr int PARTS = BF16 ? 1 : 2;
    using Z = TileSizes<DP, QT, PARTS>;
    const auto k = kv8_attn_tile_kernel<DP, QT, PARTS, BF16, MASK>;
    static const cudaError_t attr = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::smem);
    if (attr != cudaSuccess) return attr;
    return launch_pdl(k, dim3(sms()), dim3(Z::threads), Z::smem, s, p);
}
template <int DP, int QT>
cudaError_t launch_q(const Kv8AttnParams &p, bool bf16, cudaStream_t s) {
    const bool mask = p.mask != nullptr;
    if constexpr (QT == 1) {
        if (!bf16) return mask ? launch_t<DP, QT, false, true>(p, s) : launch_t<DP, QT, false, false>(p, s);
    }
    return mask ? launch_t<DP, QT, true, true>(p, s) : launch_t<DP, QT, true, false>(p, s);
}

}  // namespace

// query tiles a CTA takes at a time: two share the decoded rows where there are more than 128 queries (fp32
// queries are two parts each, as large as two tiles)
int kv8_tile_queries(int64_t queries, bool bf16) { return bf16 && queries > kRows ? 2 * kRows : kRows; }
int kv8_tile_rows() { return kRows; }
int kv8_tile_ctas() { return sms(); }

cudaError_t kv8_tile_launch(const Kv8AttnParams &p, bool bf16, cudaStream_t s) {
    const int64_t queries = static_cast<int64_t>(p.r.T) * (p.Hq / p.c.Hkv);
    if (kv8_tile_queries(queries, bf16) == 2 * kRows)
        return p.c.D <= 64 ? launch_q<64, 2>(p, bf16, s) : launch_q<128, 2>(p, bf16, s);
    return p.c.D <= 64 ? launch_q<64, 1>(p, bf16, s) : launch_q<128, 1>(p, bf16, s);
}

}  // namespace onpu_b200
