// Attention over the 8-bit KV cache for many bf16 queries a kv head (prompt chunks): the formulas of kv8_attn.cu on
// the 5th-generation tensor cores. What bounds it is the tensor pipe (4 D flops a query and row), so tiles are
// 128 queries x 128 rows:
//   S = Q . K^T      tcgen05 kind::f16, Q and the decoded codes of K from shared memory, S in tensor memory
//   O += P . V       P (fp16, written over S) from tensor memory, the decoded codes of V from shared memory
// The codes become fp16 exactly (|c| <= 127). K's scales multiply the finished scores, whose reference m is raised only when
// one passes it by 2^6 (e^4 with a mask, scores then in natural units). V's scales go into the weights' exponents,
//   w = 2^(x - m + log2 s_v - d + 8)  as fp16 (2^-11 of it; 2^-33 of the query's largest where it is tiny beside that one),
// d the query's own, raised when a weight passes it by 2^6: only rows that the query sees set it, by what they weigh.
// q is fp16 scaled by a power of two to [256, 512): exact but for values 2^-22 below the row's largest.
//
// One CTA per SM walks its part of the list of units (128 rows of one tile and kv head; Walk). Warp roles:
//  * softmax warps, eight per query tile: a thread is a query and one half of a row tile's columns, so that the time
//    from scores to weights, which the products wait for, is half as long. Per row tile: the largest score (a barrier with
//    a vote joins the halves; m and d are raised only if one asks), then the weights, 32 at a time, written over the
//    scores just read. At a segment's end O is scaled and stored (or a partial).
//  * three decode warps: codes that TMA brought (128 rows, K and V in turn, one of each ahead) to fp16 in the
//    128-byte-swizzled layout, two stages each. K is read K-major, V (rows are K of the product) MN-major.
//  * one warp issues the products and owns tensor memory.
// QT = 2 query tiles share a decoded row tile and alternate: one's softmax runs beside the other's products. QT = 1
// (at most 128 queries) alternates two S buffers instead.
//
// Measured: 512 tokens over 16.8k rows, 40 query heads on 8 kv heads of 128: 249 to 254 us (0.42 of the products' floor at the
// measured bf16 rate; 1088 us in the kernel for few queries). With the work of a role left out, the same call takes 118 us
// without any, 185 with the products alone, 209 with the decoding too: what is left besides the products is the chain from
// one role to the next, several times per 128 rows, and the softmax's part of it. 128 columns a softmax thread: 280 to 298;
// all 128 scores in registers: 382 (the unrolled code misses the instruction cache).
//
// Every wait is bounded (2 s) and reports through the error word.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.h"
#include "kv8.cuh"
#include "ptx.cuh"
#include "tc.cuh"
#include "tmap.h"

namespace onpu_b200 {
namespace {

constexpr int kRows = 128;                               // rows of a tile, queries of a tile
constexpr int kSub = kRows * 128;                        // bytes of 128 rows x 64 fp16
constexpr int kBars = 24;
constexpr float kTop = 8.f;                              // log2 of the weight that a query's largest begins as (fp16 holds 2^15)
constexpr int kDec = 3;                                  // decode warps: 12 or 20 warps in all, 3 or 5 a scheduler

template <int DP, int QT>
struct TileSizes {
    static constexpr int tile = kRows * DP * 2;          // 128 rows of DP fp16: DP / 64 sub-tiles of 64
    static constexpr int raw = kRows * DP;               // 128 rows of codes
    static constexpr int share = QT * 2 * kRows * 4;     // a float per softmax thread
    static constexpr int smem = (QT + 4) * tile + 2 * raw + share + kBars * 8 + 16;
    static_assert(smem <= 227 * 1024, "a CTA's shared memory");
    static constexpr int soft = 8 * QT, threads = (soft + kDec + 1) * 32;
};

// byte offset of 16-byte chunk c (8 fp16) of row r in a tile
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
    return static_cast<uint32_t>((c >> 3) * kSub + r * 128 + (((c ^ r) & 7) << 4));
}
__device__ __forceinline__ void sts_v4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// instruction descriptor: fp32 accumulator, fp16 A and B, B MN-major or K-major, N x 128
template <int N, bool BMN>
constexpr uint32_t kIdesc = (1u << 4) | (BMN ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
                            (static_cast<uint32_t>(kRows >> 4) << 24);

// whether any of the barrier's threads votes yes
__device__ __forceinline__ bool bar_any(int id, int count, bool vote) {
    int r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %3, 0;\n\t"
        "barrier.cta.red.or.pred q, %1, %2, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(id), "r"(count), "r"(static_cast<int>(vote))
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void tma_codes(uint32_t dst, const CUtensorMap *map, int row, int head, int seq, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(head), "r"(seq), "r"(bar)
        : "memory");
}

template <int DP, int QT, bool MASK>
__global__ void __launch_bounds__(TileSizes<DP, QT>::threads, 1)
    kv8_attn_tile_kernel(const __grid_constant__ CUtensorMap mapk, const __grid_constant__ CUtensorMap mapv,
                         const Kv8AttnParams p) {
    using Z = TileSizes<DP, QT>;
    constexpr int CH = DP / 16;                          // 16-code chunks of a row
    constexpr float U = MASK ? kLog2e : 1.f, RAISE = MASK ? 4.f : 6.f;
    constexpr int kO = 256;                              // tensor-memory column of O; S buffers at 0 and 128
    extern __shared__ __align__(1024) uint8_t smem_raw[];        // the swizzle's period
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t qs = base, ks = qs + QT * Z::tile, vs = ks + 2 * Z::tile, raw = vs + 2 * Z::tile;
    float *share = reinterpret_cast<float *>(smem_raw + (raw + 2 * Z::raw - smem_u32(smem_raw)));     // [QT][2][128]
    const uint32_t bars = raw + 2 * Z::raw + Z::share;
    const uint32_t q_full = bars, s_full = q_full + 16, p_full = s_full + 16, o_full = p_full + 16, k_full = o_full + 16,
                   k_empty = k_full + 16, v_full = k_empty + 16, v_empty = v_full + 16, raw_full = v_empty + 16, drain = raw_full + 16;
    const uint32_t slot_addr = bars + kBars * 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = gridDim.x, D = p.c.D;
    const Kv8Cache &c = p.c;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + 8 * i, 8);                // a query tile's softmax warps
            mbar_init(s_full + 8 * i, 1);                // commits
            mbar_init(p_full + 8 * i, 8);
            mbar_init(o_full + 8 * i, 1);
            mbar_init(k_full + 8 * i, 1);                // a decode thread, for all
            mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_full + 8 * i, 1);
            mbar_init(v_empty + 8 * i, 1);
            mbar_init(raw_full + 8 * i, 1);              // copies
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
        const int qt = warp >> 3, hf = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
        float *mine = share + (qt * 2 + hf) * kRows + row, *other = share + (qt * 2 + (hf ^ 1)) * kRows + row;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t otm = tmem + lanes + kO + qt * DP;
        // Product i of this query tile with V is done. QT = 1: product i - 1 may still run while the scores behind it are
        // worked on, so odd and even products have a barrier each; one parity would not tell i from i - 2.
        const auto wait_o = [&](int i) {
            return QT == 2 ? mbar_wait_bounded(o_full + 8 * qt, i & 1, kWaitNs)
                           : mbar_wait_bounded(o_full + 8 * (i & 1), i >> 1 & 1, kWaitNs);
        };
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
                } else {
                    const uint4 v = ld_nc_v4(static_cast<const uint16_t *>(p.q) + qo + d);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[2 * e] = __uint_as_float(w[e] << 16);
                        x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
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
            for (int d = hf * (DP / 2); d < (hf + 1) * (DP / 2); d += 8) {      // each thread its half of the row
                float x[8];
                load8(d, x);
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = pack_h2(x[2 * e] * fs, x[2 * e + 1] * fs);
                sts_v4(qs + qt * Z::tile + tile_off(row, d >> 3), make_uint4(w[0], w[1], w[2], w[3]));
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + 8 * qt);
            // a query that is not finite has NaN scores
            const float rs = mx < INFINITY ? fabsf(p.scale) * (MASK ? 1.f : kLog2e) / fq : __uint_as_float(0x7fc00000u);
            const int lim = ok ? wk.pos + tok : -1;              // the last row it sees
            const int edge = __shfl_sync(0xffffffffu, lim, 0) + 1;   // lane 0's is the warp's smallest, or -1: nothing valid
            const float *mrow = MASK ? p.mask + b * p.mbs + tok * p.mts : nullptr;

            // m: the scores' reference; d: the weights', above m's and in log2 units: w = 2^((x - m) U + log2(s_v) - d + kTop)
            float m = 0.f, l = 0.f, d = -INFINITY;
            bool have = false;                                   // m is a score's
            for (int j = 0; j < n; ++j) {
                const int r0 = row0 + j * kRows, buf = QT == 2 ? qt : ns & 1;
                const uint32_t stm = tmem + lanes + buf * kRows;
                const float scj = sc;
                if (j + 1 < n) sc = load_scale(r0 + kRows);
                const bool live = edge > 0;                      // a warp without a valid query leaves its lanes of P as they are
                // O times a, once its last product is done: this half of its columns (at most once a tile: the stores are waited for
                // with the weights')
                const auto rescale_o = [&](float a) {
                    if (j == 0 || !live) return;                 // O begins with this tile
                    if (!failed) failed = __any_sync(0xffffffffu, !wait_o(pv - 1));
                    tc_fence_after();
#pragma unroll 1
                    for (int ch = hf * (DP / 32); ch < (hf + 1) * (DP / 32); ++ch) {
                        uint32_t v[16];
                        tc_ld_32x32b_x16(otm + 16 * ch, v);
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * a);
                        tc_st_32x32b_x16(otm + 16 * ch, v);
                    }
                };
                // what the four 16-column groups of this half need: K's scale with the query's, the logarithm of V's
                float fk[4], lg[4], topg[4];
                {
                    const float lv = __log2f(scj);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        fk[g] = rs * __shfl_sync(0xffffffffu, scj, 4 * hf + g);
                        lg[g] = __shfl_sync(0xffffffffu, lv, 8 + 4 * hf + g);
                        topg[g] = -INFINITY;
                    }
                }
                const bool clear = !MASK && r0 + kRows <= edge;  // every query of the warp sees every row
                const uint32_t sphase = QT == 2 ? ns & 1 : ns >> 1 & 1;
                if (!failed) failed = __any_sync(0xffffffffu, !mbar_wait_bounded(s_full + 8 * buf, sphase, kWaitNs));
                ++ns;
                tc_fence_after();
                // a finished score of the tile's column, -inf where it is not seen
                const auto score = [&](uint32_t s, float f, int col) {
                    const float x = __uint_as_float(s) * f;
                    if constexpr (MASK) {
                        const float mk = col <= lim ? mrow[col] : -INFINITY;
                        return mk == -INFINITY ? -INFINITY : x + mk;
                    }
                    return col <= lim ? x : -INFINITY;
                };
                // the largest scores of this half's groups
                if (live) {
#pragma unroll
                    for (int ch = 0; ch < 2; ++ch) {
                        uint32_t s[32];
                        tc_ld_issue_x32(stm + 64 * hf + 32 * ch, s);
                        tc_wait_ld32(s);
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const float f = fk[2 * ch + g];
                            if (clear) {                         // scales are not negative
                                float t0 = __uint_as_float(s[16 * g]), t1 = __uint_as_float(s[16 * g + 1]);
#pragma unroll
                                for (int k = 2; k < 14; k += 4) {
                                    t0 = max3(t0, __uint_as_float(s[16 * g + k]), __uint_as_float(s[16 * g + k + 1]));
                                    t1 = max3(t1, __uint_as_float(s[16 * g + k + 2]), __uint_as_float(s[16 * g + k + 3]));
                                }
                                t0 = max3(t0, __uint_as_float(s[16 * g + 14]), __uint_as_float(s[16 * g + 15]));
                                topg[2 * ch + g] = fmaxf(-INFINITY, fmaxf(t0, t1) * f);      // NaN is none
                            } else {
                                float t = -INFINITY;
#pragma unroll
                                for (int k = 0; k < 16; ++k) t = fmaxf(t, score(s[16 * g + k], f, r0 + 64 * hf + 32 * ch + 16 * g + k));
                                topg[2 * ch + g] = t;
                            }
                        }
                    }
                }
                float top = fmaxf(fmaxf(topg[0], topg[1]), fmaxf(topg[2], topg[3]));
                // the largest weight, relative to m
                const auto heaviest = [&] {
                    float y = -INFINITY;
#pragma unroll
                    for (int g = 0; g < 4; ++g) y = fmaxf(y, fmaf(topg[g] - m, U, lg[g]));
                    return y;
                };
                if (bar_any(2 + qt, 256, have ? top > m + RAISE || heaviest() > d + 6.f : top > -INFINITY)) {
                    *mine = top;
                    named_bar_sync(2 + qt, 256);
                    top = fmaxf(top, *other);                    // the row's, in both its threads
                    if (have ? top > m : top > -INFINITY) {      // the weights so far stay what they are: d falls as m rises
                        const float by = have ? (m - top) * U : 0.f;
                        l *= ex2(by);
                        d += by;
                        m = top;
                        have = true;
                    }
                    named_bar_sync(2 + qt, 256);
                    float y = heaviest();
                    *mine = y;
                    named_bar_sync(2 + qt, 256);
                    y = fmaxf(y, *other);
                    float a = 1.f;
                    if (y > d + 6.f) {
                        a = ex2(d - y);
                        d = y;
                    }
                    if (__any_sync(0xffffffffu, a != 1.f)) rescale_o(a);
                }
                float sh[4];                                     // a group's log2(s_v) - d + kTop
                bool alike = true, above = true;                 // and whether 2^sh is a number that loses nothing, and 2^-sh
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    sh[g] = lg[g] - (d == -INFINITY ? 0.f : d) + kTop;
                    alike &= sh[g] < 100.f;
                    above &= sh[g] > -80.f;
                }
                const bool usual = clear && __all_sync(0xffffffffu, above);
                alike = __all_sync(0xffffffffu, alike);
                // the weights of this half
                if (live) {
#pragma unroll
                    for (int ch = 0; ch < 2; ++ch) {
                        uint32_t s[32], ph[16];
                        tc_ld_issue_x32(stm + 64 * hf + 32 * ch, s);
                        tc_wait_ld32(s);
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const float f = fk[2 * ch + g];
                            float s0 = 0.f, s1 = 0.f;
                            if (usual) {
                                // V's scales are above 0 and none is far below d: a weight is one exponential, and the sum
                                // takes it times 2^-sh
                                const float at = sh[2 * ch + g] - m;
#pragma unroll
                                for (int k = 0; k < 16; k += 2) {
                                    const float w0 = ex2(fmaf(__uint_as_float(s[16 * g + k]), f, at));
                                    const float w1 = ex2(fmaf(__uint_as_float(s[16 * g + k + 1]), f, at));
                                    s0 += w0;
                                    s1 += w1;
                                    ph[8 * g + k / 2] = pack_h2(w0, w1);
                                }
                                l = fmaf(s0 + s1, ex2(-sh[2 * ch + g]), l);
                            } else {
                                const float at = sh[2 * ch + g], wg = ex2(at);
                                const int col = r0 + 64 * hf + 32 * ch + 16 * g;
                                // a row that is not seen weighs nothing, even where its scale is NaN
                                if (alike) {
#pragma unroll
                                    for (int k = 0; k < 16; k += 2) {
                                        const float x0 = score(s[16 * g + k], f, col + k), x1 = score(s[16 * g + k + 1], f, col + k + 1);
                                        const float e0 = ex2((x0 - m) * U), e1 = ex2((x1 - m) * U);
                                        s0 += e0;
                                        s1 += e1;
                                        ph[8 * g + k / 2] = pack_h2(x0 == -INFINITY ? 0.f : e0 * wg, x1 == -INFINITY ? 0.f : e1 * wg);
                                    }
                                } else {
#pragma unroll
                                    for (int k = 0; k < 16; k += 2) {
                                        const float x0 = score(s[16 * g + k], f, col + k), x1 = score(s[16 * g + k + 1], f, col + k + 1);
                                        s0 += ex2((x0 - m) * U);
                                        s1 += ex2((x1 - m) * U);
                                        ph[8 * g + k / 2] = pack_h2(x0 == -INFINITY ? 0.f : ex2(fmaf(x0 - m, U, at)),
                                                                    x1 == -INFINITY ? 0.f : ex2(fmaf(x1 - m, U, at)));
                                    }
                                }
                                l += s0 + s1;
                            }
                        }
                        // over this half's columns that have been read
                        tc_st_32x32b_x16(stm + 64 * hf + 16 * ch, ph);
                    }
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * buf);
                ++pv;
            }
            if (!failed) failed = __any_sync(0xffffffffu, !wait_o(pv - 1));
            tc_fence_after();
            *mine = l;
            named_bar_sync(2 + qt, 256);
            l += *other;                                         // the sum of both halves
            // O 2^(d - kTop) relative to m: the output, or a partial; each half of the threads its half of the columns. The factor
            // by halves, d may pass fp32's exponents
            const float M = have ? m : -INFINITY, half = ex2(0.5f * ((d == -INFINITY ? 0.f : d) - kTop));
            float so, f = half;
            if (wk.whole()) f = out_factor<MASK>(M, l, p.sinks, hq, so) * so * half;
            const int64_t oo = (static_cast<int64_t>(b) * p.r.T + tok) * p.ldo + static_cast<int64_t>(hq) * D;
            float *po = slot_o<DP>(p.ws, QT * kRows, wk.slot(blockIdx.x)) + static_cast<int64_t>(qi) * DP;
#pragma unroll 1
            for (int ch = hf * (DP / 64); ch < (hf + 1) * (DP / 64); ++ch) {
                uint32_t v[32];
                __syncwarp();
                tc_ld_issue_x32(otm + 32 * ch, v);
                tc_wait_ld32(v);
                if (!ok) continue;
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    const int d = 32 * ch + k;
                    const float4 y = make_float4(__uint_as_float(v[k]) * half * f, __uint_as_float(v[k + 1]) * half * f,
                                                 __uint_as_float(v[k + 2]) * half * f, __uint_as_float(v[k + 3]) * half * f);
                    if (d < D) {
                        if (wk.whole()) store4<true>(p.out, oo + d, y);
                        else *reinterpret_cast<float4 *>(po + d) = y;
                    }
                }
            }
            if (ok && hf == 0 && !wk.whole()) slot_ml<DP>(p.ws, QT * kRows, G, wk.slot(blockIdx.x))[qi] = make_float2(M, l);
            tc_fence_before();
            __syncwarp();
        }
    } else if (warp < Z::soft + kDec) {
        // ============================================================ decode
        const int dt = threadIdx.x - Z::soft * 32;
        unsigned fetched = 0;                                    // bit 0, 1: the parity of thread 0's copies of K, V so far
        for (; wk.segment(p, pl); wk.next()) {
            const int row0 = wk.ua * kRows, n = wk.ub - wk.ua;
            const auto fetch = [&](int kv, int j) {              // codes of row tile j of K or V
                if (dt != 0 || j >= n || failed) return;
                const uint32_t bar = raw_full + 8 * kv;
                mbar_arrive_expect_tx(bar, Z::raw);
                tma_codes(raw + kv * Z::raw, kv ? &mapv : &mapk, row0 + j * kRows, wk.h, wk.b, bar);
                fetched ^= 1u << kv;
            };
            fetch(0, 0);
            fetch(1, 0);
            for (int j = 0; j < n; ++j, ++jt) {
                const int st = jt & 1, use = jt >> 1;
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv) {
                    const uint32_t src = raw + kv * Z::raw, dst = (kv ? vs : ks) + st * Z::tile;
                    if (!failed) failed = !mbar_wait_bounded(raw_full + 8 * kv, jt & 1, kWaitNs);
                    if (!failed && use > 0) failed = !mbar_wait_bounded((kv ? v_empty : k_empty) + 8 * st, (use - 1) & 1, kWaitNs);
#pragma unroll 4
                    for (int i = dt; i < kRows * CH; i += 32 * kDec) {
                        const int r = i / CH, ch = i % CH, odd = ch >> 2 & 1;     // odd: halves the other way round, no bank twice
                        const uint4 x = lds_v4(src + i * 16);
                        const uint32_t a = (odd ? x.z : x.x) ^ 0x80808080u, b = (odd ? x.w : x.y) ^ 0x80808080u;
                        const uint32_t e = (odd ? x.x : x.z) ^ 0x80808080u, f = (odd ? x.y : x.w) ^ 0x80808080u;
                        const uint32_t o = dst + tile_off(r, 2 * ch + odd);
                        sts_v4(o, make_uint4(h2_lo(a), h2_hi(a), h2_lo(b), h2_hi(b)));
                        sts_v4(o ^ 16, make_uint4(h2_lo(e), h2_hi(e), h2_lo(f), h2_hi(f)));
                    }
                    fence_proxy_async_smem();                    // what was stored, and that the codes have been read
                    named_bar_sync(1, 32 * kDec);
                    if (dt == 0) mbar_arrive((kv ? v_full : k_full) + 8 * st);
                    fetch(kv, j + 1);
                }
            }
        }
        if (failed && dt == 0)                                   // copies in flight, the last of each, land before the CTA ends
            for (int kv = 0; kv < 2; ++kv)
                mbar_wait_bounded(raw_full + 8 * kv, ~(fetched >> kv) & 1, kWaitNs);
    } else if (lane == 0) {
        // ============================================================ products
        auto wait = [&](uint32_t bar, uint32_t parity) {
            if (!failed && !mbar_wait_bounded(bar, parity & 1, kWaitNs)) failed = true;
            tc_fence_after();
        };
        auto qk = [&](int qt, int tile, int buf) {               // S[buf] = Q . K^T of row tile `tile`
            if (!failed) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    const uint32_t off = (kk >> 2) * kSub + (kk & 3) * 32;
                    tc_mma_f16(tmem + buf * kRows, sw128_desc(qs + qt * Z::tile + off),
                               sw128_desc(ks + (tile & 1) * Z::tile + off), kIdesc<kRows, false>, kk != 0);
                }
            }
            tc_commit(s_full + 8 * buf);                         // also after a failure: keeps the others moving
        };
        auto pvp = [&](int qt, int tile, int buf, bool more) {   // O[qt] (+)= P[buf] . V of row tile `tile`
            if (!failed) {
#pragma unroll
                for (int kk = 0; kk < kRows / 16; ++kk)          // a half's weights are over the first half of its columns
                    tc_mma_f16_ta(tmem + kO + qt * DP, tmem + buf * kRows + (kk >> 2) * 64 + (kk & 3) * 8,
                                  sw128_desc_mn(vs + (tile & 1) * Z::tile + kk * 2048, kSub), kIdesc<DP, true>,
                                  more || kk != 0);
            }
            tc_commit(o_full + 8 * (QT == 2 ? qt : tile & 1));
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
    if (failed) atomicOr(p.r.err, 1024);
    tc_fence_before();
    __syncthreads();
    if (warp == Z::soft + kDec) tmem_dealloc(tmem, 512);
}

template <int DP, int QT, bool MASK>
cudaError_t launch_t(const Kv8AttnParams &p, cudaStream_t s) {
    using Z = TileSizes<DP, QT>;
    const auto k = kv8_attn_tile_kernel<DP, QT, MASK>;
    static std::atomic<int> kept{0};
    if (!kv8_kept(kept, [&] { return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::smem) == cudaSuccess ? 1 : 0; }))
        return kv8_lookup_error();
    CUtensorMap mk, mv;
    if (!kv8_code_map(mk, p.c, p.c.k, DP, kRows, CU_TENSOR_MAP_SWIZZLE_NONE) ||
        !kv8_code_map(mv, p.c, p.c.v, DP, kRows, CU_TENSOR_MAP_SWIZZLE_NONE))
        return cudaErrorInvalidValue;
    return launch_pdl(k, dim3(kv8_sms()), dim3(Z::threads), Z::smem, s, mk, mv, p);
}
template <int DP, int QT>
cudaError_t launch_q(const Kv8AttnParams &p, cudaStream_t s) {
    return p.mask ? launch_t<DP, QT, true>(p, s) : launch_t<DP, QT, false>(p, s);
}

}  // namespace

// query tiles a CTA takes at a time: two share the decoded rows where there are more than 128 queries
int kv8_tile_queries(int64_t queries) { return queries > kRows ? 2 * kRows : kRows; }
int kv8_tile_rows() { return kRows; }
int kv8_tile_ctas() { return kv8_sms(); }

cudaError_t kv8_tile_launch(const Kv8AttnParams &p, cudaStream_t s) {
    const int64_t queries = static_cast<int64_t>(p.r.T) * (p.Hq / p.c.Hkv);
    if (kv8_tile_queries(queries) == 2 * kRows) return p.c.D <= 64 ? launch_q<64, 2>(p, s) : launch_q<128, 2>(p, s);
    return p.c.D <= 64 ? launch_q<64, 1>(p, s) : launch_q<128, 1>(p, s);
}

}  // namespace onpu_b200
