// Attention over the 8-bit KV cache (kv8.cu): query i of a sequence stands at cache row pos + i and sees rows
// 0 .. pos + i,
//   x_j = scale q . (c_j s_b(j)) + mask_j,   out = sum_j e^(x_j) v_j / (sum_j e^(x_j) + e^sink),
// with an online softmax in fp32; a query whose mask leaves no row gives zeros.
//
// The T * Hq / Hkv queries that share a kv head are the columns of the products (8 NT of them a tile), so
// each cache row is read once for all of a tile: a warp takes 16 R rows a step,
//   X[row][query] = K[row][:] . q[query][:]          m16n8k32 int8, A = 16 rows of K
//   O^T[d][query] += V^T[d][row] . P^T[row][query]   m16n8k16 fp16, A = V^T
// Which k of a product is which d or row is free, so a lane reads 16 bytes of its rows from shared memory and uses
// them as they lie; for V a lane reads the same bytes of four rows and pairs them with byte permutes, so nothing
// is transposed. K's scale multiplies the finished scores, V's the weights.
//  * q is taken as three base-256 digits of q f, f a power of two that puts the row's largest |q f| in [2^22, 2^23): 24
//    bits of the row's largest value, and sums of codes times digits that are exact. K's codes need no
//    decoding, and an int8 product has twice the k of an fp16 one at the same rate (4.4 ns a warp
//    instruction on one of an SM's four quarters, both). Against fp16 q (two parts for fp32) and decoded K, with cp.async:
//    one token over 131001 rows 65.0 -> 49.5 us, 484 warp instructions per 16 rows before.
//  * weights: w = 2^(x - m) * s_v * c, rounded to fp16 (one part for bf16 outputs: 2^-11 of a weight against the output's
//    2^-8; two parts, 22 bits, for fp32), times V's codes as fp16, exactly (|c| <= 127): 0x64uu is 1024 + uu. c is a
//    query's own: its largest weight so far stands at 2^6 or more, and is brought back to 2^6 before one could pass 2^16. What
//    it does not see or what weighs nothing does not count, however large its s_v is. Weights 2^20 below the largest (two
//    parts: 2^9) lose bits, 2^-31 of the largest at most.
//  * m is a reference within 2^6 (no mask) or e^4 (mask) of the running maximum, raised only when a score
//    passes it by more: the accumulators are rescaled a few times a sequence, not every step. With a mask
//    scores stay in natural units, x - m is formed first, so masks of the lowest finite value stay finite.
//
// Bound by HBM on the cache (2 D + 8 / block bytes a row and head) while a tile has few queries: 5.3 TB/s at 131001
// rows (0.82 of the copy bandwidth), 4.5 TB/s for 64 sequences of 100 to 8192 rows. Short calls are bound by the chain
// of one step (place in the list, TMA and queries, products, softmax, merge: 3 to 4 us) and of the join (2 us).
// The rows of all sequences, tiles and heads are one list of units of 64 R rows (from pos and cnt, on the device), cut
// evenly over one wave of CTAs whatever the lengths are; a CTA writes finished outputs for the (sequence, tile, head)
// it covers alone and a partial (reference, sum, output) for at most two it shares, which a second launch adds in CTA
// order. That one is launched while the first runs and waits only with its place in the list found.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kernels.h"
#include "kv8.cuh"
#include "ptx.cuh"

namespace onpu_b200 {
namespace {

constexpr int kWarps = 4;

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
    return d;
}
// ---------------------------------------------------------------- the split kernel
// A stage: 16 R rows of K, then of V, as TMA wrote them: rows of 64 or 128 bytes (256: two such halves one
// after the other), their 16-byte chunks exchanged by the map's swizzle.
template <int DP, int R>
constexpr int kStageBytes = 2 * 16 * R * DP;
template <int DP, int NT>
constexpr int kMergeBytes = kWarps * 8 * NT * ((DP + 4) * 4 + 8);

// byte offset of chunk c of row r in a tile of `rows` rows
template <int DP>
__device__ __forceinline__ int stage_off(int rows, int r, int c) {
    if constexpr (DP == 64) return r * 64 + ((c ^ (r >> 1 & 3)) << 4);
    else return (c >> 3) * rows * 128 + r * 128 + (((c ^ r) & 7) << 4);
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap *map, int x, int row, int head, int seq,
                                         uint32_t bar, uint64_t pol) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, "
        "%4, %5}], [%6], %7;" ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(head), "r"(seq), "r"(bar), "l"(pol)
        : "memory");
}
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8u8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// CTAs an SM that the registers are to allow; 0: the compiler's choice. For fp32 it spills to fit three: one token over 4096 rows
// 11.0 us, 9.3 with two; 64000 rows 36.1 / 29.5; 3 sequences of 1450 rows, 5 / 1 heads of 96, 10.0 / 10.9 (the join has less room beside it).
template <int DP, int NT, bool BF16>
constexpr int kMinCtas = DP == 128 && NT == 1 && !BF16 ? 2 : 0;

template <int DP, int NT, bool BF16, bool MASK, int R, int NS>
__global__ void __launch_bounds__(kWarps * 32, kMinCtas<DP, NT, BF16>)
    kv8_attn_split_kernel(const __grid_constant__ CUtensorMap mapk, const __grid_constant__ CUtensorMap mapv,
                          const Kv8AttnParams p) {
    constexpr int PARTS = BF16 ? 1 : 2;             // fp16 parts of a weight
    constexpr int KI = DP / 64;                     // 16-byte chunks of a K row per lane
    constexpr int VW = DP / 32;                     // 4-byte words of a V row per lane
    constexpr int ROWS = 16 * R, STB = kStageBytes<DP, R>;
    constexpr float U = MASK ? kLog2e : 1.f, RAISE = MASK ? 4.f : 6.f;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[kWarps * NS];
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);      // the swizzle's period
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int G = gridDim.x, D = p.c.D;
    const Kv8Cache &c = p.c;
    const uint32_t wbase = smem_u32(smem) + warp * NS * STB, bar0 = smem_u32(bars) + warp * NS * 8;
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < NS; ++s) mbar_init(bar0 + 8 * s, 1);
        mbar_init_fence();
        if (warp == 0) {                  // the maps are launch parameters: their fetch need not wait
            asm volatile("prefetch.tensormap [%0];" ::"l"(&mapk) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&mapv) : "memory");
        }
    }
    const uint64_t pol = l2_evict_first_policy();
    __syncwarp();
    pdl_wait_prerequisites();
    pdl_launch_dependents();              // after the wait: the join may read pos and cnt as it starts

    const Plan pl(p, 8 * NT, kWarps * ROWS);
    Walk wk;
    if (!wk.start(p, pl, lane, blockIdx.x, G)) return;

    bool failed = false;
    int stage = 0, filled = 0;                     // the next stage to read and its parity, the next to fill
    uint32_t parity = 0;
    // this lane's rows of a 16-row block: for V (4 of them) and, of those that lanes 4 (g / 2) .. hold, for K
    // (two). Rows 2p and (2p ^ 4) + 1 [+ 8]: in the swizzled tile the eight lanes of a phase never meet in a bank.
    const int vr0 = 2 * t, vr1 = ((2 * t) ^ 4) + 1;
    const int kp = g >> 1, ra = g & 1 ? ((2 * kp) ^ 4) + 1 : 2 * kp, rb = ra + 8;
    for (; wk.segment(p, pl); wk.next()) {
        const int b = wk.b, h = wk.h, pos = wk.pos, nq = wk.nq;
        const int64_t q0 = wk.q0;
        const int row0 = wk.ua * kWarps * ROWS;
        const int row1 = static_cast<int>(min(static_cast<int64_t>(wk.len), static_cast<int64_t>(wk.ub) * kWarps * ROWS));
        const int nstep = (row1 - row0 + ROWS - 1) / ROWS;
        const float *ksb = c.ks + b * c.sbs + h * c.shs, *vsb = c.vs + b * c.sbs + h * c.shs;

        auto issue = [&](int s) {                  // step s (every kWarps-th is this warp's) into the next stage
            if (s < nstep && !failed) {
                if (lane == 0) {
                    const uint32_t st = wbase + filled * STB, bar = bar0 + 8 * filled;
                    const int r0 = row0 + s * ROWS;
                    mbar_arrive_expect_tx(bar, STB);
#pragma unroll
                    for (int x = 0; x < DP; x += 128) {
                        tma_rows(st + x * ROWS, &mapk, x, r0, h, b, bar, pol);
                        tma_rows(st + DP * ROWS + x * ROWS, &mapv, x, r0, h, b, bar, pol);
                    }
                }
                filled = filled + 1 == NS ? 0 : filled + 1;
            }
        };
#pragma unroll
        for (int s = 0; s < NS - 1; ++s) issue(warp + s * kWarps);
        float ksc[R], vsc[R];                      // the scales of this warp's next step
        auto load_scales = [&](int s) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int r = row0 + s * ROWS + 16 * i;
                ksc[i] = r < row1 ? ksb[r >> c.blk_log2] : 0.f;
                vsc[i] = r < row1 ? vsb[r >> c.blk_log2] : 0.f;
            }
        };
        load_scales(warp);

        // q^T as B fragments of base-256 digits: q f = 2^16 d0 + 2^8 d1 + d2, d0 signed, f the power of two that puts
        // the row's largest |q f| in [2^22, 2^23). Lane t's k slots of step (i, s) are d = 16 (t + 4i) + 8s + 0 .. 7.
        uint32_t qf[3][NT][KI * 2][2];
        float rs[NT][2];
        int lim[NT][2];
        int64_t moff[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int qi = 8 * nt + g;
            const bool ok = qi < nq;
            const int tok = static_cast<int>(div64(q0 + (ok ? qi : 0), pl.rep));
            const int hq = h * pl.rep + static_cast<int>((q0 + (ok ? qi : 0)) - static_cast<int64_t>(tok) * pl.rep);
            const int64_t qo = (static_cast<int64_t>(b) * p.r.T + tok) * p.ldq + static_cast<int64_t>(hq) * D;
            float x[KI * 4][4];
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < KI; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int d = 16 * (t + 4 * i) + 4 * w;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (ok && d < D) {
                        if constexpr (BF16) {
                            const uint2 r = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p.q) + qo + d);
                            v = make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u),
                                            __uint_as_float(r.y << 16), __uint_as_float(r.y & 0xffff0000u));
                        } else {
                            v = *reinterpret_cast<const float4 *>(static_cast<const float *>(p.q) + qo + d);
                        }
                    }
                    x[i * 4 + w][0] = v.x;
                    x[i * 4 + w][1] = v.y;
                    x[i * 4 + w][2] = v.z;
                    x[i * 4 + w][3] = v.w;
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx = max_nan(mx, fabsf(x[i * 4 + w][k]));
                }
            mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float f = pow2_to(mx, 22);
#pragma unroll
            for (int s = 0; s < KI * 4; ++s) {
                uint32_t dg[3] = {0, 0, 0};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int Q = min(__float2int_rn(x[s][k] * f), 0x7fffff);     // 2^23 - 1/2 rounds up to 2^23
#pragma unroll
                    for (int j = 0; j < 3; ++j) dg[j] |= static_cast<uint32_t>(Q >> (16 - 8 * j) & 0xff) << (8 * k);
                }
#pragma unroll
                for (int j = 0; j < 3; ++j) qf[j][nt][s >> 1][s & 1] = dg[j];
            }
            // what a lane's columns 2t, 2t + 1 of the scores need; a query that is not finite has NaN scores
            const float rsg = mx < INFINITY ? p.scale * (MASK ? 1.f : kLog2e) / f : __uint_as_float(0x7fc00000u);
            const int lg = ok ? pos + tok : -1;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                rs[nt][k] = __shfl_sync(0xffffffffu, rsg, (2 * t + k) * 4);
                lim[nt][k] = __shfl_sync(0xffffffffu, lg, (2 * t + k) * 4);
                if constexpr (MASK) moff[nt][k] = b * p.mbs + __shfl_sync(0xffffffffu, tok, (2 * t + k) * 4) * p.mts;
            }
        }
        // the first row that some query of the tile must not see (queries past nq do not matter)
        const int edge = pos + static_cast<int>(div64(q0, pl.rep)) + 1;

        // cw: what the weights are times, 0 before a query's first weight
        float o[VW * 2][NT][4], m[NT][2], l[NT][2], cw[NT][2], cmax = INFINITY;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < VW * 2; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int k = 0; k < 2; ++k) cw[nt][k] = lim[nt][k] < 0 ? 0x1p-126f : 0.f;     // no query: nothing to set
        }
        float mk[R][NT][4];                                    // the mask of this warp's next step
        auto load_mask = [&](int s) {
            if constexpr (MASK) {
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int j = row0 + s * ROWS + 16 * i + (k & 2 ? rb : ra);
                            mk[i][nt][k] = s < nstep && j <= lim[nt][k & 1] ? p.mask[moff[nt][k & 1] + j] : -INFINITY;
                        }
            }
        };
        load_mask(warp);
        for (int s = warp; s < nstep && !failed; s += kWarps) {
            __syncwarp();                                      // every lane is past its reads of the stage refilled here
            issue(s + (NS - 1) * kWarps);
            failed = __any_sync(0xffffffffu, !mbar_wait_bounded(bar0 + 8 * stage, parity, kWaitNs));
            if (failed) {                                      // no more steps; the copies in flight, this one first, once more
                do {
                    mbar_wait_bounded(bar0 + 8 * stage, parity, kWaitNs);
                    stage = stage + 1 == NS ? 0 : stage + 1;
                    parity ^= stage == 0;
                } while (stage != filled);
                break;
            }
            const uint32_t kb = wbase + stage * STB, vb = kb + DP * ROWS;
            stage = stage + 1 == NS ? 0 : stage + 1;
            parity ^= stage == 0;
            const int r0 = row0 + s * ROWS;
            float x[R][NT][4], sv[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                int acc[3][NT][4];
#pragma unroll
                for (int j = 0; j < 3; ++j)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) acc[j][nt][0] = acc[j][nt][1] = acc[j][nt][2] = acc[j][nt][3] = 0;
#pragma unroll
                for (int k = 0; k < KI; ++k) {
                    const uint4 va = lds_v4(kb + stage_off<DP>(ROWS, 16 * i + ra, t + 4 * k));
                    const uint4 vv = lds_v4(kb + stage_off<DP>(ROWS, 16 * i + rb, t + 4 * k));
                    const uint32_t a[2][4] = {{va.x, vv.x, va.y, vv.y}, {va.z, vv.z, va.w, vv.w}};
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_s8(acc[0][nt], a[w], qf[0][nt][k * 2 + w][0], qf[0][nt][k * 2 + w][1]);
                            mma_s8u8(acc[1][nt], a[w], qf[1][nt][k * 2 + w][0], qf[1][nt][k * 2 + w][1]);
                            mma_s8u8(acc[2][nt], a[w], qf[2][nt][k * 2 + w][0], qf[2][nt][k * 2 + w][1]);
                        }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float f[2] = {ksc[i] * rs[nt][0], ksc[i] * rs[nt][1]};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {              // |acc[0] 2^8 + acc[1]| < 2^31
                        const float a = fmaf(static_cast<float>(acc[0][nt][k] * 256 + acc[1][nt][k]), 256.f,
                                             static_cast<float>(acc[2][nt][k]));
                        x[i][nt][k] = a * f[k & 1];
                        if constexpr (MASK)
                            x[i][nt][k] = mk[i][nt][k] == -INFINITY ? -INFINITY : x[i][nt][k] + mk[i][nt][k];
                    }
                }
                sv[i] = vsc[i];
            }
            load_scales(s + kWarps);
            load_mask(s + kWarps);
            if (!MASK && r0 + ROWS > edge) {                   // MASK: load_mask gave -inf beyond the limits
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (r0 + 16 * i + (k & 2 ? rb : ra) > lim[nt][k & 1]) x[i][nt][k] = -INFINITY;
            }
            bool up = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float mx = fmaxf(x[0][nt][k], x[0][nt][k + 2]);
#pragma unroll
                    for (int i = 1; i < R; ++i) mx = fmaxf(mx, fmaxf(x[i][nt][k], x[i][nt][k + 2]));
                    up |= mx > m[nt][k] + RAISE;
                }
            float svm = sv[0];
#pragma unroll
            for (int i = 1; i < R; ++i) svm = fmaxf(svm, sv[i]);
            // m and the weights' factors: looked at where a score passes m, where a weight might pass fp16's range, and while a
            // query has had no weight (cmax is inf then)
            if (__any_sync(0xffffffffu, up) || svm * cmax > 1000.f || cmax == INFINITY) {
                cmax = 0.f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float top[R], mn = m[nt][k];           // the largest score of each 16 rows
#pragma unroll
                        for (int i = 0; i < R; ++i) {
                            top[i] = fmaxf(x[i][nt][k], x[i][nt][k + 2]);
                            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 4));
                            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 8));
                            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 16));
                            mn = fmaxf(mn, top[i]);
                        }
                        float wm = 0.f;                        // the step's largest weight; rows that are not seen have none
#pragma unroll
                        for (int i = 0; i < R; ++i)
                            if (top[i] != -INFINITY) wm = fmaxf(wm, ex2((top[i] - mn) * U) * sv[i]);
                        const float by = mn == -INFINITY ? 0.f : (m[nt][k] - mn) * U, c0 = cw[nt][k];
                        m[nt][k] = mn;
                        l[nt][k] *= ex2(by);
                        // m raised, the weights so far stay what they are times a larger factor; o changes with them only where
                        // the new ones need a smaller one
                        float cn = c0 > 0.f ? fminf(c0 * ex2(-by), 0x1p126f) : 0.f;
                        const bool over = wm * cn > 1000.f;
                        if (over || (c0 == 0.f && wm > 0.f)) cn = pow2_to(wm, 6);
                        if (c0 > 0.f && (over || cn == 0x1p126f)) {        // o 2^by cn / c0, cn a power of two
                            const int d = static_cast<int>(__float_as_uint(cn) >> 23) - static_cast<int>(__float_as_uint(c0) >> 23);
                            const float a = __fdividef(ex2(by + d), __uint_as_float((__float_as_uint(c0) & 0x7fffffu) | 0x3f800000u));
#pragma unroll
                            for (int i = 0; i < VW * 2; ++i) {
                                o[i][nt][k] *= a;
                                o[i][nt][k + 2] *= a;
                            }
                        }
                        cw[nt][k] = cn;
                        cmax = fmaxf(cmax, cn == 0.f ? INFINITY : cn);
                    }
                cmax = fmaxf(cmax, __shfl_xor_sync(0xffffffffu, cmax, 1));
                cmax = fmaxf(cmax, __shfl_xor_sync(0xffffffffu, cmax, 2));
            }
            uint32_t pb[R][PARTS][NT][2];
#pragma unroll
            for (int i = 0; i < R; ++i) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float mr = m[nt][k & 1] == -INFINITY ? 0.f : m[nt][k & 1];
                        const float e2 = ex2((x[i][nt][k] - mr) * U);
                        l[nt][k & 1] += e2;
                        w[k] = e2 * sv[i] * cw[nt][k & 1];     // in this order: a large scale that hardly weighs stays finite
                        // a row that is not seen weighs nothing, even where its scale is NaN
                        if (x[i][nt][k] == -INFINITY) w[k] = 0.f;
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t hi = pack_h2(w[2 * k], w[2 * k + 1]);
                        pb[i][0][nt][k] = movmatrix_trans(hi);
                        if constexpr (PARTS == 2) {
                            const float2 r = unpack_h2(hi);
                            pb[i][PARTS - 1][nt][k] = movmatrix_trans(pack_h2(w[2 * k] - r.x, w[2 * k + 1] - r.y));
                        }
                    }
                }
            }
            // V: this lane's words of its four rows, MMA rows (2t, 2t + 1 | 2t + 8, 2t + 9) of the weights
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int v = 0; v < (DP == 256 ? 2 : 1); ++v) {
                    uint32_t wd[4][DP == 64 ? 2 : 4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = 16 * i + (r & 1 ? vr1 : vr0) + (r & 2 ? 8 : 0);
                        if constexpr (DP == 64) {
                            const uint2 q2 = lds_v2(vb + stage_off<DP>(ROWS, row, g >> 1) + (g & 1) * 8);
                            wd[r][0] = q2.x;
                            wd[r][1] = q2.y;
                        } else {
                            const uint4 q4 = lds_v4(vb + stage_off<DP>(ROWS, row, g + 8 * v));
                            wd[r][0] = q4.x;
                            wd[r][1] = q4.y;
                            wd[r][2] = q4.z;
                            wd[r][3] = q4.w;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < (DP == 64 ? 2 : 4); ++w) {
                        uint32_t y[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) y[r] = wd[r][w] ^ 0x80808080u;
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {       // d = 4w + 2 hf + (0, 1)
                            const uint32_t r01 = prmt(y[0], y[1], hf ? 0x7362u : 0x5140u);
                            const uint32_t r23 = prmt(y[2], y[3], hf ? 0x7362u : 0x5140u);
                            const uint32_t a0 = h2_lo(r01), a1 = h2_hi(r01), a2 = h2_lo(r23), a3 = h2_hi(r23);
                            if constexpr (PARTS == 1) {
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
                                    mma_f16(o[(v * 4 + w) * 2 + hf][nt], a0, a1, a2, a3, pb[i][0][nt][0], pb[i][0][nt][1]);
                            } else {
                                // the tensor core cuts its sums off (towards 0), which adds up over a long run of rows: the
                                // two products of 16 rows on their own, added in fp32 (64 sequences of 16k rows: 4.2e-6 of
                                // the result's norm off without, 3.5e-7 with)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                    for (int pt = PARTS - 1; pt >= 0; --pt)
                                        mma_f16(t, a0, a1, a2, a3, pb[i][pt][nt][0], pb[i][pt][nt][1]);
#pragma unroll
                                    for (int k = 0; k < 4; ++k) o[(v * 4 + w) * 2 + hf][nt][k] += t[k];
                                }
                            }
                        }
                    }
                }
        }
        // merge the warps in shared memory: every copy has been waited for
        __syncthreads();
        float *osm = reinterpret_cast<float *>(smem);                              // [warps][8 NT][DP + 4]
        float2 *msm = reinterpret_cast<float2 *>(osm + kWarps * 8 * NT * (DP + 4));    // [warps][8 NT] reference, sum
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float inv = cw[nt][k] == 0.f ? 1.f : __fdividef(1.f, cw[nt][k]);
                float s = l[nt][k];
                s += __shfl_xor_sync(0xffffffffu, s, 4);
                s += __shfl_xor_sync(0xffffffffu, s, 8);
                s += __shfl_xor_sync(0xffffffffu, s, 16);
                const int q = warp * 8 * NT + 8 * nt + 2 * t + k;
                if (g == 0) msm[q] = make_float2(m[nt][k], s);
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    const int d = DP == 64 ? 8 * g + 4 * w : 128 * (w >> 2) + 16 * g + 4 * (w & 3);
                    *reinterpret_cast<float4 *>(osm + q * (DP + 4) + d) =
                        make_float4(o[2 * w][nt][k] * inv, o[2 * w][nt][k + 2] * inv, o[2 * w + 1][nt][k] * inv,
                                    o[2 * w + 1][nt][k + 2] * inv);
                }
            }
        __syncthreads();
        const bool whole = wk.whole();
        const int slot = wk.slot(blockIdx.x);
        const int dv = D >> 2;
        for (int i = threadIdx.x; i < nq * dv; i += kWarps * 32) {
            const int q = i / dv, d = (i - q * dv) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, msm[w * 8 * NT + q].x);
            const float ref = M == -INFINITY ? 0.f : M;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            float L = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 ml = msm[w * 8 * NT + q];
                const float f = ex2((ml.x - ref) * U);
                const float4 v = *reinterpret_cast<const float4 *>(osm + (w * 8 * NT + q) * (DP + 4) + d);
                L = fmaf(ml.y, f, L);
                y.x = fmaf(v.x, f, y.x);
                y.y = fmaf(v.y, f, y.y);
                y.z = fmaf(v.z, f, y.z);
                y.w = fmaf(v.w, f, y.w);
            }
            if (whole) {
                const int tok = static_cast<int>(div64(q0 + q, pl.rep));
                const int hq = h * pl.rep + static_cast<int>(q0 + q - static_cast<int64_t>(tok) * pl.rep);
                float so;
                const float f = out_factor<MASK>(M, L, p.sinks, hq, so) * so;
                store4<BF16>(p.out, (static_cast<int64_t>(b) * p.r.T + tok) * p.ldo + static_cast<int64_t>(hq) * D + d,
                             make_float4(y.x * f, y.y * f, y.z * f, y.w * f));
            } else {
                *reinterpret_cast<float4 *>(slot_o<DP>(p.ws, 8 * NT, slot) + q * DP + d) = y;
                if (d == 0) slot_ml<DP>(p.ws, 8 * NT, G, slot)[q] = make_float2(M, L);
            }
        }
        fence_proxy_async_smem();
        __syncthreads();                                       // before the stages are filled again
    }
    if (failed && lane == 0) atomicOr(p.r.err, 1024);
}

// ---------------------------------------------------------------- the shared segments
// One CTA per query: where several CTAs of the split kernel hold a part of its rows, adds their partials
// in order (each warp every kJoinWarps-th part, four values a lane, so up to 4 kJoinWarps parts are in flight at
// once). The list is read before the split kernel is done (that one starts after everything before it).
constexpr int kJoinWarps = 8;

template <int DP, bool BF16, bool MASK>
__global__ void __launch_bounds__(kJoinWarps * 32) kv8_attn_join_kernel(const Kv8AttnParams p, int G, int tile, int unit) {
    constexpr float U = MASK ? kLog2e : 1.f;
    constexpr int V = DP == 256 ? 2 : 1;
    __shared__ float red[kJoinWarps];
    __shared__ float4 acc[kJoinWarps][DP / 4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.c.D;
    const Plan pl(p, tile, unit);
    const int eh = blockIdx.x / tile, q = blockIdx.x - eh * tile, e = eh / p.c.Hkv, h = eh - e * p.c.Hkv;
    const Shares sh(p, pl, lane, e, h, G);
    const int64_t qr = sh.q0 + q;
    const int i0 = sh.i0, i1 = qr < static_cast<int64_t>(sh.cnt) * pl.rep ? sh.i1 : i0, b = sh.b;
    const auto slot = [&](int i) { return sh.slot(i); };
    const int tok = static_cast<int>(div64(qr, pl.rep)), hq = h * pl.rep + static_cast<int>(qr - static_cast<int64_t>(tok) * pl.rep);
    pdl_wait_prerequisites();
    pdl_launch_dependents();
    if (i0 == i1) return;                                      // one CTA had it all and wrote the output
    float M = -INFINITY;
    for (int i = i0 + lane; i <= i1; i += 32) M = fmaxf(M, slot_ml<DP>(p.ws, tile, G, slot(i))[q].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 y[V];
#pragma unroll
    for (auto &v : y) v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = i0 + warp; i <= i1; i += kJoinWarps) {
        const int s = slot(i);
        const float2 ml = slot_ml<DP>(p.ws, tile, G, s)[q];
        const float f = ex2((ml.x - ref) * U);
        L = fmaf(ml.y, f, L);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int d = 128 * k + 4 * lane;
            if (d < D) {
                const float4 v = *reinterpret_cast<const float4 *>(slot_o<DP>(p.ws, tile, s) + q * DP + d);
                y[k].x = fmaf(v.x, f, y[k].x);
                y[k].y = fmaf(v.y, f, y[k].y);
                y[k].z = fmaf(v.z, f, y[k].z);
                y[k].w = fmaf(v.w, f, y[k].w);
            }
        }
    }
    if (lane == 0) red[warp] = L;
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (32 * k + lane < DP / 4) acc[warp][32 * k + lane] = y[k];
    __syncthreads();
    const int d = 4 * threadIdx.x;
    if (d < D) {
        L = red[0];
        float4 s = acc[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < kJoinWarps; ++w) {
            const float4 v = acc[w][threadIdx.x];
            L += red[w];
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
        float so;
        const float f = out_factor<MASK>(M, L, p.sinks, hq, so) * so;
        store4<BF16>(p.out, (static_cast<int64_t>(b) * p.r.T + tok) * p.ldo + static_cast<int64_t>(hq) * D + d,
                     make_float4(s.x * f, s.y * f, s.z * f, s.w * f));
    }
}

// The same where a segment has few parts: up to kJoinRows queries of a tile a CTA, a warp at a time on each of its
// share (a CTA for each query took 161 us of a 512-token chunk's 450). Of more segments than the split kernel has CTAs at most
// one is shared over each border between two of them, so CTAs are for borders then (BORDERS): each goes through the list once, where
// a CTA for every segment did so as the square of their number. The whole call, by segments / by borders: one token of 4096
// sequences of up to 100 rows 1282 / 335 us, of 512 of up to 1000 rows 120 / 109; 2048 fp32 tokens of 8 sequences 26.4 / 7.9 ms.
constexpr int kJoinRows = 32;

template <int DP, bool BF16, bool MASK, bool BORDERS>
__global__ void __launch_bounds__(kJoinWarps * 32) kv8_attn_join_rows_kernel(const Kv8AttnParams p, int G, int tile, int unit) {
    constexpr float U = MASK ? kLog2e : 1.f;
    constexpr int V = DP == 256 ? 2 : 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.c.D, rows = min(tile, kJoinRows), groups = tile / rows;
    const Plan pl(p, tile, unit);
    const int at = blockIdx.x / groups, qg = (blockIdx.x - at * groups) * rows;
    const Shares sh = [&] {
        if constexpr (BORDERS) return Shares(p, pl, at, G, std::integral_constant<int, kJoinWarps * 32>{});
        else return Shares(p, pl, lane, at / p.c.Hkv, at % p.c.Hkv, G);
    }();
    const int h = sh.h;
    pdl_wait_prerequisites();
    pdl_launch_dependents();
    if (sh.i0 == sh.i1) return;                                // one CTA had it all and wrote the outputs
    const int last = static_cast<int>(min(static_cast<int64_t>(qg + rows), static_cast<int64_t>(sh.cnt) * pl.rep - sh.q0));
#pragma unroll 2
    for (int q = qg + warp; q < last; q += kJoinWarps) {
        float M = -INFINITY;
        for (int i = sh.i0 + lane; i <= sh.i1; i += 32) M = fmaxf(M, slot_ml<DP>(p.ws, tile, G, sh.slot(i))[q].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float ref = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 y[V];
#pragma unroll
        for (auto &v : y) v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = sh.i0; i <= sh.i1; ++i) {
            const int s = sh.slot(i);
            const float2 ml = slot_ml<DP>(p.ws, tile, G, s)[q];
            const float f = ex2((ml.x - ref) * U);
            L = fmaf(ml.y, f, L);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int d = 128 * k + 4 * lane;
                if (d < D) {
                    const float4 v = *reinterpret_cast<const float4 *>(slot_o<DP>(p.ws, tile, s) + static_cast<int64_t>(q) * DP + d);
                    y[k].x = fmaf(v.x, f, y[k].x);
                    y[k].y = fmaf(v.y, f, y[k].y);
                    y[k].z = fmaf(v.z, f, y[k].z);
                    y[k].w = fmaf(v.w, f, y[k].w);
                }
            }
        }
        const int64_t qr = sh.q0 + q;
        const int tok = static_cast<int>(div64(qr, pl.rep)), hq = h * pl.rep + static_cast<int>(qr - static_cast<int64_t>(tok) * pl.rep);
        float so;
        const float f = out_factor<MASK>(M, L, p.sinks, hq, so) * so;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int d = 128 * k + 4 * lane;
            if (d < D)
                store4<BF16>(p.out, (static_cast<int64_t>(sh.b) * p.r.T + tok) * p.ldo + static_cast<int64_t>(hq) * D + d,
                             make_float4(y[k].x * f, y[k].y * f, y[k].z * f, y[k].w * f));
        }
    }
}

// ---------------------------------------------------------------- host side
// Query tiles: 8 NT queries; larger ones share the decoded codes and are limited by registers (the queries'
// digits take 3 DP / 16 * NT, the outputs DP / 4 * NT of them).
int pick_nt(int DP, int64_t queries) {
    return queries <= 8 || DP == 256 ? 1 : 2;
}
// More queries a kv head than this go to 128-query tiles (kv8_tile.cu), where heads fit them and they are bf16 (the tiles'
// sums over rows stay in the tensor core, which cuts them off: 7.4e-6 off after 16k rows, too much for fp32). us, tiles / this kernel,
// at 40, 72, 96, 128 queries (bf16, 8 heads of 128): one sequence of 700 rows 16 / 13, 18 / 16, 19 / 18, 21 / 19, of 16000 rows
// 34 / 33, 36 / 43, 39 / 53, 43 / 66; 8 sequences of 2250 rows 39 / 36, 41 / 53, 43 / 60, 46 / 76. Of 2 heads: one sequence of
// 700 rows 12 / 11, 13 / 11, 15 / 11, 16 / 12, of 16000 rows 24 / 22, 26 / 20, 28 / 26, 31 / 28, of 64000 rows 33 / 35, 35 / 44, 37 / 49,
// 40 / 60. What decides is the rows of all sequences and heads, which the host does not know; the few microseconds that
// short calls lose are less than what long ones would.
constexpr int kTileFrom = 64;
bool use_tiles(int D, int64_t queries, bool bf16) { return bf16 && D <= 128 && queries > kTileFrom; }
int padded_dim(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// after a split kernel of G CTAs over units of `unit` rows and tiles of `tile` queries
template <int DP, bool BF16, bool MASK>
cudaError_t join_launch(const Kv8AttnParams &p, int G, int tile, int unit, cudaStream_t s) {
    const int64_t tiles = (static_cast<int64_t>(p.r.T) * (p.Hq / p.c.Hkv) + tile - 1) / tile;
    // with a quarter as many segments as CTAs or more a segment has about five parts at most; with fewer, a whole CTA adds
    // one query's. One token of 64 sequences (256 segments): 51.9 us by rows, 58.1 by queries; one sequence of 131001 rows
    // (8 segments, 55 parts each): 56.8 by rows, 49.4 by queries.
    const int64_t segments = tiles * p.c.B * p.c.Hkv;
    const bool by_rows = segments * 4 >= G, borders = segments > G - 1;
    const int64_t joins = borders ? static_cast<int64_t>(G - 1) * (tile / std::min(tile, kJoinRows))
                                  : segments * (by_rows ? tile / std::min(tile, kJoinRows) : tile);
    if (joins == 0) return cudaSuccess;
    const auto k = borders   ? kv8_attn_join_rows_kernel<DP, BF16, MASK, true>
                   : by_rows ? kv8_attn_join_rows_kernel<DP, BF16, MASK, false>
                             : kv8_attn_join_kernel<DP, BF16, MASK>;
    return launch_pdl(k, dim3(static_cast<unsigned>(joins)), dim3(kJoinWarps * 32), 0, s, p, G, tile, unit);
}

template <int DP, int NT, bool BF16, bool MASK>
struct Split {
    // rows a warp takes in a step, stages: 12 warps per SM (the registers' limit for small tiles) x 2 x 8 KB
    static constexpr int R = DP == 256 ? 1 : 2, NS = R == 1 ? 3 : 2;
    static constexpr int ring = kWarps * NS * kStageBytes<DP, R>, merge = kMergeBytes<DP, NT>;
    static constexpr int smem = 1024 + (ring > merge ? ring : merge);
    static int ctas() {                                        // one resident wave; 0: the lookup failed
        static std::atomic<int> kept{0};
        return kv8_kept(kept, [] {
            auto k = kv8_attn_split_kernel<DP, NT, BF16, MASK, R, NS>;
            int per = 0;
            if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
                cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, k, kWarps * 32, smem) != cudaSuccess)
                return 0;
            return per * kv8_sms();
        });
    }
    static cudaError_t launch(const Kv8AttnParams &p, cudaStream_t s) {
        const int G = ctas(), rep = p.Hq / p.c.Hkv;
        if (G < 1) return kv8_lookup_error();
        const int64_t tiles = (static_cast<int64_t>(p.r.T) * rep + 8 * NT - 1) / (8 * NT);
        if (tiles * p.c.B > 0x7fffffff) return cudaErrorInvalidConfiguration;
        CUtensorMap mk, mv;
        const auto swz = DP == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
        if (!kv8_code_map(mk, p.c, p.c.k, DP, 16 * R, swz) || !kv8_code_map(mv, p.c, p.c.v, DP, 16 * R, swz))
            return cudaErrorInvalidValue;
        const cudaError_t e = launch_pdl(kv8_attn_split_kernel<DP, NT, BF16, MASK, R, NS>, dim3(G), dim3(kWarps * 32), smem, s,
                                         mk, mv, p);
        if (e != cudaSuccess) return e;
        return join_launch<DP, BF16, MASK>(p, G, 8 * NT, kWarps * 16 * R, s);
    }
};

// f(Split<...>) for the call's sizes and types
template <int DP, bool BF16, bool MASK, typename F>
auto with_nt(int nt, F f) {
    if constexpr (DP != 256) {
        if (nt == 2) return f(Split<DP, 2, BF16, MASK>{});
    }
    return f(Split<DP, 1, BF16, MASK>{});
}
template <int DP, typename F>
auto with_types(int nt, bool bf16, bool mask, F f) {
    if (bf16) return mask ? with_nt<DP, true, true>(nt, f) : with_nt<DP, true, false>(nt, f);
    return mask ? with_nt<DP, false, true>(nt, f) : with_nt<DP, false, false>(nt, f);
}
template <typename F>
auto with_split(int D, int64_t queries, bool bf16, bool mask, F f) {
    const int DP = padded_dim(D), nt = pick_nt(DP, queries);
    return DP == 64    ? with_types<64>(nt, bf16, mask, f)
           : DP == 128 ? with_types<128>(nt, bf16, mask, f)
                       : with_types<256>(nt, bf16, mask, f);
}

}  // namespace

int64_t kv8_attn_ws_bytes(int Hq, int Hkv, int D, int T, bool bf16) {
    const int64_t queries = static_cast<int64_t>(T) * (Hq / Hkv);
    const int DP = padded_dim(D);
    int64_t G = 0, tile = 8 * pick_nt(DP, queries);
    if (use_tiles(D, queries, bf16)) {
        G = kv8_tile_ctas();
        tile = kv8_tile_queries(queries);
        if (G < 1) return -1;
    } else {
        for (const bool mask : {false, true}) {
            const int64_t g = with_split(D, queries, bf16, mask, [](auto k) { return static_cast<int64_t>(k.ctas()); });
            if (g < 1) return -1;
            G = g > G ? g : G;
        }
    }
    return 2 * G * tile * (DP + 2) * 4;
}

cudaError_t kv8_attn_launch(const Kv8AttnParams &p, bool bf16, cudaStream_t s) {
    const int64_t queries = static_cast<int64_t>(p.r.T) * (p.Hq / p.c.Hkv);
    if (!use_tiles(p.c.D, queries, bf16))
        return with_split(p.c.D, queries, bf16, p.mask != nullptr, [&](auto k) { return k.launch(p, s); });
    const int G = kv8_tile_ctas(), tile = kv8_tile_queries(queries), unit = kv8_tile_rows();
    if (G < 1) return kv8_lookup_error();
    if ((queries + tile - 1) / tile * p.c.B > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const cudaError_t e = kv8_tile_launch(p, s);
    if (e != cudaSuccess) return e;
    const auto join = [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        return p.mask ? join_launch<DP, true, true>(p, G, tile, unit, s) : join_launch<DP, true, false>(p, G, tile, unit, s);
    };
    return p.c.D <= 64 ? join(std::integral_constant<int, 64>{}) : join(std::integral_constant<int, 128>{});
}

}  // namespace onpu_b200
