// Attention over the 8-bit KV cache (kv8.cu): query i of a sequence stands at cache row pos + i and sees rows
// 0 .. pos + i,
//   x_j = scale q . (c_j s_b(j)) + mask_j,   out = sum_j e^(x_j) v_j / (sum_j e^(x_j) + e^sink),
// with an online softmax in fp32; a query whose mask leaves no row gives zeros.
//
// The T * Hq / Hkv queries that share a kv head are the columns of the products (8 NT of them a tile), so
// each cache row is read once for all of a tile: a warp takes 16 rows a step,
//   X[row][query] = K[row][:] . q[query][:]       mma m16n8k16, A = 16 rows of K
//   O^T[d][query] += V^T[d][row] . P^T[row][query]   A = V^T
// The codes become fp16 exactly (|c| <= 127). Which k of the product is which d is free, so a lane reads 16
// bytes of its rows from shared memory and uses them as they lie; for V a lane reads the same bytes of
// four rows and pairs them with byte permutes, so nothing is transposed. K's scale multiplies the finished
// scores, V's the weights.
//  * q is scaled by a power of two to [256, 512) and rounded to fp16: exact for bf16 but for values 2^-22
//    below the row's largest, and two fp16 parts (22 bits) for fp32 calls.
//  * weights: w = 2^(x - m) * s_v * c, c a power of two that keeps s_v * c in [2^7, 2^9], rounded to fp16 (one
//    part for bf16 outputs: 2^-11 of a weight against the output's 2^-8; two parts, 22 bits, for fp32).
//  * m is a reference within 2^6 (no mask) or e^4 (mask) of the running maximum, raised only when a score
//    passes it by more: the accumulators are rescaled a few times a sequence, not every step. With a mask
//    scores stay in natural units, x - m is formed first, so masks of the lowest finite value stay finite.
//
// Bound by HBM on the cache (2 D + 8 / block bytes a row and head) while a tile has few queries. The rows
// of all sequences, tiles and heads are one list of 64-row units (from pos and cnt, on the device), cut
// evenly over one wave of CTAs whatever the lengths are; a CTA writes finished outputs for the
// (sequence, tile, head) it covers alone and a partial (reference, sum, output) for at most two it shares, which a second launch
// adds in CTA order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "kernels.h"
#include "kv8.cuh"
#include "ptx.cuh"

namespace onpu_b200 {
namespace {

constexpr int kWarps = 4, kStep = 16, kUnit = kWarps * kStep;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}
// two biased codes u = c + 128 in bytes (lo: 0 and 1, hi: 2 and 3 of x) -> fp16 pair c: 0x64uu is 1024 + u
__device__ __forceinline__ uint32_t h2_lo(uint32_t x) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(prmt(x, 0x64646464u, 0x4140u)), "r"(0x64806480u));
    return d;
}
__device__ __forceinline__ uint32_t h2_hi(uint32_t x) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(prmt(x, 0x64646464u, 0x4342u)), "r"(0x64806480u));
    return d;
}
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
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t x) { return __half22float2(*reinterpret_cast<__half2 *>(&x)); }
// 2^(top - exponent of x), its exponent kept within +-100: x times it is in [2^top, 2^(top + 1)); 1 for 0, inf and NaN
__device__ __forceinline__ float pow2_to(float x, int top) {
    const int e = static_cast<int>(__float_as_uint(x) >> 23 & 0xff);
    if (e == 255 || !(fabsf(x) > 0.f)) return 1.f;
    return __uint_as_float(static_cast<uint32_t>(127 + min(100, max(-100, top + 127 - e))) << 23);
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---------------------------------------------------------------- the list of units
// An entry is a (sequence, query tile); its rows are counted in 64-row units, once per kv head.
struct Plan {
    int rep, tile, tiles, entries;    // query heads per kv head, queries a tile, tiles a sequence, B * tiles
    __device__ __forceinline__ Plan(const Kv8AttnParams &p, int tile_) {
        rep = p.Hq / p.c.Hkv;
        tile = tile_;
        tiles = static_cast<int>((static_cast<int64_t>(p.r.T) * rep + tile - 1) / tile);
        entries = p.c.B * tiles;
    }
    // rows that entry e's tile sees (0: nothing of it is valid)
    __device__ __forceinline__ int rows(const Kv8AttnParams &p, int e, int &pos, int &cnt) const {
        const int b = e / tiles;
        if (!kv8_rows(p.r, b, p.c.S, pos, cnt)) return 0;
        const int64_t r0 = static_cast<int64_t>(e - b * tiles) * tile;
        const int first = static_cast<int>(r0 / rep), last = static_cast<int>((r0 + tile - 1) / rep);
        if (first >= cnt) return 0;
        return pos + min(last, cnt - 1) + 1;
    }
    __device__ __forceinline__ int units(const Kv8AttnParams &p, int e) const {
        int pos, cnt;
        return static_cast<int>((static_cast<int64_t>(rows(p, e, pos, cnt)) + kUnit - 1) / kUnit);
    }
};
__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// units of all entries and heads (every lane of the warp gets it)
__device__ __forceinline__ int64_t total_units(const Kv8AttnParams &p, const Plan &pl, int lane) {
    int64_t n = 0;
    for (int e = lane; e < pl.entries; e += 32) n += pl.units(p, e);
    return warp_sum64(n) * p.c.Hkv;
}
// CTA i of W takes units [cta_first(i), cta_first(i + 1)), at least one each: W = min(grid, N)
__device__ __forceinline__ int64_t cta_first(int64_t N, int cta, int W) { return N * cta / W; }
__device__ __forceinline__ int cta_of(int64_t N, int64_t u, int W) { return static_cast<int>(((u + 1) * W - 1) / N); }

// ws: per CTA two slots of [tile][DP] outputs, then per slot [tile] (reference, sum) pairs
template <int DP>
__device__ __forceinline__ float *slot_o(void *ws, int tile, int slot) {
    return static_cast<float *>(ws) + static_cast<int64_t>(slot) * tile * DP;
}
template <int DP>
__device__ __forceinline__ float2 *slot_ml(void *ws, int tile, int G, int slot) {
    return reinterpret_cast<float2 *>(static_cast<float *>(ws) + static_cast<int64_t>(2) * G * tile * DP) +
           static_cast<int64_t>(slot) * tile;
}

template <bool BF16>
__device__ __forceinline__ void store4(void *out, int64_t o, float4 y) {
    if constexpr (BF16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y), b = __floats2bfloat162_rn(y.z, y.w);
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(out) + o) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {
        *reinterpret_cast<float4 *>(static_cast<float *>(out) + o) = y;
    }
}
// sums -> outputs: divide by the sum and the sink's share, zeros where nothing is left
template <bool MASK>
__device__ __forceinline__ float out_factor(float M, float Lsum, const float *sinks, int hq, float &scale_o) {
    // returns 1 / total and, in scale_o, the factor that takes sums relative to M onto the common reference
    float total = Lsum;
    scale_o = 1.f;
    if (sinks) {
        const float sk = MASK ? sinks[hq] : sinks[hq] * kLog2e, U = MASK ? kLog2e : 1.f;
        const float top = fmaxf(M, sk), ref = top == -INFINITY ? 0.f : top;
        scale_o = ex2((M - ref) * U);
        total = Lsum * scale_o + ex2((sk - ref) * U);
    }
    return total == 0.f ? 0.f : 1.f / total;
}

// ---------------------------------------------------------------- the split kernel
template <int DP>
constexpr int kStageBytes = 2 * kStep * DP + 16;              // 16 rows of K and V, their two scales
template <int DP, int NT>
constexpr int kMergeBytes = kWarps * 8 * NT * ((DP + 4) * 4 + 8);

// byte offset of 16-byte chunk c of row r (of 16) in a staged tile: chunks are exchanged so that neither the
// eight-lane phases of the K reads (rows r, r + 1, four chunks) nor those of the V reads (rows 4 apart, one
// or two chunks) meet in a bank
template <int DP>
__device__ __forceinline__ int stage_off(int r, int c) {
    if constexpr (DP == 64) return r * DP + ((c ^ (r >> 2 & 3)) << 4);
    else return r * DP + ((c ^ (((r ^ (r >> 3)) & 1) << 2 | (r >> 2 & 1) << 1)) << 4);
}

template <int DP, int NT, bool BF16, bool MASK, int NS>
__global__ void __launch_bounds__(kWarps * 32) kv8_attn_split_kernel(const Kv8AttnParams p) {
    constexpr int PARTS = BF16 ? 1 : 2;
    constexpr int KI = DP / 64;                     // 16-byte chunks of a K row per lane
    constexpr int VW = DP / 32;                     // 4-byte words of a V row per lane
    constexpr int CH = DP / 16;                     // chunks per row
    constexpr int STB = kStageBytes<DP>;
    constexpr float U = MASK ? kLog2e : 1.f, RAISE = MASK ? 4.f : 6.f;
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int G = gridDim.x, D = p.c.D, nch = D >> 4;
    const Kv8Cache &c = p.c;
    uint8_t *wbuf = smem + warp * NS * STB;
    const uint32_t wbase = smem_u32(wbuf);
    pdl_wait_prerequisites();

    const Plan pl(p, 8 * NT);
    const int64_t N = total_units(p, pl, lane);
    const int W = static_cast<int>(min(N, static_cast<int64_t>(G)));
    if (static_cast<int>(blockIdx.x) >= W) return;
    int64_t u = cta_first(N, blockIdx.x, W);
    const int64_t u1 = cta_first(N, blockIdx.x + 1, W);
    // the entry that holds unit u, and its first unit
    int e = 0, n = 0;
    int64_t e0 = 0;
    for (int base = 0;; base += 32) {
        const int mine = base + lane < pl.entries ? pl.units(p, base + lane) : 0;
        int64_t incl = static_cast<int64_t>(mine) * c.Hkv;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, e0 + incl > u);
        if (hit) {
            const int src = __ffs(hit) - 1;
            n = __shfl_sync(0xffffffffu, mine, src);
            e0 += __shfl_sync(0xffffffffu, incl, src) - static_cast<int64_t>(n) * c.Hkv;
            e = base + src;
            break;
        }
        e0 += __shfl_sync(0xffffffffu, incl, 31);
    }

    bool first_seg = true;
    const int ra = 4 * (g >> 1) + (g & 1), rb = ra + 2;       // this lane's K rows of a step
    while (u < u1) {
        while (n == 0 || u >= e0 + static_cast<int64_t>(n) * c.Hkv) {     // the next entry with rows
            e0 += static_cast<int64_t>(n) * c.Hkv;
            n = pl.units(p, ++e);
        }
        const int h = static_cast<int>((u - e0) / n), ua = static_cast<int>(u - e0 - static_cast<int64_t>(h) * n);
        const int ub = static_cast<int>(min(static_cast<int64_t>(n), ua + (u1 - u)));
        int pos, cnt;
        const int len = pl.rows(p, e, pos, cnt), b = e / pl.tiles;
        const int64_t q0 = static_cast<int64_t>(e - b * pl.tiles) * pl.tile;         // the tile's first query
        const int nq = static_cast<int>(min(static_cast<int64_t>(pl.tile), static_cast<int64_t>(cnt) * pl.rep - q0));
        const int row0 = ua * kUnit, row1 = static_cast<int>(min(static_cast<int64_t>(len), static_cast<int64_t>(ub) * kUnit));
        const int nstep = (row1 - row0 + kStep - 1) / kStep;
        const int8_t *Kb = c.k + b * c.bs + h * c.hs, *Vb = c.v + b * c.bs + h * c.hs;
        const float *ksb = c.ks + b * c.sbs + h * c.shs, *vsb = c.vs + b * c.sbs + h * c.shs;

        auto issue = [&](int s, int stage) {                    // step s (every kWarps-th is this warp's) into a stage
            if (s < nstep) {
                const int r0 = row0 + s * kStep;
                const uint32_t st = wbase + stage * STB;
#pragma unroll
                for (int i = 0; i < kStep * CH / 32; ++i) {
                    const int idx = lane + 32 * i, r = idx / CH, ch = idx % CH;
                    if (r0 + r < row1 && ch < nch) {
                        const int64_t go = static_cast<int64_t>(r0 + r) * c.rs + ch * 16;
                        const int so = stage_off<DP>(r, ch);
                        cp_async_16(st + so, Kb + go, 16);
                        cp_async_16(st + kStep * DP + so, Vb + go, 16);
                    }
                }
                if (lane < 2) cp_async_4(st + 2 * kStep * DP + 4 * lane, (lane ? vsb : ksb) + (r0 >> c.blk_log2));
            }
            cp_commit();
        };
#pragma unroll
        for (int s = 0; s < NS - 1; ++s) issue(warp + s * kWarps, s);

        // q^T as B fragments: k slots (2t, 2t+1 | 2t+8, 2t+9) of step (i, w) are d = 16 (t + 4i) + 4w + (0, 1 | 2, 3)
        uint32_t qf[PARTS][NT][KI * 4][2];
        float rs[NT][2];
        int lim[NT][2];
        int64_t moff[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int qi = 8 * nt + g;
            const bool ok = qi < nq;
            const int tok = static_cast<int>((q0 + (ok ? qi : 0)) / pl.rep);
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
                    for (int k = 0; k < 4; ++k) mx = fmaxf(mx, fabsf(x[i * 4 + w][k]));
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float f = pow2_to(mx, 8);
#pragma unroll
            for (int s = 0; s < KI * 4; ++s)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float v0 = x[s][2 * k] * f, v1 = x[s][2 * k + 1] * f;
                    qf[0][nt][s][k] = pack_h2(v0, v1);
                    if constexpr (PARTS == 2) {
                        const float2 r = unpack_h2(qf[0][nt][s][k]);
                        qf[PARTS - 1][nt][s][k] = pack_h2(v0 - r.x, v1 - r.y);
                    }
                }
            // what a lane's columns 2t, 2t + 1 of the scores need
            const float rsg = p.scale * (MASK ? 1.f : kLog2e) / f;
            const int lg = ok ? pos + tok : -1;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                rs[nt][k] = __shfl_sync(0xffffffffu, rsg, (2 * t + k) * 4);
                lim[nt][k] = __shfl_sync(0xffffffffu, lg, (2 * t + k) * 4);
                if constexpr (MASK) moff[nt][k] = b * p.mbs + __shfl_sync(0xffffffffu, tok, (2 * t + k) * 4) * p.mts;
            }
        }
        // the first row that some query of the tile must not see (queries past nq do not matter)
        const int edge = pos + static_cast<int>(q0 / pl.rep) + 1;

        float o[VW * 2][NT][4], m[NT][2], l[NT][2], cv = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < VW * 2; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }
        float mk[NT][4];                                       // the mask of this warp's next step
        auto load_mask = [&](int s) {
            if constexpr (MASK) {
                const int ja = row0 + s * kStep + ra;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int j = ja + (k & 2);
                        mk[nt][k] = s < nstep && j <= lim[nt][k & 1] ? p.mask[moff[nt][k & 1] + j] : -INFINITY;
                    }
            }
        };
        load_mask(warp);
        int stage = 0;
        for (int s = warp; s < nstep; s += kWarps) {
            __syncwarp();                                      // every lane is past its reads of the stage refilled here
            issue(s + (NS - 1) * kWarps, stage == 0 ? NS - 1 : stage - 1);
            cp_wait<NS - 1>();
            __syncwarp();
            const uint32_t kb = wbase + stage * STB, vb = kb + kStep * DP;
            stage = stage + 1 == NS ? 0 : stage + 1;
            const float2 ksv = *reinterpret_cast<const float2 *>(smem + (vb + kStep * DP - smem_u32(smem)));
            const int r0 = row0 + s * kStep;
            float x[NT][4];
            {
                float acc[NT][2][4];                           // two chains a tile
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[nt][0][k] = acc[nt][1][k] = 0.f;
#pragma unroll
                for (int i = 0; i < KI; ++i) {
                    const uint4 va = lds_v4(kb + stage_off<DP>(ra, t + 4 * i)), vv = lds_v4(kb + stage_off<DP>(rb, t + 4 * i));
                    const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vv.x, vv.y, vv.z, vv.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t xa = wa[w] ^ 0x80808080u, xb = wb[w] ^ 0x80808080u;
                        const uint32_t a0 = h2_lo(xa), a1 = h2_lo(xb), a2 = h2_hi(xa), a3 = h2_hi(xb);
#pragma unroll
                        for (int pt = 0; pt < PARTS; ++pt)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                mma_f16(acc[nt][w & 1], a0, a1, a2, a3, qf[pt][nt][i * 4 + w][0], qf[pt][nt][i * 4 + w][1]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float f0 = ksv.x * rs[nt][0], f1 = ksv.x * rs[nt][1];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        x[nt][k] = (acc[nt][0][k] + acc[nt][1][k]) * (k & 1 ? f1 : f0);
                        if constexpr (MASK) x[nt][k] = mk[nt][k] == -INFINITY ? -INFINITY : x[nt][k] + mk[nt][k];
                    }
                }
            }
            load_mask(s + kWarps);
            if (!MASK && r0 + kStep > edge) {                  // MASK: load_mask gave -inf beyond the limits
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (r0 + (k & 2 ? rb : ra) > lim[nt][k & 1]) x[nt][k] = -INFINITY;
            }
            bool up = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 4; ++k) up |= x[nt][k] > m[nt][k & 1] + RAISE;
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float mx = fmaxf(x[nt][k], x[nt][k + 2]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float mn = fmaxf(m[nt][k], mx);
                        const float a = mn == -INFINITY ? 1.f : ex2((m[nt][k] - mn) * U);
                        m[nt][k] = mn;
                        l[nt][k] *= a;
#pragma unroll
                        for (int i = 0; i < VW * 2; ++i) {
                            o[i][nt][k] *= a;
                            o[i][nt][k + 2] *= a;
                        }
                    }
            }
            if (ksv.y * cv > 512.f || (cv == 0.f && ksv.y > 0.f)) {         // uniform: the weights' power of two
                const float cn = pow2_to(ksv.y, 7), a = cv == 0.f ? 1.f : cn / cv;
                cv = cn;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < VW * 2; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[i][nt][k] *= a;
            }
            const float sv = ksv.y * cv;
            uint32_t pb[PARTS][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float mr = m[nt][k & 1] == -INFINITY ? 0.f : m[nt][k & 1];
                    const float e2 = ex2((x[nt][k] - mr) * U);
                    l[nt][k & 1] += e2;
                    w[k] = e2 * sv;
                    // a row that is not seen weighs nothing, even where its scale is NaN
                    if (x[nt][k] == -INFINITY) w[k] = 0.f;
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t hi = pack_h2(w[2 * k], w[2 * k + 1]);
                    pb[0][nt][k] = movmatrix_trans(hi);
                    if constexpr (PARTS == 2) {
                        const float2 r = unpack_h2(hi);
                        pb[PARTS - 1][nt][k] = movmatrix_trans(pack_h2(w[2 * k] - r.x, w[2 * k + 1] - r.y));
                    }
                }
            }
            // V: words of rows 4t .. 4t + 3
#pragma unroll
            for (int v = 0; v < (DP == 256 ? 2 : 1); ++v) {
                uint32_t wd[4][DP == 64 ? 2 : 4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (DP == 64) {
                        const uint2 q2 = lds_v2(vb + stage_off<DP>(4 * t + r, g >> 1) + (g & 1) * 8);
                        wd[r][0] = q2.x;
                        wd[r][1] = q2.y;
                    } else {
                        const uint4 q4 = lds_v4(vb + stage_off<DP>(4 * t + r, g + 8 * v));
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
                    for (int hf = 0; hf < 2; ++hf) {           // d = 4w + 2 hf + (0, 1)
                        const uint32_t r01 = prmt(y[0], y[1], hf ? 0x7362u : 0x5140u);
                        const uint32_t r23 = prmt(y[2], y[3], hf ? 0x7362u : 0x5140u);
                        const uint32_t a0 = h2_lo(r01), a1 = h2_hi(r01), a2 = h2_lo(r23), a3 = h2_hi(r23);
#pragma unroll
                        for (int pt = 0; pt < PARTS; ++pt)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                mma_f16(o[(v * 4 + w) * 2 + hf][nt], a0, a1, a2, a3, pb[pt][nt][0], pb[pt][nt][1]);
                    }
                }
            }
        }
        // merge the warps in shared memory (every copy has landed: the last NS - 1 groups are empty)
        cp_wait<0>();
        __syncthreads();
        float *osm = reinterpret_cast<float *>(smem);                              // [warps][8 NT][DP + 4]
        float2 *msm = reinterpret_cast<float2 *>(osm + kWarps * 8 * NT * (DP + 4));    // [warps][8 NT] reference, sum
        const float inv = cv == 0.f ? 1.f : 1.f / cv;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
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
        const bool whole = ua == 0 && ub == n;
        const int slot = 2 * blockIdx.x + (first_seg ? 0 : 1);
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
                const int tok = static_cast<int>((q0 + q) / pl.rep);
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
        __syncthreads();                                       // before the stages are filled again
        first_seg = false;
        u += ub - ua;
    }
}

// ---------------------------------------------------------------- the shared segments
// One CTA per query: where several CTAs of the split kernel hold a part of its rows, adds their partials
// in order (each warp every fourth part, four values a lane).
constexpr int kJoinWarps = 4;

template <int DP, int NT, bool BF16, bool MASK>
__global__ void __launch_bounds__(kJoinWarps * 32) kv8_attn_join_kernel(const Kv8AttnParams p, int G) {
    constexpr float U = MASK ? kLog2e : 1.f;
    constexpr int TILE = 8 * NT;
    __shared__ float red[kJoinWarps][2];
    __shared__ float4 acc[kJoinWarps][DP / 4];
    pdl_launch_dependents();
    pdl_wait_prerequisites();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.c.D;
    const Plan pl(p, TILE);
    const int q = blockIdx.x % TILE, h = blockIdx.x / TILE % p.c.Hkv, e = blockIdx.x / TILE / p.c.Hkv;
    int pos, cnt;
    const int len = pl.rows(p, e, pos, cnt), b = e / pl.tiles;
    const int64_t qr = static_cast<int64_t>(e - b * pl.tiles) * TILE + q;
    if (len == 0 || qr >= static_cast<int64_t>(cnt) * pl.rep) return;
    const int n = (len - 1) / kUnit + 1;
    int64_t before = 0, all = 0;
    for (int i = lane; i < pl.entries; i += 32) {
        const int v = pl.units(p, i);
        all += v;
        if (i < e) before += v;
    }
    const int64_t N = warp_sum64(all) * p.c.Hkv, u = warp_sum64(before) * p.c.Hkv + static_cast<int64_t>(h) * n;
    const int W = static_cast<int>(min(N, static_cast<int64_t>(G)));
    const int i0 = cta_of(N, u, W), i1 = cta_of(N, u + n - 1, W);
    if (i0 == i1) return;                                      // one CTA had it all and wrote the output
    // a CTA's first segment is in its slot 0, a later one that it shares (its last) in slot 1
    const auto slot = [&](int i) { return 2 * i + (i == i0 && cta_first(N, i, W) < u ? 1 : 0); };
    float M = -INFINITY;
    for (int i = i0 + lane; i <= i1; i += 32) M = fmaxf(M, slot_ml<DP>(p.ws, TILE, G, slot(i))[q].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 y[DP == 256 ? 2 : 1];
#pragma unroll
    for (auto &v : y) v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = i0 + warp; i <= i1; i += kJoinWarps) {
        const int s = slot(i);
        const float2 ml = slot_ml<DP>(p.ws, TILE, G, s)[q];
        const float f = ex2((ml.x - ref) * U);
        L = fmaf(ml.y, f, L);
#pragma unroll
        for (int k = 0; k < (DP == 256 ? 2 : 1); ++k) {
            const int d = 128 * k + 4 * lane;
            if (d < D) {
                const float4 v = *reinterpret_cast<const float4 *>(slot_o<DP>(p.ws, TILE, s) + q * DP + d);
                y[k].x = fmaf(v.x, f, y[k].x);
                y[k].y = fmaf(v.y, f, y[k].y);
                y[k].z = fmaf(v.z, f, y[k].z);
                y[k].w = fmaf(v.w, f, y[k].w);
            }
        }
    }
    if (lane == 0) red[warp][0] = L;
#pragma unroll
    for (int k = 0; k < (DP == 256 ? 2 : 1); ++k)
        if (32 * k + lane < DP / 4) acc[warp][32 * k + lane] = y[k];
    __syncthreads();
    L = 0.f;
    for (int w = 0; w < kJoinWarps; ++w) L += red[w][0];
    const int tok = static_cast<int>(qr / pl.rep), hq = h * pl.rep + static_cast<int>(qr - static_cast<int64_t>(tok) * pl.rep);
    float so;
    const float f = out_factor<MASK>(M, L, p.sinks, hq, so) * so;
    const int d = 4 * threadIdx.x;
    if (d < D) {
        float4 t = acc[0][threadIdx.x];
        for (int w = 1; w < kJoinWarps; ++w) {
            const float4 v = acc[w][threadIdx.x];
            t.x += v.x;
            t.y += v.y;
            t.z += v.z;
            t.w += v.w;
        }
        store4<BF16>(p.out, (static_cast<int64_t>(b) * p.r.T + tok) * p.ldo + static_cast<int64_t>(hq) * D + d,
                     make_float4(t.x * f, t.y * f, t.z * f, t.w * f));
    }
}

// ---------------------------------------------------------------- host side
int device_sms() {
    static const int n = [] {
        int dev = 0, v = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
        return v > 0 ? v : 1;
    }();
    return n;
}

// Query tiles: 8 NT queries; larger ones share the decoded codes and are limited by registers (the queries'
// fragments take DP / 8 * NT * parts, the outputs DP / 4 * NT of them).
int pick_nt(int DP, int64_t queries, bool bf16) {
    const int most = DP == 64 ? 4 : DP == 128 ? (bf16 ? 4 : 2) : (bf16 ? 2 : 1);
    const int want = queries <= 8 ? 1 : queries <= 16 ? 2 : 4;
    return want < most ? want : most;
}
int padded_dim(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

template <int DP, int NT, bool BF16, bool MASK>
struct Split {
    static constexpr int NS = DP == 256 ? 3 : 4;
    static constexpr int ring = kWarps * NS * kStageBytes<DP>, merge = kMergeBytes<DP, NT>;
    static constexpr int smem = ring > merge ? ring : merge;
    static int ctas() {                                        // one resident wave
        static const int n = [] {
            auto k = kv8_attn_split_kernel<DP, NT, BF16, MASK, NS>;
            int per = 0;
            if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
                cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, k, kWarps * 32, smem) != cudaSuccess || per < 1)
                per = 1;
            return per * device_sms();
        }();
        return n;
    }
    static cudaError_t launch(const Kv8AttnParams &p, cudaStream_t s) {
        const int G = ctas(), rep = p.Hq / p.c.Hkv;
        const int64_t tiles = (static_cast<int64_t>(p.r.T) * rep + 8 * NT - 1) / (8 * NT);
        const int64_t joins = tiles * p.c.B * p.c.Hkv * 8 * NT;
        if (tiles * p.c.B > 0x7fffffff || joins > 0x7fffffff) return cudaErrorInvalidConfiguration;
        const cudaError_t e = launch_pdl(kv8_attn_split_kernel<DP, NT, BF16, MASK, NS>, dim3(G), dim3(kWarps * 32), smem, s, p);
        if (e != cudaSuccess) return e;
        return launch_pdl(kv8_attn_join_kernel<DP, NT, BF16, MASK>, dim3(static_cast<unsigned>(joins)), dim3(kJoinWarps * 32),
                          0, s, p, G);
    }
};

// f(Split<...>) for the call's sizes and types
template <int DP, bool BF16, bool MASK, typename F>
auto with_nt(int nt, F f) {
    if constexpr (DP == 64 || (DP == 128 && BF16)) {
        if (nt == 4) return f(Split<DP, 4, BF16, MASK>{});
    }
    if constexpr (DP != 256 || BF16) {
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
    const int DP = padded_dim(D), nt = pick_nt(DP, queries, bf16);
    return DP == 64    ? with_types<64>(nt, bf16, mask, f)
           : DP == 128 ? with_types<128>(nt, bf16, mask, f)
                       : with_types<256>(nt, bf16, mask, f);
}

}  // namespace

int64_t kv8_attn_ws_bytes(int Hq, int Hkv, int D, int T, bool bf16) {
    const int64_t queries = static_cast<int64_t>(T) * (Hq / Hkv);
    const int DP = padded_dim(D), tile = 8 * pick_nt(DP, queries, bf16);
    int64_t G = 0;
    for (const bool mask : {false, true}) {
        const int64_t g = with_split(D, queries, bf16, mask, [](auto k) { return k.ctas(); });
        G = g > G ? g : G;
    }
    return 2 * G * tile * (DP + 2) * 4;
}

cudaError_t kv8_attn_launch(const Kv8AttnParams &p, bool bf16, cudaStream_t stream) {
    return with_split(p.c.D, static_cast<int64_t>(p.r.T) * (p.Hq / p.c.Hkv), bf16, p.mask != nullptr,
                      [&](auto k) { return k.launch(p, stream); });
}

}  // namespace onpu_b200
