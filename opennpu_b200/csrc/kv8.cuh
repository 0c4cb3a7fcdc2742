// Device helpers the 8-bit KV cache's kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kernels.h"
#include "tmap.h"

namespace onpu_b200 {

// The rows of sequence b: cache rows pos .. pos + cnt - 1. False (and bit 32 of *err) where they are not
// all inside the cache of S rows or cnt is not in [0, T]; the sequence is then skipped.
__device__ __forceinline__ bool kv8_rows(const Kv8Rows &r, int b, int S, int &pos, int &cnt) {
    pos = r.pos[b];
    cnt = r.cnt ? r.cnt[b] : r.T;
    if (cnt >= 0 && cnt <= r.T && pos >= 0 && pos <= S - cnt) return true;
    atomicOr(r.err, 32);
    return false;
}

// ---------------------------------------------------------------- attention
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint64_t kWaitNs = 2000000000ull;   // bound of every wait for a copy

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
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t x) { return __half22float2(*reinterpret_cast<__half2 *>(&x)); }
// 2^(top - exponent of x), at most 2^126: x times it is in [2^top, 2^(top + 1)) (less for x below 2^(top - 126)); 1 for 0, inf and NaN
__device__ __forceinline__ float pow2_to(float x, int top) {
    const int e = static_cast<int>(__float_as_uint(x) >> 23 & 0xff);
    if (e == 255 || !(fabsf(x) > 0.f)) return 1.f;
    return __uint_as_float(static_cast<uint32_t>(127 + min(126, max(-126, top + 127 - e))) << 23);
}
__device__ __forceinline__ float max_nan(float a, float b) {     // NaN where either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// a / b, in 32 bits where they fit (they all but always do; a 64-bit division costs a few hundred instructions)
__device__ __forceinline__ int64_t div64(int64_t a, int64_t b) {
    if (((a | b) >> 31) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// ---------------------------------------------------------------- the list of units
// An entry is a (sequence, query tile); its rows are counted in units of `unit` rows, once per kv head.
struct Plan {
    int rep, tile, tiles, entries, unit;    // query heads per kv head, queries a tile, tiles a sequence, B * tiles
    int shift;                              // unit = 1 << shift
    __device__ __forceinline__ Plan(const Kv8AttnParams &p, int tile_, int unit_) {
        rep = p.Hq / p.c.Hkv;
        tile = tile_;
        unit = unit_;
        shift = 31 - __clz(unit);
        tiles = static_cast<int>((static_cast<int64_t>(p.r.T) * rep + tile - 1) / tile);
        entries = p.c.B * tiles;
    }
    // rows that entry e's tile sees (0: nothing of it is valid)
    __device__ __forceinline__ int rows(const Kv8AttnParams &p, int e, int &pos, int &cnt) const {
        const int b = tiles == 1 ? e : e / tiles;
        if (!kv8_rows(p.r, b, p.c.S, pos, cnt)) return 0;
        if (tiles == 1) return cnt > 0 ? pos + cnt : 0;
        const int64_t r0 = static_cast<int64_t>(e - b * tiles) * tile;
        const int first = static_cast<int>(div64(r0, rep)), last = static_cast<int>(div64(r0 + tile - 1, rep));
        if (first >= cnt) return 0;
        return pos + min(last, cnt - 1) + 1;
    }
    __device__ __forceinline__ int units_of(int len) const {
        return static_cast<int>((static_cast<unsigned>(len) + unit - 1) >> shift);
    }
    __device__ __forceinline__ int units(const Kv8AttnParams &p, int e) const {
        int pos, cnt;
        return units_of(rows(p, e, pos, cnt));
    }
};
__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// units a CTA takes: N units over G CTAs; CTA i has units [i * per, (i + 1) * per) of the list. (At least two each: one
// token over 4096 rows 10.0 us against 10.5, over 77 rows 9.5 against 6.3.)
__device__ __forceinline__ int64_t units_per_cta(int64_t N, int G) { return max(int64_t{1}, div64(N + G - 1, G)); }

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
// Where CTA i of the list stands: the entry that holds unit u (every lane of the warp gets it), its units
// and its first one
__device__ __forceinline__ void find_entry(const Kv8AttnParams &p, const Plan &pl, int lane, int64_t u, int &e, int &n,
                                           int64_t &e0) {
    e0 = 0;
    for (int base = 0;; base += 32) {
        const int mine = base + lane < pl.entries ? pl.units(p, base + lane) : 0;
        int64_t incl = static_cast<int64_t>(mine) * p.c.Hkv;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, e0 + incl > u);
        if (hit) {
            const int src = __ffs(hit) - 1;
            n = __shfl_sync(0xffffffffu, mine, src);
            e0 += __shfl_sync(0xffffffffu, incl, src) - static_cast<int64_t>(n) * p.c.Hkv;
            e = base + src;
            return;
        }
        e0 += __shfl_sync(0xffffffffu, incl, 31);
        if (base + 32 >= pl.entries) {           // only if pos or cnt changed under the call: nothing for this CTA
            e = pl.entries - 1;
            n = 0;
            return;
        }
    }
}
// units of all entries and heads
__device__ __forceinline__ int64_t total_units(const Kv8AttnParams &p, const Plan &pl, int lane) {
    int64_t N = 0;
    for (int e = lane; e < pl.entries; e += 32) N += pl.units(p, e);
    return warp_sum64(N) * p.c.Hkv;
}
// A CTA's way through the list: segments, each a run of one entry's units for one kv head
struct Walk {
    int64_t u, u1, e0;                // the next unit, the end of this CTA's, the entry's first
    int e, n, pos, cnt, len;          // the entry, its units (per head), its sequence's rows, the rows it sees
    bool first;                       // no segment taken yet
    // the segment at u
    int b, h, ua, ub, nq;
    int64_t q0;                       // the tile's first query
    __device__ __forceinline__ bool start(const Kv8AttnParams &p, const Plan &pl, int lane, int cta, int G) {
        first = true;
        if (pl.entries <= 32) {       // one round of loads: an entry a lane (their units fit 32 bits)
            int ps = 0, cn = 0, ln = 0;
            if (lane < pl.entries) ln = pl.rows(p, lane, ps, cn);
            const unsigned mine = pl.units_of(ln);
            unsigned incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            const int64_t N = static_cast<int64_t>(__shfl_sync(0xffffffffu, incl, 31)) * p.c.Hkv, per = units_per_cta(N, G);
            u = per * cta;
            u1 = min(N, u + per);
            if (u >= u1) return false;
            e = __ffs(__ballot_sync(0xffffffffu, static_cast<int64_t>(incl) * p.c.Hkv > u)) - 1;
            n = __shfl_sync(0xffffffffu, mine, e);
            e0 = (static_cast<int64_t>(__shfl_sync(0xffffffffu, incl, e)) - n) * p.c.Hkv;
            pos = __shfl_sync(0xffffffffu, ps, e);
            cnt = __shfl_sync(0xffffffffu, cn, e);
            len = __shfl_sync(0xffffffffu, ln, e);
            return true;
        }
        const int64_t N = total_units(p, pl, lane), per = units_per_cta(N, G);
        u = per * cta;
        u1 = min(N, u + per);
        if (u >= u1) return false;
        find_entry(p, pl, lane, u, e, n, e0);
        len = pl.rows(p, e, pos, cnt);
        return true;
    }
    __device__ __forceinline__ bool segment(const Kv8AttnParams &p, const Plan &pl) {
        if (u >= u1) return false;
        while (n == 0 || u >= e0 + static_cast<int64_t>(n) * p.c.Hkv) {     // the next entry with rows
            e0 += static_cast<int64_t>(n) * p.c.Hkv;
            if (++e >= pl.entries) return false;     // only if pos or cnt changed under the call
            len = pl.rows(p, e, pos, cnt);
            n = pl.units_of(len);
        }
        h = static_cast<int>(div64(u - e0, n));
        ua = static_cast<int>(u - e0 - static_cast<int64_t>(h) * n);
        ub = static_cast<int>(min(static_cast<int64_t>(n), ua + (u1 - u)));
        b = pl.tiles == 1 ? e : e / pl.tiles;
        q0 = static_cast<int64_t>(e - b * pl.tiles) * pl.tile;
        nq = static_cast<int>(min(static_cast<int64_t>(pl.tile), static_cast<int64_t>(cnt) * pl.rep - q0));
        return true;
    }
    __device__ __forceinline__ bool whole() const { return ua == 0 && ub == n; }
    __device__ __forceinline__ int slot(int cta) const { return 2 * cta + (first ? 0 : 1); }
    __device__ __forceinline__ void next() {
        first = false;
        u += ub - ua;
    }
};


// Which CTAs hold an entry's rows for one head, and in which of their slots: a CTA's first segment is in its slot 0, its
// last in slot 1. i0 == i1: one has them all.
struct Shares {
    int b, cnt, h, i0, i1, s0;
    int64_t q0;                       // the tile's first query
    // entry e's for head h_; every lane of the warp goes through the list
    __device__ __forceinline__ Shares(const Kv8AttnParams &p, const Plan &pl, int lane, int e, int h_, int G) {
        int64_t before = 0, all = 0;
        for (int i = lane; i < pl.entries; i += 32) {
            const int v = pl.units(p, i);
            all += v;
            if (i < e) before += v;
        }
        int pos;
        const int n = pl.units_of(pl.rows(p, e, pos, cnt));
        h = h_;
        tile_of(pl, e);
        const int64_t N = warp_sum64(all) * p.c.Hkv, u = warp_sum64(before) * p.c.Hkv + static_cast<int64_t>(h) * n;
        set(u, n, units_per_cta(N, G));
    }
    // those that CTA i's last segment is shared with, where it is the first to have a part of it (else none: i0 == i1). A block
    // of THREADS goes through the list together, a run of entries a thread.
    template <int THREADS>
    __device__ __forceinline__ Shares(const Kv8AttnParams &p, const Plan &pl, int i, int G, std::integral_constant<int, THREADS>) {
        __shared__ int64_t sums[THREADS / 32], at_e0;
        __shared__ int at_e, at_n;
        const int t = threadIdx.x, lane = t & 31, run = (pl.entries + THREADS - 1) / THREADS;
        const int e0 = static_cast<int>(min(static_cast<int64_t>(pl.entries), static_cast<int64_t>(t) * run));
        const int e1 = static_cast<int>(min(static_cast<int64_t>(pl.entries), static_cast<int64_t>(e0) + run));
        int64_t mine = 0;
        for (int e = e0; e < e1; ++e) mine += pl.units(p, e);
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) sums[t >> 5] = incl;
        if (t == 0) at_n = 0;
        __syncthreads();
        int64_t N = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < t >> 5) incl += sums[w];
            N += sums[w];
        }
        N *= p.c.Hkv;
        const int64_t per = units_per_cta(N, G), border = per * (i + 1);
        int64_t u = (incl - mine) * p.c.Hkv;
        if (border >= u && border < incl * p.c.Hkv) {              // one thread's, if any
            for (int e = e0; e < e1; ++e) {
                const int n = pl.units(p, e);
                if (border < u + static_cast<int64_t>(n) * p.c.Hkv) {
                    at_e = e;
                    at_n = n;
                    at_e0 = u;
                    break;
                }
                u += static_cast<int64_t>(n) * p.c.Hkv;
            }
        }
        __syncthreads();
        b = cnt = h = i0 = i1 = s0 = 0;
        q0 = 0;
        const int n = at_n;
        if (n == 0) return;                                        // the list ends before the border
        h = static_cast<int>(div64(border - at_e0, n));
        u = at_e0 + static_cast<int64_t>(h) * n;
        if (u == border) return;                                   // a segment begins there
        set(u, n, per);
        if (i0 != i) i1 = i0;                                      // an earlier border's
        int pos;
        pl.rows(p, at_e, pos, cnt);
        tile_of(pl, at_e);
    }
    __device__ __forceinline__ int slot(int i) const { return i == i0 ? s0 : 2 * i; }

private:
    __device__ __forceinline__ void tile_of(const Plan &pl, int e) {
        b = pl.tiles == 1 ? e : e / pl.tiles;
        q0 = static_cast<int64_t>(e - b * pl.tiles) * pl.tile;
    }
    __device__ __forceinline__ void set(int64_t u, int n, int64_t per) {
        i0 = n ? static_cast<int>(div64(u, per)) : 0;
        i1 = n ? static_cast<int>(div64(u + n - 1, per)) : 0;
        s0 = 2 * i0 + (i0 * per < u ? 1 : 0);
    }
};

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

// (host) f()'s value where it is above 0 (kept from then on), else what a lookup that failed gave: asked for again at the next call
template <typename F>
int kv8_kept(std::atomic<int> &kept, F f) {
    int n = kept.load(std::memory_order_relaxed);
    if (n <= 0) {
        n = f();
        if (n > 0) kept.store(n, std::memory_order_relaxed);
    }
    return n;
}
// (host) the error of such a lookup
inline cudaError_t kv8_lookup_error() {
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : cudaErrorInvalidConfiguration;
}
// (host) SMs of the current device; 0: the lookup failed
inline int kv8_sms() {
    static std::atomic<int> kept{0};
    return kv8_kept(kept, [] {
        int dev = 0, v = 0;
        return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? v : 0;
    });
}
// (host) a map of [batch][heads][rows][dim] codes whose boxes are `rows` rows of at most 128 codes, their 16-byte
// chunks exchanged by `swizzle`; columns and rows past the ends read 0
inline bool kv8_code_map(CUtensorMap &map, const Kv8Cache &c, int8_t *codes, int DP, int rows, CUtensorMapSwizzle swizzle) {
    const auto fn = tensor_map_encode_fn();
    if (!fn) return false;
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(DP < 128 ? DP : 128), static_cast<cuuint32_t>(rows), 1, 1};
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.D), static_cast<cuuint64_t>(c.S), static_cast<cuuint64_t>(c.Hkv),
                                static_cast<cuuint64_t>(c.B)};
    // a lone head's or sequence's stride is not used: any valid one
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(c.rs), static_cast<cuuint64_t>(c.Hkv > 1 ? c.hs : c.rs),
                                   static_cast<cuuint64_t>(c.B > 1 ? c.bs : c.rs)};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    return fn(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, codes, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
              swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace onpu_b200
