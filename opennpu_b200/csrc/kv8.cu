// The 8-bit KV cache's writer and reader: rows of K and V quantised as they are appended, and rows read
// back. One fp32 scale s per (sequence, kv head, block of R rows); a value is code * s, the code an int8 in
// [-127, 127]. Appending rows pos .. pos + cnt - 1 of a sequence, for each block that holds one of them:
//   s_old = the stored scale if the block holds rows before pos, else 0 (a block's first row starts it anew)
//   s     = max(s_old, a / 127), a the largest |x| of the block's new rows (the division rounded to fp32)
//   new rows: code = rint(x / s), ties to even, of the exact quotient; at most +-127; 0 where s is 0
//   old rows, where the scale grew: code = rint(code * s_old / s), of the exact quotient
// so a block's codes always span its largest value, whatever order and sizes its rows come in. A new
// value that is not finite makes its block's scale NaN (its rows read back as NaN, and stay so until the
// block is begun again); its codes are 0.
//
// x / s's nearest integer n comes from x * (1 / s) in fp32 and is put right by the remainder x - n s, which one
// fused multiply-add gives exactly, against s / 2: bf16 rows have exact halves often (x / a is a quotient of 8-bit
// integers), so there is no branch around it. code * s_old / s needs two-float products and is looked
// at only where the fp32 quotient is within 1e-4 of a half. Scales below 2^-60 are taken times 2^64 first, so
// that nothing of this underflows.
//
// Bound by memory: a row costs its own bytes, its codes and, seldom, its block's older codes. 4 x 2048 bf16 rows of 8 heads
// of 128 written and read back (101 MB): 30.4 us, 3.3 TB/s (0.51 of the copy bandwidth; the writer's CTAs each wait for
// pos, then their rows); 8 x 8192 rows read back (403 MB): 73.9 us, 5.5 TB/s (0.83). One token: 3.3 us, two launches' latency.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kernels.h"
#include "kv8.cuh"
#include "ptx.cuh"

namespace onpu_b200 {
namespace {

// the low bytes of eight floats that 1.5 * 2^23 was added to: their integers
constexpr float kMagic = 12582912.f;
__device__ __forceinline__ uint2 low_bytes(const float (&t)[8]) {
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t lo = __byte_perm(__float_as_uint(t[4 * k]), __float_as_uint(t[4 * k + 1]), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(t[4 * k + 2]), __float_as_uint(t[4 * k + 3]), 0x0040);
        w[k] = __byte_perm(lo, hi, 0x5410);
    }
    return make_uint2(w[0], w[1]);
}
// codes of eight values: rint(x / s) of the exact quotient. CLAMP: a subnormal scale is coarse, quotients may
// pass 127.
template <bool CLAMP>
__device__ __forceinline__ uint2 kv8_codes8(const float (&x)[8], float inv, float s) {
    const uint32_t over = __float_as_uint(0.5f * s) + 1;   // the first float above s / 2
    float t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        t[e] = fmaf(x[e], inv, kMagic);
        const float rem = fmaf(-(t[e] - kMagic), s, x[e]);
        // past s / 2, or at it with t odd: one further
        const float lim = __uint_as_float(over - (__float_as_uint(t[e]) & 1));
        if (fabsf(rem) >= lim) t[e] += copysignf(1.f, rem);
        if constexpr (CLAMP) t[e] = fminf(fmaxf(t[e], kMagic - 127.f), kMagic + 127.f);
    }
    return low_bytes(t);
}
// older codes onto a larger scale: rint(code * s_old / s) of the exact quotient; ratio = s_old / s
__device__ __forceinline__ uint2 kv8_recode8(const float (&code)[8], float ratio, float s_old, float s) {
    float t[8], off = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float r = code[e] * ratio;
        t[e] = r + kMagic;
        off = fmaxf(off, fabsf(r - (t[e] - kMagic)));
    }
    if (off > 0.4999f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float r = code[e] * ratio, h = floorf(r) + 0.5f;
            if (!(fabsf(r - h) < 1e-4f)) continue;
            const float a = code[e] * s_old, b = h * s;
            const float d = (a - b) + (fmaf(code[e], s_old, -a) - fmaf(h, s, -b));      // its sign is code s_old - h s's
            const float lo = h - 0.5f, hi = h + 0.5f;
            t[e] = (d > 0.f ? hi : d < 0.f ? lo : 2.f * rintf(0.5f * h)) + kMagic;       // halfway: the even one of lo, hi
        }
    }
    return low_bytes(t);
}
__device__ __forceinline__ void widen8(uint2 q, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? q.x : q.y) >> (8 * (e & 3))));
}

template <bool BF16>
__device__ __forceinline__ void load8(const void *p, int64_t i, float (&f)[8]) {
    if constexpr (BF16) {
        const uint4 v = ld_nc_v4(static_cast<const uint16_t *>(p) + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[2 * e] = __uint_as_float(w[e] << 16);
            f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 v = ld_nc_v4(static_cast<const float *>(p) + i + 4 * h);
            f[4 * h] = __uint_as_float(v.x);
            f[4 * h + 1] = __uint_as_float(v.y);
            f[4 * h + 2] = __uint_as_float(v.z);
            f[4 * h + 3] = __uint_as_float(v.w);
        }
    }
}

// vectors of 8 in a row of D (a multiple of 16 up to 256): v / vpr of v < 2048 as a multiplication
struct RowDiv {
    int vpr, inv;                     // inv = ceil(2^16 / vpr): off by less than v / 2^16 <= 1 / 32 <= 1 / vpr
    explicit RowDiv(int D) : vpr(D / 8), inv((65536 + D / 8 - 1) / (D / 8)) {}
    __device__ __forceinline__ int div(int v) const { return v * inv >> 16; }
};

struct Kv8In {
    const void *x[2];                 // K rows, V rows
    int64_t ld[2];
};

// A group of G threads (a warp, or the CTA) writes one block of one head of K or V: NV vectors of 8 values
// per thread hold all of the block's new rows, so they are read once.
// CTAs of C threads, at least MINB of them an SM (what is in flight is their rows).
template <bool BF16, int G, int NV, int C, int MINB>
__global__ void __launch_bounds__(C, MINB) kv8_append_kernel(const Kv8Cache c, const Kv8Rows r, const Kv8In in,
                                                             unsigned groups, const RowDiv rd) {
    pdl_launch_dependents();
    pdl_wait_prerequisites();
    constexpr int kOld = 4;                                // older vectors in flight
    __shared__ uint32_t red[C / 32];
    const unsigned gi = blockIdx.x * (C / G) + threadIdx.x / G;      // of sequence b: block, K / V, head
    if (gi >= groups) return;                              // whole groups leave: G = 32, or one group a CTA
    const int tid = threadIdx.x % G, b = blockIdx.y, w = gi / (2 * c.Hkv);
    const int kvh = gi - w * 2 * c.Hkv, kv = kvh >= c.Hkv, h = kvh - (kv ? c.Hkv : 0);
    int pos, cnt;
    if (!kv8_rows(r, b, c.S, pos, cnt)) return;
    const int blk = (pos >> c.blk_log2) + w, row0 = blk << c.blk_log2;      // this block and its first row
    const int lo = max(pos, row0), hi = min(pos + cnt, row0 + (1 << c.blk_log2));
    if (lo >= hi) return;
    const int vpr = rd.vpr, nvec = (hi - lo) * vpr;       // vectors per row, and in all
    const int64_t xb = (static_cast<int64_t>(b) * r.T + (lo - pos)) * in.ld[kv] + static_cast<int64_t>(h) * c.D;
    float f[NV][8];
    int rr[NV], cc[NV];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = tid + i * G;
        rr[i] = rd.div(v);
        cc[i] = (v - rr[i] * vpr) * 8;
        if (v < nvec) {
            load8<BF16>(in.x[kv], xb + rr[i] * in.ld[kv] + cc[i], f[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(f[i][e]) & 0x7fffffffu);
        }
    }
    float *sp = (kv ? c.vs : c.ks) + b * c.sbs + h * c.shs + blk;
    const float s_old = row0 < pos ? *sp : 0.f;
    amax = __reduce_max_sync(0xffffffffu, amax);
    if constexpr (G > 32) {
        if ((tid & 31) == 0) red[tid >> 5] = amax;
        __syncthreads();                                   // also: every thread has read *sp
#pragma unroll
        for (int i = 0; i < G / 32; ++i) amax = max(amax, red[i]);
    } else {
        __syncwarp();
    }
    const bool bad = amax >= 0x7f800000u || s_old != s_old;
    const float s = bad ? __uint_as_float(0x7fc00000u) : fmaxf(s_old, __fdiv_rn(__uint_as_float(amax), 127.f));
    const bool tiny = s < 0x1p-60f;
    const float up = tiny ? 0x1p64f : 1.f, su = s * up, inv = 1.0f / su;
    int8_t *base = (kv ? c.v : c.k) + b * c.bs + h * c.hs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (tid + i * G < nvec) {
            uint2 q = make_uint2(0, 0);
            if (tiny) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[i][e] *= up;
                if (s > 0.f) q = kv8_codes8<true>(f[i], inv, su);
            } else if (!bad) {
                q = kv8_codes8<false>(f[i], inv, su);
            }
            *reinterpret_cast<uint2 *>(base + static_cast<int64_t>(lo + rr[i]) * c.rs + cc[i]) = q;
        }
    }
    if (s > s_old && row0 < pos) {                         // the block's older rows onto the larger scale
        const float so = s_old * up, ratio = so / su;
        const int nold = (pos - row0) * vpr;
        for (int v0 = tid; v0 < nold; v0 += kOld * G) {    // kOld vectors in flight
            uint2 old[kOld], *at[kOld];
#pragma unroll
            for (int i = 0; i < kOld; ++i) {
                const int v = v0 + i * G, ro = rd.div(v);
                at[i] = reinterpret_cast<uint2 *>(base + static_cast<int64_t>(row0 + ro) * c.rs + (v - ro * vpr) * 8);
                if (v < nold) old[i] = *at[i];
            }
#pragma unroll
            for (int i = 0; i < kOld; ++i) {
                float g[8];
                widen8(old[i], g);
                if (v0 + i * G < nold) *at[i] = kv8_recode8(g, ratio, so, su);
            }
        }
    }
    if (tid == 0) *sp = s;
}

template <bool BF16, int G, int NV, int C, int MINB>
cudaError_t append_t(const Kv8Cache &c, const Kv8Rows &r, const Kv8In &in, int nblk, cudaStream_t s) {
    const int64_t groups = static_cast<int64_t>(nblk) * 2 * c.Hkv;
    if (groups > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const unsigned ctas = static_cast<unsigned>((groups - 1) / (C / G) + 1);
    return launch_pdl(kv8_append_kernel<BF16, G, NV, C, MINB>, dim3(ctas, c.B), dim3(C), 0, s, c, r, in,
                      static_cast<unsigned>(groups), RowDiv(c.D));
}

template <bool BF16>
cudaError_t append_f(const Kv8Cache &c, const Kv8Rows &r, const Kv8In &in, cudaStream_t s) {
    const int R = 1 << c.blk_log2;
    const int nblk = static_cast<int>((static_cast<int64_t>(r.T) + R - 2) / R + 1);   // blocks T rows can touch
    const int nvec = (r.T < R ? r.T : R) * c.D / 8;                                    // a block's new vectors
    if (nvec <= 32) return append_t<BF16, 32, 1, 128, 4>(c, r, in, nblk, s);
    if (nvec <= 128) return append_t<BF16, 32, 4, 128, 4>(c, r, in, nblk, s);
    if (nvec <= 256) return append_t<BF16, 128, 2, 128, 8>(c, r, in, nblk, s);
    if (nvec <= 512) return append_t<BF16, 128, 4, 128, 8>(c, r, in, nblk, s);
    if (nvec <= 1024) return append_t<BF16, 256, 4, 256, 4>(c, r, in, nblk, s);
    return append_t<BF16, 256, 8, 256, 2>(c, r, in, nblk, s);                          // at most 64 rows of 256
}

// ---------------------------------------------------------------- read back
constexpr int kReadThreads = 256;

struct Kv8Out {
    void *y[2];
    int64_t ld[2];
};

// A CTA reads `rows` tokens of K or V, 8 codes a thread and kReadFly of them in flight, in the order of the
// output: D values of a head, heads of a token, tokens. Positions advance by kReadThreads vectors as digits
// (token, head, vector), without divisions.
constexpr int kReadFly = 4;

template <bool BF16>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(const Kv8Cache c, const Kv8Rows r, const Kv8Out out,
                                                                int rows, const RowDiv rd) {
    pdl_launch_dependents();
    pdl_wait_prerequisites();
    const int b = blockIdx.y >> 1, kv = blockIdx.y & 1, vpr = rd.vpr;
    const int sr = rd.div(kReadThreads), sv = kReadThreads - sr * vpr, si = sr / c.Hkv, sh = sr - si * c.Hkv;
    const int tr = rd.div(threadIdx.x), ti = tr / c.Hkv;
    int v = threadIdx.x - tr * vpr, h = tr - ti * c.Hkv;
    int pos, cnt;
    if (!kv8_rows(r, b, c.S, pos, cnt)) return;
    const int i0 = min(cnt, static_cast<int>(blockIdx.x) * rows), i1 = min(cnt, i0 + rows);
    const int8_t *base = (kv ? c.v : c.k) + b * c.bs;
    const float *sc = (kv ? c.vs : c.ks) + b * c.sbs;
    int i = i0 + ti;
    while (i < i1) {
        uint2 q[kReadFly];
        float s[kReadFly];
        int64_t o[kReadFly];
        bool ok[kReadFly];
#pragma unroll
        for (int k = 0; k < kReadFly; ++k) {
            ok[k] = i < i1;
            if (ok[k]) {
                const int row = pos + i;
                q[k] = *reinterpret_cast<const uint2 *>(base + h * c.hs + static_cast<int64_t>(row) * c.rs + v * 8);
                s[k] = sc[h * c.shs + (row >> c.blk_log2)];
                o[k] = (static_cast<int64_t>(b) * r.T + i) * out.ld[kv] + h * c.D + v * 8;
            }
            v += sv;
            h += sh + (v >= vpr);
            v -= v >= vpr ? vpr : 0;
            i += si + (h >= c.Hkv);
            h -= h >= c.Hkv ? c.Hkv : 0;
        }
#pragma unroll
        for (int k = 0; k < kReadFly; ++k) {
            if (!ok[k]) continue;
            float f[8];
            widen8(q[k], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= s[k];
            if constexpr (BF16) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
                    w[e] = *reinterpret_cast<const uint32_t *>(&t);
                }
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out.y[kv]) + o[k]) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                float4 *y = reinterpret_cast<float4 *>(static_cast<float *>(out.y[kv]) + o[k]);
                y[0] = make_float4(f[0], f[1], f[2], f[3]);
                y[1] = make_float4(f[4], f[5], f[6], f[7]);
            }
        }
    }
}

}  // namespace

cudaError_t kv8_append_launch(const Kv8Cache &c, const Kv8Rows &r, const void *k, int64_t ldk, const void *v,
                              int64_t ldv, bool bf16, cudaStream_t stream) {
    const Kv8In in{{k, v}, {ldk, ldv}};
    return bf16 ? append_f<true>(c, r, in, stream) : append_f<false>(c, r, in, stream);
}

cudaError_t kv8_read_launch(const Kv8Cache &c, const Kv8Rows &r, void *k, int64_t ldk, void *v, int64_t ldv,
                            bool bf16, cudaStream_t stream) {
    const Kv8Out out{{k, v}, {ldk, ldv}};
    // a CTA's rows: at least one vector for each of its threads, at most four rounds of kReadFly; in between
    // as many as leave eight CTAs for each SM
    const int64_t one = std::max<int64_t>(1, kReadThreads / (static_cast<int64_t>(c.Hkv) * c.D / 8));
    const int64_t spread = static_cast<int64_t>(r.T) * 2 * c.B / (8 * std::max(1, kv8_sms()));
    const int rows = static_cast<int>(std::min(std::max(one, spread), 4 * kReadFly * one));
    const dim3 grid((r.T - 1) / rows + 1, 2 * c.B);
    return bf16 ? launch_pdl(kv8_read_kernel<true>, grid, dim3(kReadThreads), 0, stream, c, r, out, rows, RowDiv(c.D))
                : launch_pdl(kv8_read_kernel<false>, grid, dim3(kReadThreads), 0, stream, c, r, out, rows, RowDiv(c.D));
}

}  // namespace onpu_b200
