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
// The quotient's nearest integer is taken from x * (1 / s) in fp32 (within 2^-16 of the quotient, which is
// at most 127) unless that lies within 1e-4 of the middle of two integers; there, and where 1 / s
// overflows, it is taken from the division in fp64, whose error (2^-46) is below the least distance of an
// inexact quotient of two fp32 numbers from such a middle (2^-27).
//
// Bound by memory: a row costs its own bytes, its codes and, seldom, its block's older codes.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.h"
#include "kv8.cuh"
#include "ptx.cuh"

namespace onpu_b200 {
namespace {

// rint(x / s) of the exact quotient, in [-127, 127]; inv = 1 / s, s > 0
__device__ __forceinline__ int kv8_code(float x, float s, float inv) {
    const float r = x * inv;
    float n = rintf(r);
    if (!(fabsf(r - n) <= 0.4999f)) n = static_cast<float>(rint(static_cast<double>(x) / static_cast<double>(s)));
    return static_cast<int>(fminf(fmaxf(n, -127.f), 127.f));
}
// rint(code * s_old / s) of the exact quotient; 0 <= s_old < s
__device__ __forceinline__ int kv8_recode(int code, float s_old, float s, float ratio) {
    const float r = static_cast<float>(code) * ratio;
    float n = rintf(r);
    if (!(fabsf(r - n) <= 0.4999f))
        n = static_cast<float>(rint(static_cast<double>(code) * static_cast<double>(s_old) / static_cast<double>(s)));
    return static_cast<int>(n);
}
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (a & 0xff) | ((b & 0xff) << 8) | ((c & 0xff) << 16) | (static_cast<uint32_t>(d) << 24);
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

constexpr int kAppendThreads = 256;

struct Kv8In {
    const void *x[2];                 // K rows, V rows
    int64_t ld[2];
};

// A group of G threads (a warp, or the CTA) writes one block of one head of K or V: NV vectors of 8 values
// per thread hold all of the block's new rows, so they are read once.
template <bool BF16, int G, int NV>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const Kv8Cache c, const Kv8Rows r, const Kv8In in,
                                                                    int nblk, int64_t groups) {
    pdl_launch_dependents();
    pdl_wait_prerequisites();
    __shared__ uint32_t red[kAppendThreads / 32];
    const int64_t gi = static_cast<int64_t>(blockIdx.x) * (kAppendThreads / G) + threadIdx.x / G;
    if (gi >= groups) return;                              // whole groups leave: G = 32, or one group a CTA
    const int tid = threadIdx.x % G;
    const int h = static_cast<int>(gi % c.Hkv), kv = static_cast<int>(gi / c.Hkv & 1);
    const int64_t bw = gi / c.Hkv / 2;
    const int b = static_cast<int>(bw / nblk), w = static_cast<int>(bw % nblk);
    int pos, cnt;
    if (!kv8_rows(r, b, c.S, pos, cnt)) return;
    const int blk = (pos >> c.blk_log2) + w, row0 = blk << c.blk_log2;      // this block and its first row
    const int lo = max(pos, row0), hi = min(pos + cnt, row0 + (1 << c.blk_log2));
    if (lo >= hi) return;
    const int vpr = c.D / 8, nvec = (hi - lo) * vpr;       // vectors per row, and in all
    const int64_t xb = (static_cast<int64_t>(b) * r.T + (lo - pos)) * in.ld[kv] + static_cast<int64_t>(h) * c.D;
    float f[NV][8];
    int rr[NV], cc[NV];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = tid + i * G;
        rr[i] = v / vpr;
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
    const float inv = 1.0f / s;
    int8_t *base = (kv ? c.v : c.k) + b * c.bs + h * c.hs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (tid + i * G < nvec) {
            int q[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = s > 0.f ? kv8_code(f[i][e], s, inv) : 0;
            *reinterpret_cast<uint2 *>(base + static_cast<int64_t>(lo + rr[i]) * c.rs + cc[i]) =
                make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
        }
    }
    if (s > s_old && row0 < pos) {                         // the block's older rows onto the larger scale
        const float ratio = s_old / s;
        const int nold = (pos - row0) * vpr;
        for (int v = tid; v < nold; v += G) {
            const int ro = v / vpr;
            uint2 *p = reinterpret_cast<uint2 *>(base + static_cast<int64_t>(row0 + ro) * c.rs + (v - ro * vpr) * 8);
            const uint2 o = *p;
            uint32_t n[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t x = k ? o.y : o.x;
                int q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) q[e] = kv8_recode(static_cast<int8_t>(x >> (8 * e)), s_old, s, ratio);
                n[k] = pack4(q[0], q[1], q[2], q[3]);
            }
            *p = make_uint2(n[0], n[1]);
        }
    }
    if (tid == 0) *sp = s;
}

template <bool BF16, int G, int NV>
cudaError_t append_t(const Kv8Cache &c, const Kv8Rows &r, const Kv8In &in, int nblk, cudaStream_t s) {
    const int64_t groups = static_cast<int64_t>(c.B) * nblk * 2 * c.Hkv;
    const int64_t ctas = (groups + kAppendThreads / G - 1) / (kAppendThreads / G);
    if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return launch_pdl(kv8_append_kernel<BF16, G, NV>, dim3(static_cast<unsigned>(ctas)), dim3(kAppendThreads), 0, s, c,
                      r, in, nblk, groups);
}

template <bool BF16>
cudaError_t append_f(const Kv8Cache &c, const Kv8Rows &r, const Kv8In &in, cudaStream_t s) {
    const int R = 1 << c.blk_log2;
    const int nblk = static_cast<int>((static_cast<int64_t>(r.T) + R - 2) / R + 1);   // blocks T rows can touch
    const int nvec = (r.T < R ? r.T : R) * c.D / 8;                                    // a block's new vectors
    if (nvec <= 32) return append_t<BF16, 32, 1>(c, r, in, nblk, s);
    if (nvec <= 128) return append_t<BF16, 32, 4>(c, r, in, nblk, s);
    if (nvec <= 512) return append_t<BF16, 256, 2>(c, r, in, nblk, s);
    if (nvec <= 1024) return append_t<BF16, 256, 4>(c, r, in, nblk, s);
    return append_t<BF16, 256, 8>(c, r, in, nblk, s);      // at most 64 rows of 256
}

// ---------------------------------------------------------------- read back
constexpr int kReadThreads = 256;

struct Kv8Out {
    void *y[2];
    int64_t ld[2];
};

// 8 codes a thread, in the order of the output: D values of a head, heads of a token, tokens
template <bool BF16>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(const Kv8Cache c, const Kv8Rows r, const Kv8Out out) {
    pdl_launch_dependents();
    pdl_wait_prerequisites();
    const int b = blockIdx.y >> 1, kv = blockIdx.y & 1, vpr = c.D / 8, vpt = vpr * c.Hkv;
    int pos, cnt;
    if (!kv8_rows(r, b, c.S, pos, cnt)) return;
    const int64_t nvec = static_cast<int64_t>(cnt) * vpt;
    const int8_t *base = (kv ? c.v : c.k) + b * c.bs;
    const float *sc = (kv ? c.vs : c.ks) + b * c.sbs;
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * kReadThreads + threadIdx.x; v < nvec;
         v += static_cast<int64_t>(gridDim.x) * kReadThreads) {
        const int i = static_cast<int>(v / vpt), hd = static_cast<int>(v - static_cast<int64_t>(i) * vpt);
        const int h = hd / vpr, d = (hd - h * vpr) * 8, row = pos + i;
        const uint2 q = *reinterpret_cast<const uint2 *>(base + h * c.hs + static_cast<int64_t>(row) * c.rs + d);
        const float s = sc[h * c.shs + (row >> c.blk_log2)];
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? q.x : q.y) >> (8 * (e & 3)))) * s;
        const int64_t o = (static_cast<int64_t>(b) * r.T + i) * out.ld[kv] + static_cast<int64_t>(h) * c.D + d;
        if constexpr (BF16) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
                w[e] = *reinterpret_cast<const uint32_t *>(&t);
            }
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out.y[kv]) + o) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            float4 *y = reinterpret_cast<float4 *>(static_cast<float *>(out.y[kv]) + o);
            y[0] = make_float4(f[0], f[1], f[2], f[3]);
            y[1] = make_float4(f[4], f[5], f[6], f[7]);
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
    const int64_t nvec = static_cast<int64_t>(r.T) * c.Hkv * c.D / 8;
    const int64_t ctas = (nvec + kReadThreads - 1) / kReadThreads;
    const dim3 grid(static_cast<unsigned>(ctas < 0x7fffffff ? ctas : 0x7fffffff), 2 * c.B);
    return bf16 ? launch_pdl(kv8_read_kernel<true>, grid, dim3(kReadThreads), 0, stream, c, r, out)
                : launch_pdl(kv8_read_kernel<false>, grid, dim3(kReadThreads), 0, stream, c, r, out);
}

}  // namespace onpu_b200
