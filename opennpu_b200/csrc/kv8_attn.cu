// Attention over the 8-bit KV cache (kv8.cu): query i of a sequence stands at cache row pos + i and sees rows
// 0 .. pos + i,
//   x_j = scale q . (c_j s_b(j)) + mask_j,   out = sum_j e^(x_j) v_j / (sum_j e^(x_j) + e^sink),
// with an online softmax in fp32; a query whose mask leaves no row gives zeros.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "kernels.h"
#include "kv8.cuh"
#include "ptx.cuh"

namespace onpu_b200 {
namespace {

constexpr int kWarps = 8;

// one CTA per (query, head): each warp takes every eighth row, a lane D / 32 values (at most 8)
template <bool BF16>
__global__ void __launch_bounds__(kWarps * 32) kv8_attn_simple_kernel(const Kv8AttnParams p) {
    pdl_launch_dependents();
    pdl_wait_prerequisites();
    __shared__ float sm[kWarps], sl[kWarps], so[kWarps][256];
    const Kv8Cache &c = p.c;
    const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z, kh = h / (p.Hq / c.Hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = c.D;
    int pos, cnt;
    if (!kv8_rows(p.r, b, c.S, pos, cnt) || i >= cnt) return;
    const int64_t qo = (static_cast<int64_t>(b) * p.r.T + i) * p.ldq + static_cast<int64_t>(h) * D;
    float q[8], o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int d = lane + 32 * e;
        q[e] = d >= D ? 0.f : BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p.q)[qo + d])
                                   : static_cast<const float *>(p.q)[qo + d];
        o[e] = 0.f;
    }
    const int8_t *K = c.k + b * c.bs + kh * c.hs, *V = c.v + b * c.bs + kh * c.hs;
    const float *ks = c.ks + b * c.sbs + kh * c.shs, *vs = c.vs + b * c.sbs + kh * c.shs;
    float m = -INFINITY, l = 0.f;
    for (int j = warp; j <= pos + i; j += kWarps) {
        const float mk = p.mask ? p.mask[b * p.mbs + i * p.mts + j] : 0.f;
        if (mk == -INFINITY) continue;
        const int8_t *kr = K + static_cast<int64_t>(j) * c.rs, *vr = V + static_cast<int64_t>(j) * c.rs;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < D) s = fmaf(q[e], static_cast<float>(kr[lane + 32 * e]), s);
#pragma unroll
        for (int k = 16; k; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
        const float x = s * ks[j >> c.blk_log2] * p.scale + mk;
        const float mn = fmaxf(m, x), a = m == -INFINITY ? 0.f : expf(m - mn), w = mn == -INFINITY ? 0.f : expf(x - mn);
        m = mn;
        l = l * a + w;
        const float wv = w * vs[j >> c.blk_log2];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < D) o[e] = fmaf(wv, static_cast<float>(vr[lane + 32 * e]), o[e] * a);
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) so[warp][lane + 32 * e] = o[e];
    __syncthreads();
    const float sink = p.sinks ? p.sinks[h] : -INFINITY;
    float mx = sink;
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm[w]);
    const int64_t oo = (static_cast<int64_t>(b) * p.r.T + i) * p.ldo + static_cast<int64_t>(h) * D;
    for (int d = threadIdx.x; d < D; d += kWarps * 32) {
        float y = 0.f, t = mx == -INFINITY ? 0.f : expf(sink - mx);
        for (int w = 0; w < kWarps; ++w) {
            if (sm[w] == -INFINITY) continue;
            const float a = expf(sm[w] - mx);
            t = fmaf(sl[w], a, t);
            y = fmaf(so[w][d], a, y);
        }
        y = t == 0.f ? 0.f : y / t;
        if (BF16) static_cast<__nv_bfloat16 *>(p.out)[oo + d] = __float2bfloat16_rn(y);
        else static_cast<float *>(p.out)[oo + d] = y;
    }
}

}  // namespace

int64_t kv8_attn_ws_bytes(int, int, int, int, bool) { return 16; }

cudaError_t kv8_attn_launch(const Kv8AttnParams &p, bool bf16, cudaStream_t stream) {
    const dim3 grid(p.Hq, p.r.T, p.c.B);
    return bf16 ? launch_pdl(kv8_attn_simple_kernel<true>, grid, dim3(kWarps * 32), 0, stream, p)
                : launch_pdl(kv8_attn_simple_kernel<false>, grid, dim3(kWarps * 32), 0, stream, p);
}

}  // namespace onpu_b200
