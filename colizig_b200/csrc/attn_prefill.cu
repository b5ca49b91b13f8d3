// Causal attention over packed prompts: query i of sequence b (nq queries, nk keys,
// aligned at their ends) sees the keys j <= i + nk - nq;
//   out = sum_j p_j v_j,  p = softmax_j(scale q . k_j),  zeros when it sees none.
// One warp per (query, head), running maximum and sum of the softmax in f32.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cz_common.cuh"
#include "cz_internal.h"

namespace cz {
namespace {

constexpr int kWarps = 4;

template <int D>
__global__ void __launch_bounds__(kWarps * 32) attn_prefill_kernel(const AttnPrefillParams p) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    const uint64_t item = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (item >= (uint64_t)p.Tq * p.q_heads) return;
    const int t = (int)(item / p.q_heads);
    const uint32_t h = (uint32_t)(item % p.q_heads), kh = h / (p.q_heads / p.kv_heads);
    int b = 0;
    while (b < p.B && __ldg(p.cu_q + b + 1) <= t) ++b;
    int n = 0, k0 = 0;
    if (b < p.B) {
        const int q0 = __ldg(p.cu_q + b), q1 = __ldg(p.cu_q + b + 1);
        k0 = __ldg(p.cu_k + b);
        const int k1 = __ldg(p.cu_k + b + 1);
        if (q0 < 0 || q1 > p.Tq || k0 < 0 || k1 < k0 || k1 > p.Tk) {
            if (lane == 0) atomicOr(p.err, kAttnErrIndex);
        } else {
            n = t - q0 + 1 + (k1 - k0) - (q1 - q0);
        }
    }
    float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = bf16_bits_to_f32(__ldg(p.q + t * p.q_stride + (uint64_t)h * D + lane * N + i));
        o[i] = 0.f;
    }
    for (int j = 0; j < n; ++j) {
        const uint16_t* kr = p.k + (uint64_t)(k0 + j) * p.k_stride + (uint64_t)kh * D + lane * N;
        const uint16_t* vr = p.v + (uint64_t)(k0 + j) * p.v_stride + (uint64_t)kh * D + lane * N;
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) d = __fmaf_rn(q[i], bf16_bits_to_f32(__ldg(kr + i)), d);
        const float s = warp_sum(d) * p.scale;
        const float mn = fmaxf(m, s), a = m == mn ? 1.f : expf(m - mn), w = s == mn ? 1.f : expf(s - mn);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = __fmaf_rn(w, bf16_bits_to_f32(__ldg(vr + i)), o[i] * a);
        l = __fmaf_rn(l, a, w);
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const __nv_bfloat16 v = __float2bfloat16_rn(l > 0.f ? o[i] / l : 0.f);
        p.out[((uint64_t)t * p.q_heads + h) * D + lane * N + i] = *reinterpret_cast<const uint16_t*>(&v);
    }
}

}  // namespace

int attn_prefill_launch(const AttnPrefillParams& p, int, cudaStream_t st) {
    const uint32_t grid = (uint32_t)(((uint64_t)p.Tq * p.q_heads + kWarps - 1) / kWarps);
    if (p.head_dim == 128)
        attn_prefill_kernel<128><<<grid, kWarps * 32, 0, st>>>(p);
    else
        attn_prefill_kernel<64><<<grid, kWarps * 32, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? CZ_OK : CZ_ELAUNCH;
}

}  // namespace cz
