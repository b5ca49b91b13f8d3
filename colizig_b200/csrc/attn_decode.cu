// Attention of one new token per sequence over the paged cache:
//   out[b,h] = sum_j p_j v_j,  p = softmax_j(scale q[b,h] . k_j),  j < lens[b].
// One warp per (sequence, query head) with the running maximum m and sum l of
// the softmax in f32: o <- o 2^(m - m') + 2^(s_j - m') v_j in one pass over the
// cache.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cz_common.cuh"
#include "cz_internal.h"

namespace cz {
namespace {

constexpr int kWarps = 4;

template <int N>
__device__ __forceinline__ void load_row(const uint8_t* base, uint64_t at, int e4m3, float* f) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        f[i] = e4m3 ? e4m3x2_to_f32x2((uint16_t)__ldg(base + at + i)).x
                    : bf16_bits_to_f32(__ldg(reinterpret_cast<const uint16_t*>(base) + at + i));
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32) attn_decode_kernel(const AttnDecodeParams p) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    const uint64_t item = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (item >= (uint64_t)p.B * p.q_heads) return;
    const uint32_t b = (uint32_t)(item / p.q_heads), h = (uint32_t)(item % p.q_heads);
    const uint32_t kh = h / (p.q_heads / p.kv.kv_heads);
    int n = __ldg(p.lens + b);
    if (n < 0 || (uint64_t)n > (uint64_t)p.table_width * p.kv.page_size) {
        if (lane == 0) atomicOr(p.err, kAttnErrIndex);
        n = n < 0 ? 0 : (int)(p.table_width * p.kv.page_size);
    }
    const float ks = p.kv.k_scale ? __ldg(p.kv.k_scale + kh) : 1.f;
    const float vs = p.kv.v_scale ? __ldg(p.kv.v_scale + kh) : 1.f;
    float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = bf16_bits_to_f32(__ldg(p.q + b * p.q_stride + (uint64_t)h * D + lane * N + i)) * p.scale;
        o[i] = 0.f;
    }
    for (int j = 0; j < n; ++j) {
        const int page = __ldg(p.table + b * p.table_stride + j / p.kv.page_size);
        if (page < 0 || (uint32_t)page >= p.kv.pages) {
            if (lane == 0) atomicOr(p.err, kAttnErrIndex);
            continue;
        }
        const uint64_t at = ((uint64_t)kh * p.kv.page_size + j % p.kv.page_size) * D + lane * N;
        float x[N], d = 0.f;
        load_row<N>(p.kv.k, page * p.kv.k_page + at, p.kv.e4m3, x);
#pragma unroll
        for (int i = 0; i < N; ++i) d = __fmaf_rn(q[i], x[i], d);
        const float s = warp_sum(d) * ks;
        const float mn = fmaxf(m, s), a = m == mn ? 1.f : expf(m - mn), w = s == mn ? 1.f : expf(s - mn);
        load_row<N>(p.kv.v, page * p.kv.v_page + at, p.kv.e4m3, x);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = __fmaf_rn(w, x[i], o[i] * a);
        l = __fmaf_rn(l, a, w);
        m = mn;
    }
    const float r = l > 0.f ? vs / l : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const __nv_bfloat16 v = __float2bfloat16_rn(l > 0.f ? o[i] * r : 0.f);
        p.out[((uint64_t)b * p.q_heads + h) * D + lane * N + i] = *reinterpret_cast<const uint16_t*>(&v);
    }
}

}  // namespace

size_t attn_decode_workspace_bytes(int) { return 256; }

int attn_decode_launch(const AttnDecodeParams& p, int, cudaStream_t st) {
    const uint32_t grid = (uint32_t)(((uint64_t)p.B * p.q_heads + kWarps - 1) / kWarps);
    if (p.kv.head_dim == 128)
        attn_decode_kernel<128><<<grid, kWarps * 32, 0, st>>>(p);
    else
        attn_decode_kernel<64><<<grid, kWarps * 32, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? CZ_OK : CZ_ELAUNCH;
}

}  // namespace cz
