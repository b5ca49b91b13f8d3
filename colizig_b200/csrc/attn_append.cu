// Norm, position rotation and cache write of a step's q/k/v projections (the
// part of the decoder layer between src/qwen3moe/attn.zig:46-78's q/k/v and the
// attention itself).  Per token and head x[D]:
//   y = x / sqrt(mean(x^2) + eps) * w                          (q and k, when w is given)
//   y[i], y[i+R/2] = y[i] c_i - y[i+R/2] s_i, y[i+R/2] c_i + y[i] s_i,   i < R/2
// with c, s read from the caller's table (made from 64-bit angles: an f32 angle
// of position 1e5 is off by 4e-3 in the fastest pair, more than bf16 resolves).
// All arithmetic is f32; one rounding at the store (bf16, or E4M3 of x / scale,
// saturated), which is the cache's own type.
//
// D / 8 lanes share a head, 8 elements each (two 16-byte loads of f32 or one of
// bf16, one 16-byte store); the sum of squares and the rotation partner, R/2
// elements away = R/16 lanes, go through shuffles, so nothing is staged.  A
// group of lanes takes kHeads heads of one token, whose loads are all in
// flight together and share the token's cosines and sines in registers.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cz_common.cuh"
#include "cz_internal.h"

namespace cz {
namespace {

constexpr int kThreads = 256;

template <int XBF16>
__device__ __forceinline__ void load8(const void* base, uint64_t at, float* f) {
    if (XBF16) {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + at));
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
        const float4 a = __ldg(s), b = __ldg(s + 1);
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
        f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
}

__device__ __forceinline__ uint4 pack_bf16x8(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// E4M3 of x / scale, saturated at +-448 (NaN stays NaN).
__device__ __forceinline__ uint2 pack_e4m3x8(const float* f, float scale) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t u = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 v = make_float2(__fdiv_rn(f[4 * i + 2 * j], scale), __fdiv_rn(f[4 * i + 2 * j + 1], scale));
            u |= (uint32_t)__nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3) << (16 * j);
        }
        w[i] = u;
    }
    return make_uint2(w[0], w[1]);
}

// D: head size; XBF16: projections are bf16; HEADS: heads of one token per group of lanes.
template <int D, int XBF16, int HEADS>
__global__ void __launch_bounds__(kThreads) attn_append_kernel(const AppendParams p) {
    constexpr int L = D / 8;
    const int sub = threadIdx.x % L;
    const uint32_t hq = p.q_heads, hk = p.kv.kv_heads;
    const uint32_t per_token = (hq + 2 * hk + HEADS - 1) / HEADS;  // groups of lanes
    const uint64_t item = (uint64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;
    const bool live = item < (uint64_t)p.T * per_token;  // the whole group agrees; dead groups still join the shuffles
    const uint32_t t = live ? (uint32_t)(item / per_token) : 0;
    const uint32_t g = live ? (uint32_t)(item % per_token) : 0;

    float f[HEADS][8];
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
        const uint32_t h = g + j * per_token;
        if (!live || h >= hq + 2 * hk) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[j][i] = 0.f;
        } else if (h < hq) {
            load8<XBF16>(p.q, t * p.q_stride + (uint64_t)h * D + sub * 8, f[j]);
        } else if (h < hq + hk) {
            load8<XBF16>(p.k, t * p.k_stride + (uint64_t)(h - hq) * D + sub * 8, f[j]);
        } else {
            load8<XBF16>(p.v, t * p.v_stride + (uint64_t)(h - hq - hk) * D + sub * 8, f[j]);
        }
    }
    // this lane's cosines and sines: elements 8 sub .. 8 sub + 7 lie in one half of the
    // rotated part (R/2 is a multiple of 8); outside it c = 1, s = 0
    float c[8], s[8];
    const int half = (int)p.rot / 2;
    const int e0 = sub * 8;
    const bool turned = p.rot != 0 && e0 < (int)p.rot;
    const bool upper = turned && e0 >= half;
    const int partner = !turned ? sub : upper ? sub - half / 8 : sub + half / 8;
    if (turned) {
        int pos = live ? __ldg(p.positions + t) : 0;
        if (pos < 0 || (uint32_t)pos >= p.rope_len) {
            atomicOr(p.err, kAttnErrIndex);
            pos = 0;
        }
        const float* row = p.rope + (uint64_t)pos * p.rot + (e0 - (upper ? half : 0));
        load8<0>(row, 0, c);
        load8<0>(row, half, s);
        if (!upper) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = -s[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
    }
    const int64_t slot = live ? __ldg(p.slots + t) : -1;
    const bool in_cache = slot >= 0 && slot < (int64_t)p.kv.pages * p.kv.page_size;
    if (slot >= 0 && !in_cache && sub == 0) atomicOr(p.err, kAttnErrIndex);
    const uint64_t page = in_cache ? (uint64_t)slot / p.kv.page_size : 0;
    const uint64_t row = in_cache ? (uint64_t)slot % p.kv.page_size : 0;

#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
        const uint32_t h = g + j * per_token;
        const bool is_v = h >= hq + hk;
        const float* w = h < hq ? p.q_norm : is_v ? nullptr : p.k_norm;
        float y[8];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __fmaf_rn(f[j][i], f[j][i], ss);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        float wv[8];
        if (w) {
            load8<0>(w, e0, wv);
            const float r = 1.f / sqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = f[j][i] * r * wv[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = f[j][i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float o = __shfl_sync(0xffffffffu, y[i], partner, L);
            if (!is_v && turned) y[i] = __fmaf_rn(o, s[i], y[i] * c[i]);
        }
        if (!live || h >= hq + 2 * hk) continue;
        if (h < hq) {
            *reinterpret_cast<uint4*>(p.q_out + ((uint64_t)t * hq + h) * D + e0) = pack_bf16x8(y);
            continue;
        }
        const uint32_t kh = is_v ? h - hq - hk : h - hq;
        uint16_t* packed = is_v ? p.v_out : p.k_out;
        const uint4 b = pack_bf16x8(y);
        if (packed) *reinterpret_cast<uint4*>(packed + ((uint64_t)t * hk + kh) * D + e0) = b;
        if (!in_cache) continue;
        const uint64_t at = page * (is_v ? p.kv.v_page : p.kv.k_page) + ((uint64_t)kh * p.kv.page_size + row) * D + e0;
        uint8_t* base = is_v ? p.kv.v : p.kv.k;
        if (p.kv.e4m3) {
            const float* sc = is_v ? p.kv.v_scale : p.kv.k_scale;
            *reinterpret_cast<uint2*>(base + at) = pack_e4m3x8(y, sc ? __ldg(sc + kh) : 1.f);
        } else {
            *reinterpret_cast<uint4*>(base + at * 2) = b;
        }
    }
}

template <int D, int XBF16>
void launch(const AppendParams& p, cudaStream_t st) {
    constexpr int H = 4;
    const uint64_t items = (uint64_t)p.T * ((p.q_heads + 2 * p.kv.kv_heads + H - 1) / H);
    const uint32_t per = kThreads / (D / 8);
    attn_append_kernel<D, XBF16, H><<<(uint32_t)((items + per - 1) / per), kThreads, 0, st>>>(p);
}

}  // namespace

int attn_append_launch(const AppendParams& p, cudaStream_t st) {
    if (p.kv.head_dim == 128)
        p.x_bf16 ? launch<128, 1>(p, st) : launch<128, 0>(p, st);
    else
        p.x_bf16 ? launch<64, 1>(p, st) : launch<64, 0>(p, st);
    return cudaGetLastError() == cudaSuccess ? CZ_OK : CZ_ELAUNCH;
}

}  // namespace cz
