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
// D / 8 lanes share a head.  A lane holds four consecutive elements and the four they are
// turned with (R/2 further on; beyond the rotated part, two runs of four that are left as they
// are), so that the rotation needs no exchange and a lane reads four cosines and four sines;
// only the sum of squares goes through shuffles.  A group of lanes takes four heads of one
// token (two when that would leave SMs without a block), whose loads are all in flight together
// and share the cosines and sines.
//
// Bound by memory: 8,192 tokens of 32 + 2 x 4 heads of 128 in f32 to bf16, with packed copies, are 272 MB
// and take 54.9 us, 4.96 TB/s (0.77 of a copy's rate).  Four heads against two: 54.9 and 55.8 us there,
// 5.4 and 6.2 us for 1,531 tokens of 16 + 32 heads of 64 in bf16; for 96 tokens 3.9 and 3.1 us, for one 3.1
// and 2.4 us.  The launch bounds make each instance spill 24 to 80 bytes a thread; two blocks fewer an SM spill
// nothing, but take 59.4 and 6.5 us (one token 2.2, 96 tokens 2.9): more loads in flight are worth more.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cz_common.cuh"
#include "cz_internal.h"

namespace cz {
namespace {

constexpr int kThreads = 128;

// Four elements, read once: not kept in L1 (the rotation table is).
template <int XBF16>
__device__ __forceinline__ void load4(const void* base, uint64_t at, float* f) {
    if (XBF16) {
        uint2 r;
        asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
                     : "=r"(r.x), "=r"(r.y)
                     : "l"(reinterpret_cast<const uint16_t*>(base) + at));
        f[0] = __uint_as_float(r.x << 16), f[1] = __uint_as_float(r.x & 0xffff0000u);
        f[2] = __uint_as_float(r.y << 16), f[3] = __uint_as_float(r.y & 0xffff0000u);
    } else {
        asm volatile("ld.global.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3])
                     : "l"(reinterpret_cast<const float*>(base) + at));
    }
}

__device__ __forceinline__ float4 ldg4(const float* p) { return ld_now(reinterpret_cast<const float4*>(p)); }

__device__ __forceinline__ uint2 pack_bf16x4(const float* f) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// E4M3 of x / scale, saturated at +-448 (NaN stays NaN).
__device__ __forceinline__ uint32_t pack_e4m3x4(const float* f, float scale) {
    uint32_t u = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float2 v = make_float2(__fdiv_rn(f[2 * j], scale), __fdiv_rn(f[2 * j + 1], scale));
        u |= (uint32_t)__nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3) << (16 * j);
    }
    return u;
}

// D: head size; XBF16: projections are bf16; HEADS: heads of one token per group of lanes.
template <int D, int XBF16, int HEADS>
__global__ void __launch_bounds__(kThreads, HEADS == 4 ? 8 : 10) attn_append_kernel(const AppendParams p) {
    constexpr int L = D / 8;
    const int sub = threadIdx.x % L;
    pdl_wait();
    const uint32_t hq = p.q_heads, hk = p.kv.kv_heads;
    const uint32_t per_token = (hq + 2 * hk + HEADS - 1) / HEADS;  // groups of lanes
    const uint32_t item = blockIdx.x * (kThreads / L) + threadIdx.x / L;
    const bool live = item < (uint32_t)p.T * per_token;  // the whole group agrees; dead groups still join the shuffles
    const uint32_t t = live ? item / per_token : 0;
    const uint32_t g = live ? item % per_token : 0;
    // this lane's two runs of four
    const int rot = (int)p.rot, turning = rot / 8;  // lanes of the rotated part
    const bool turned = sub < turning;
    const int e0 = turned ? 4 * sub : rot + 4 * (sub - turning);
    const int e1 = e0 + (turned ? rot : D - rot) / 2;

    int pos = turned && live ? ld_now(p.positions + t) : 0;
    const int64_t slot = live ? ld_now(p.slots + t) : -1;
    float f[HEADS][8];
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
        const uint32_t h = g + j * per_token;
        const bool some = live && h < hq + 2 * hk;
        const void* x = h < hq ? p.q : h < hq + hk ? p.k : p.v;
        const uint64_t at = h < hq        ? t * p.q_stride + (uint64_t)h * D
                            : h < hq + hk ? t * p.k_stride + (uint64_t)(h - hq) * D
                                          : t * p.v_stride + (uint64_t)(h - hq - hk) * D;
        if (some) {
            load4<XBF16>(x, at + e0, f[j]);
            load4<XBF16>(x, at + e1, f[j] + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[j][i] = 0.f;
        }
    }
    float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (turned) {
        if (pos < 0 || (uint32_t)pos >= p.rope_len) {
            atomicOr(p.err, kAttnErrIndex);
            pos = 0;
        }
        const float* row = p.rope + (uint64_t)pos * rot + e0;
        c = ldg4(row);
        s = ldg4(row + rot / 2);
    }
    const bool in_cache = slot >= 0 && slot < (int64_t)p.kv.pages * p.kv.page_size;
    if (slot >= 0 && !in_cache && sub == 0) atomicOr(p.err, kAttnErrIndex);
    const uint32_t page = in_cache ? (uint32_t)slot / p.kv.page_size : 0;  // (a cache has fewer than 2^32 rows)
    const uint32_t row = in_cache ? (uint32_t)slot - page * p.kv.page_size : 0;

#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
        const uint32_t h = g + j * per_token;
        const bool is_v = h >= hq + hk;
        float* y = f[j];
        const float* w = h < hq ? p.q_norm : is_v ? nullptr : p.k_norm;
        if (p.q_norm || p.k_norm) {  // (all lanes agree, for the shuffles)
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __fmaf_rn(y[i], y[i], ss);
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (w) {
                const float4 w0 = ldg4(w + e0), w1 = ldg4(w + e1);
                const float r = 1.f / sqrtf(ss * (1.f / D) + p.eps);
                y[0] *= r * w0.x, y[1] *= r * w0.y, y[2] *= r * w0.z, y[3] *= r * w0.w;
                y[4] *= r * w1.x, y[5] *= r * w1.y, y[6] *= r * w1.z, y[7] *= r * w1.w;
            }
        }
        if (!is_v && turned) {
            const float cc[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = y[i], b = y[i + 4];
                y[i] = __fmaf_rn(a, cc[i], -b * sn[i]);
                y[i + 4] = __fmaf_rn(b, cc[i], a * sn[i]);
            }
        }
        if (!live || h >= hq + 2 * hk) continue;
        const uint2 lo = pack_bf16x4(y), hi = pack_bf16x4(y + 4);
        if (h < hq) {
            uint16_t* dst = p.q_out + ((uint64_t)t * hq + h) * D;
            *reinterpret_cast<uint2*>(dst + e0) = lo;
            *reinterpret_cast<uint2*>(dst + e1) = hi;
            continue;
        }
        const uint32_t kh = is_v ? h - hq - hk : h - hq;
        uint16_t* packed = is_v ? p.v_out : p.k_out;
        if (packed) {
            packed += ((uint64_t)t * hk + kh) * D;
            *reinterpret_cast<uint2*>(packed + e0) = lo;
            *reinterpret_cast<uint2*>(packed + e1) = hi;
        }
        if (!in_cache) continue;
        const uint64_t at = (uint64_t)page * (is_v ? p.kv.v_page : p.kv.k_page) + ((uint64_t)kh * p.kv.page_size + row) * D;
        uint8_t* base = is_v ? p.kv.v : p.kv.k;
        if (p.kv.e4m3) {
            const float* sc = is_v ? p.kv.v_scale : p.kv.k_scale;
            const float scale = sc ? ld_now(sc + kh) : 1.f;
            *reinterpret_cast<uint32_t*>(base + at + e0) = pack_e4m3x4(y, scale);
            *reinterpret_cast<uint32_t*>(base + at + e1) = pack_e4m3x4(y + 4, scale);
        } else {
            *reinterpret_cast<uint2*>(base + (at + e0) * 2) = lo;
            *reinterpret_cast<uint2*>(base + (at + e1) * 2) = hi;
        }
    }
}

template <int D, int XBF16>
int launch(const AppendParams& p, int num_sms, cudaStream_t st) {
    const uint32_t heads = p.q_heads + 2 * p.kv.kv_heads, per = kThreads / (D / 8);
    const uint64_t four = ((uint64_t)p.T * ((heads + 3) / 4) + per - 1) / per;
    const uint64_t two = ((uint64_t)p.T * ((heads + 1) / 2) + per - 1) / per;
    if (two * per >= 0xffff0000u) return CZ_ESHAPE;  // (counted in 32 bits)
    const bool ok = four >= 2 * (uint64_t)num_sms
                        ? launch_early(attn_append_kernel<D, XBF16, 4>, (uint32_t)four, kThreads, 0, st, p)
                        : launch_early(attn_append_kernel<D, XBF16, 2>, (uint32_t)two, kThreads, 0, st, p);
    return ok ? CZ_OK : CZ_ELAUNCH;
}

}  // namespace

int attn_append_launch(const AppendParams& p, int num_sms, cudaStream_t st) {
    if (p.kv.head_dim == 128) return p.x_bf16 ? launch<128, 1>(p, num_sms, st) : launch<128, 0>(p, num_sms, st);
    return p.x_bf16 ? launch<64, 1>(p, num_sms, st) : launch<64, 0>(p, num_sms, st);
}

}  // namespace cz
