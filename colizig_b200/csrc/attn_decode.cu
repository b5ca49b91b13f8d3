// Attention of one new token per sequence over the paged cache:
//   out[b,h] = sum_j p_j v_j,  p = softmax_j(scale q[b,h] . k_j),  j < lens[b],
// in one pass with a running maximum m and sum l (f32):
//   o <- o 2^(m - m') + sum_j 2^(t_j - m') v_j,  t_j = scale log2(e) q.k_j,  out = o / l.
//
// Bound by reading the cache once.  The G query heads of a key/value head are
// the columns of one matrix tile, so a key or value row is read once for all of
// them:  S^T[16 keys x 8 heads] = K q^T and O^T[16 dims x 8 heads] += V^T P^T
// with mma.m16n8k16.  Keys (not heads) on the 16-row side: a group of 8 heads
// fills the tile, where the other way round half of it would be padding; P^T
// moves from accumulator to operand layout with two movmatrix.  tcgen05 would
// want 128 rows for 8 used ones, and the tensor pipe is idle either way.
//
// Work split.  The cache of all (sequence, key/value head) pairs is one long line
// of 64-key units, cut into equal parts, one per SM, whatever the lengths are (read
// on the device, so a captured graph follows them).  A part may end inside a pair:
// its partial (o, m, l) then goes to the workspace and the last CTA of the pair to
// arrive joins the parts in order, so results do not depend on timing.
//
// In a CTA, 8 warps take the segment's steps in turn, each with a ring of its own
// (3 stages of 8 KB of keys and values, TMA boxes of 16 rows, page numbers looked
// up one batch ahead): nothing but the join at a segment's end synchronises them,
// and the rings run on across segments.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cz_common.cuh"
#include "cz_internal.h"

namespace cz {
namespace {

constexpr int kWarps = 8;
constexpr int kStages = 3;
constexpr int kStageBytes = 8192;  // keys, then values, of one step
constexpr int kUnit = 64;          // keys per unit of the work split
// A CTA takes at least this many units where that leaves CTAs idle: below 256 keys the
// join over the workspace costs more than the shorter loop gains.
constexpr int kMinUnits = 4;
constexpr int kMaxTiles = 2;       // 8-head column tiles per pass
constexpr int kSlotFloats = kMaxTiles * 8 * 128 + kMaxTiles * 8 * 2;  // o, then (m, l) per head

struct DecodeArgs {
    CUtensorMap kmap, vmap;  // [pages][kv_heads][page_size][head_dim], boxes of 16 rows x up to 128 bytes
    AttnDecodeParams p;
    uint32_t group, tiles;   // query heads per kv head; passes of NT * 8 of them
    float* slots;            // workspace: [grid][2][kSlotFloats]
    uint32_t* counters;      // workspace: [grid] arrivals at the pair that begins in this CTA and goes on
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void tma4d(uint32_t dst, const CUtensorMap* m, int x, int row, int head, int page,
                                      uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
template <bool F16>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if (F16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two E4M3 bytes -> two f16 (exact).
__device__ __forceinline__ uint32_t cvt_e4m3x2(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return h;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (F16)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The length of sequence b, bounded by its page table.
__device__ __forceinline__ int seq_len(const AttnDecodeParams& p, int b) {
    const int n = __ldg(p.lens + b);
    const int most = (int)(p.table_width * p.kv.page_size);
    return n < 0 ? 0 : n > most ? most : n;
}
__device__ __forceinline__ uint32_t units_of(int n) { return (uint32_t)(n + kUnit - 1) / kUnit; }

// Walks this CTA's part [pos, end) of the line.  The line holds, sequence by sequence,
// `items` stretches (kv heads x passes) of units_of(len) units each, rounded up to
// whole kMinUnits when `pad`.
struct Walk {
    uint32_t pos, end, off;  // place on the line; units of the current item before it
    int b, item, len;
    uint32_t n, npad;

    __device__ void enter(const AttnDecodeParams& p, int bb, bool pad) {
        for (b = bb; b < p.B; ++b) {
            len = seq_len(p, b);
            if (len > 0) break;
        }
        n = b < p.B ? units_of(len) : 0;
        npad = pad ? (n + kMinUnits - 1) / kMinUnits * kMinUnits : n;
    }
    // The next stretch with keys in it: tokens [t0, t1) of (b, item).  start = the item's own
    // place on the line.  False at the part's end.
    __device__ bool next(const AttnDecodeParams& p, int items, bool pad, int& sb, int& sitem, int& t0, int& t1,
                         uint32_t& start, uint32_t& sn) {
        while (pos < end && b < p.B) {
            const uint32_t u0 = off, take = min(npad - off, end - pos), u1 = min(u0 + take, n);
            sb = b;
            sitem = item;
            t0 = (int)(u0 * kUnit);
            t1 = min(len, (int)(u1 * kUnit));
            start = pos - u0;
            sn = n;
            pos += take;
            off += take;
            if (off == npad) {
                off = 0;
                if (++item == items) {
                    item = 0;
                    enter(p, b + 1, pad);
                }
            }
            if (u1 > u0) return true;
        }
        return false;
    }
};

template <int D, bool F8, int NT>
struct Cfg {
    static constexpr int ROWB = D * (F8 ? 1 : 2);
    static constexpr int BOXB = ROWB < 128 ? ROWB : 128;
    static constexpr int NBX = ROWB / BOXB;
    static constexpr int TS = kStageBytes / 2 / ROWB;  // keys per step
    static constexpr int NSUB = TS / 16;
    static constexpr int BOX = 16 * BOXB;
    static constexpr int JROW = D + 4;
    static constexpr int RING = kWarps * kStages * kStageBytes;
    static constexpr int JOIN = kWarps * 8 * JROW * 4;
};

// Byte offset of 16-byte chunk c of row r (0..15) in a sub-tile: boxes of 16 rows, TMA's
// 128- or 64-byte swizzle.
template <int BOXB>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    if (BOXB == 128) return (uint32_t)((c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

template <int D, bool F8, int NT>
__global__ void __launch_bounds__(kWarps * 32, 1) attn_decode_kernel(const __grid_constant__ DecodeArgs A) {
    using C = Cfg<D, F8, NT>;
    constexpr int KS = D / 16;  // k-steps of q.k, and 16-dim tiles of the output
    const AttnDecodeParams& p = A.p;
    extern __shared__ uint8_t raw[];
    uint8_t* base = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    float* join = reinterpret_cast<float*>(base + C::RING);           // [warp][8][JROW]; the prologue's prefix before
    float* stat = join + kWarps * 8 * C::JROW;                        // [warp][8][2]
    __shared__ uint64_t full[kWarps][kStages];
    __shared__ uint32_t scan[kWarps + 1];
    __shared__ int abort_flag, never;
    __shared__ uint32_t last_flag;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t4 = lane & 3;
    const int items = (int)(p.kv.kv_heads * A.tiles);

    if (tid == 0) abort_flag = never = 0;
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], 1);
        fence_mbarrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tensormap(&A.kmap);
        prefetch_tensormap(&A.vmap);
    }

    // ---- this CTA's part of the line ----
    uint32_t* prefix = reinterpret_cast<uint32_t*>(join);  // units before each sequence (one item's)
    uint32_t total = 0;
    bool pad = false;
    for (int round = 0; round < 2; ++round) {
        const int per = (p.B + kWarps * 32 - 1) / (kWarps * 32);
        uint32_t mine = 0;
        for (int i = 0; i < per; ++i) {
            const int b = tid * per + i;
            if (b >= p.B) break;
            const int n = seq_len(p, b);
            if (round == 0 && blockIdx.x == 0 && __ldg(p.lens + b) != n) atomicOr(p.err, kAttnErrIndex);
            const uint32_t u = units_of(n);
            mine += pad ? (u + kMinUnits - 1) / kMinUnits * kMinUnits : u;
        }
        uint32_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = inc;
        __syncthreads();
        uint32_t before = inc - mine;
        total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += scan[w];
            total += scan[w];
        }
        for (int i = 0; i < per; ++i) {
            const int b = tid * per + i;
            if (b >= p.B) break;
            prefix[b] = before;
            const uint32_t u = units_of(seq_len(p, b));
            before += pad ? (u + kMinUnits - 1) / kMinUnits * kMinUnits : u;
        }
        total *= items;
        if (pad || (total + gridDim.x - 1) / gridDim.x >= kMinUnits) break;
        pad = true;  // little work: whole kMinUnits per item, so that short caches are not split
    }
    __syncthreads();
    const uint32_t quota = max((uint32_t)kMinUnits, (total + gridDim.x - 1) / gridDim.x);
    // a sequence with nothing cached: zeros
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
        if (seq_len(p, b) != 0) continue;
        uint4* o = reinterpret_cast<uint4*>(p.out + (uint64_t)b * p.q_heads * D);
        for (uint32_t i = tid; i < p.q_heads * D / 8; i += kWarps * 32) o[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    Walk w0;
    w0.pos = blockIdx.x * quota;
    w0.end = min(total, w0.pos + quota);
    if (w0.pos >= total) return;
    {
        int lo = 0, hi = p.B;  // the last sequence that begins at or before pos (empty ones are skipped by enter)
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (prefix[mid] * items <= w0.pos) lo = mid;
            else hi = mid;
        }
        w0.enter(p, lo, pad);
        const uint32_t in = w0.pos - prefix[lo] * items;
        w0.item = (int)(in / w0.npad);
        w0.off = in % w0.npad;
    }
    __syncthreads();  // the prefix's room becomes the join's

    // ---- producer side: batches of this warp's steps, page numbers one batch ahead ----
    constexpr int SPB = 32 / C::NSUB;  // steps per batch: a lane looks up one 16-key sub-tile
    struct Batch {
        int kh, tok, t1, steps, page;  // first key, segment end, steps, this lane's page
    };
    Walk wp = w0;
    int pb = 0, pitem = 0, pt0 = 0, pt1 = 0;  // the producer's segment and what is left of it
    bool pmore = true;
    auto fetch = [&](Batch& x) {
        uint32_t st, sn;
        x.steps = 0;
        while (pmore) {
            const int first = pt0 + warp * C::TS;
            if (first < pt1) {
                x.kh = pitem / (int)A.tiles;
                x.tok = first;
                x.t1 = pt1;
                x.steps = min(SPB, (pt1 - first + kWarps * C::TS - 1) / (kWarps * C::TS));
                const int tk = first + (lane / C::NSUB) * (kWarps * C::TS) + (lane % C::NSUB) * 16;
                x.page = tk < pt1 ? __ldg(p.table + (uint64_t)pb * p.table_stride + (uint32_t)tk / p.kv.page_size) : 0;
                pt0 += SPB * kWarps * C::TS;
                return;
            }
            pmore = wp.next(p, items, pad, pb, pitem, pt0, pt1, st, sn);
        }
    };
    Batch cur, nxt;
    cur.steps = 0;
    fetch(nxt);
    int bstep = 0, pstage = 0;
    uint8_t* ring = base + warp * kStages * kStageBytes;
    auto produce = [&]() {
        if (bstep == cur.steps) {
            cur = nxt;
            bstep = 0;
            if (cur.steps == 0) return;
            fetch(nxt);
        }
        const int tok = cur.tok + bstep * (kWarps * C::TS);
        const int subs = min(C::NSUB, (cur.t1 - tok + 15) / 16);
        uint64_t* bar = &full[warp][pstage];
        const uint32_t dst = smem_u32(ring + pstage * kStageBytes);
        if (lane == 0) mbar_arrive_expect_tx(bar, subs * 16 * C::ROWB * 2);
#pragma unroll
        for (int s = 0; s < C::NSUB; ++s) {
            int page = __shfl_sync(0xffffffffu, cur.page, bstep * C::NSUB + s);
            if (lane == 0 && s < subs) {
                if ((uint32_t)page >= p.kv.pages) {  // not followed
                    atomicOr(p.err, kAttnErrIndex);
                    page = 0;
                }
                const int row = (int)((uint32_t)(tok + s * 16) % p.kv.page_size);
#pragma unroll
                for (int x = 0; x < C::NBX; ++x) {
                    const uint32_t d = dst + s * 16 * C::ROWB + x * C::BOX;
                    const int col = x * C::BOXB / (F8 ? 1 : 2);
                    tma4d(d, &A.kmap, col, row, cur.kh, page, bar);
                    tma4d(d + kStageBytes / 2, &A.vmap, col, row, cur.kh, page, bar);
                }
            }
        }
        ++bstep;
        pstage = pstage + 1 == kStages ? 0 : pstage + 1;
    };
    __syncwarp();
#pragma unroll
    for (int s = 0; s < kStages; ++s) produce();

    // ---- consumer side ----
    Walk wc = w0;
    int cstage = 0;
    uint32_t cphase = 0;
    int b, item, t0, t1;
    uint32_t start, units;
    while (wc.next(p, items, pad, b, item, t0, t1, start, units)) {
        const int kh = item / (int)A.tiles, head0 = (item % (int)A.tiles) * NT * 8;
        const int heads = min(NT * 8, (int)A.group - head0);  // of this pass
        const uint64_t hbase = (uint64_t)kh * A.group + head0;
        const float ks = p.kv.k_scale ? __ldg(p.kv.k_scale + kh) : 1.f;

        // q as the B operand.  E4M3 caches multiply in f16, which holds every E4M3 value; q (bf16)
        // goes there as q 2^-e, e the exponent of the head's largest element: exact but for elements
        // under 2^-15 of it, whose error is under 2^-25 of it.
        uint32_t qf[NT][KS][2];
        float ct[NT][2];  // scale log2(e) (times the key scale and 2^e) of heads 2 t4, 2 t4 + 1
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const bool used = n * 8 + g < heads;
            const uint16_t* qr = p.q + (uint64_t)b * p.q_stride + (hbase + n * 8 + (used ? g : 0)) * D;
            if (!F8) {
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        qf[n][k][j] =
                            used ? __ldg(reinterpret_cast<const uint32_t*>(qr + k * 16 + j * 8 + t4 * 2)) : 0u;
                ct[n][0] = ct[n][1] = p.scale * 1.4426950408889634f;
            } else {
                // the four bytes a lane gets of a key chunk are dims 4 t4 .. 4 t4 + 3: so here too
                uint2 rq[KS];
                uint32_t big = 0;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    rq[k] = used ? __ldg(reinterpret_cast<const uint2*>(qr + k * 16 + t4 * 4)) : make_uint2(0u, 0u);
                    big = max(max(big, rq[k].x & 0x7fffu), (rq[k].x >> 16) & 0x7fffu);
                    big = max(max(big, rq[k].y & 0x7fffu), (rq[k].y >> 16) & 0x7fffu);
                }
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                int e = (int)(big >> 7) - 127;
                if (e == 128 || big == 0) e = 0;
                if (e < -126) e = -126;
                const float down = e == 127 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)(127 - e) << 23);
                const float up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const float2 lo = make_float2(__uint_as_float(rq[k].x << 16), __uint_as_float(rq[k].x & 0xffff0000u));
                    const float2 hi = make_float2(__uint_as_float(rq[k].y << 16), __uint_as_float(rq[k].y & 0xffff0000u));
                    qf[n][k][0] = pack2<true>(lo.x * down, lo.y * down);
                    qf[n][k][1] = pack2<true>(hi.x * down, hi.y * down);
                }
                const float c = p.scale * up * ks * 1.4426950408889634f;
                ct[n][0] = __shfl_sync(0xffffffffu, c, t4 * 8);
                ct[n][1] = __shfl_sync(0xffffffffu, c, t4 * 8 + 4);
            }
        }

        float o[NT][KS][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][k][i] = 0.f;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }

        for (int tok = t0 + warp * C::TS; tok < t1; tok += kWarps * C::TS) {
            uint64_t* bar = &full[warp][cstage];
            if (!mbar_wait_bounded(bar, cphase, &abort_flag)) {
                // reported, and carried on with what is there: every warp keeps its place in the joins
                abort_flag = 1;
                if (lane == 0) atomicOr(p.err, kAttnErrWait);
                mbar_wait_slow(bar, cphase, &never);  // no copy stays in flight behind the kernel's end
            }
            const uint32_t kt = smem_u32(ring + cstage * kStageBytes), vt = kt + kStageBytes / 2;
            const int valid = t1 - tok;  // keys from here to the segment's end
            if (valid < C::TS && (valid & 15)) {
                // rows of the last sub-tile past the end may hold anything, NaN included: their weights are 0,
                // but 0 * NaN is not
                uint8_t* vs = ring + cstage * kStageBytes + kStageBytes / 2 + (valid >> 4) * 16 * C::ROWB;
                for (int i = lane; i < (16 - (valid & 15)) * C::NBX * (C::BOXB / 16); i += 32) {
                    const int r = (valid & 15) + i / (C::NBX * (C::BOXB / 16)), c = i % (C::NBX * (C::BOXB / 16));
                    *reinterpret_cast<uint4*>(vs + chunk_at<C::BOXB>(r, c)) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();  // before the ring's next copy into this stage
                __syncwarp();
            }
            // S^T = K q^T
            float s[C::NSUB][NT][4];
#pragma unroll
            for (int u = 0; u < C::NSUB; ++u) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[u][n][i] = 0.f;
                if (u * 16 < valid) {
                    const uint32_t kb = kt + u * 16 * C::ROWB;
                    float s2[NT][4];  // a second chain: consecutive products do not wait for one another
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s2[n][i] = 0.f;
#pragma unroll
                    for (int k = 0; k < KS; k += 2) {
                        uint32_t a0[4], a1[4];
                        if (!F8) {
                            ldsm4(a0, kb + chunk_at<C::BOXB>(lane & 15, 2 * k + (lane >> 4)));
                            ldsm4(a1, kb + chunk_at<C::BOXB>(lane & 15, 2 * k + 2 + (lane >> 4)));
                        } else {
                            uint32_t r[4];
                            ldsm4(r, kb + chunk_at<C::BOXB>(lane & 15, k + (lane >> 4)));
                            a0[0] = cvt_e4m3x2(r[0]), a0[1] = cvt_e4m3x2(r[1]);
                            a0[2] = cvt_e4m3x2(r[0] >> 16), a0[3] = cvt_e4m3x2(r[1] >> 16);
                            a1[0] = cvt_e4m3x2(r[2]), a1[1] = cvt_e4m3x2(r[3]);
                            a1[2] = cvt_e4m3x2(r[2] >> 16), a1[3] = cvt_e4m3x2(r[3] >> 16);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma<F8>(s[u][n], a0, qf[n][k][0], qf[n][k][1]);
                            mma<F8>(s2[n], a1, qf[n][k + 1][0], qf[n][k + 1][1]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[u][n][i] = (s[u][n][i] + s2[n][i]) * ct[n][i & 1];
                }
                if ((u + 1) * 16 > valid) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (u * 16 + g + (i >> 1) * 8 >= valid) s[u][n][i] = -INFINITY;
                }
            }
            // running maximum and sum; P^T as the B operand
            uint32_t pf[C::NSUB][NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float mx[2] = {m[n][0], m[n][1]};
#pragma unroll
                for (int u = 0; u < C::NSUB; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx[i & 1] = fmaxf(mx[i & 1], s[u][n][i]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1)
#pragma unroll
                    for (int i = 0; i < 2; ++i) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], d));
                if (__any_sync(0xffffffffu, mx[0] != m[n][0] || mx[1] != m[n][1])) {
                    // (a maximum of -inf: nothing but masked or -inf scores so far, o and l are 0)
                    const float a0 = m[n][0] == mx[0] ? 1.f : ex2(m[n][0] - mx[0]);
                    const float a1 = m[n][1] == mx[1] ? 1.f : ex2(m[n][1] - mx[1]);
                    l[n][0] *= a0;
                    l[n][1] *= a1;
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        o[n][k][0] *= a0, o[n][k][1] *= a1;
                        o[n][k][2] *= a0, o[n][k][3] *= a1;
                    }
                    m[n][0] = mx[0];
                    m[n][1] = mx[1];
                }
                const float z0 = mx[0] == -INFINITY ? 0.f : mx[0], z1 = mx[1] == -INFINITY ? 0.f : mx[1];
#pragma unroll
                for (int u = 0; u < C::NSUB; ++u) {
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[i] = ex2(s[u][n][i] - (i & 1 ? z1 : z0));
                    l[n][0] += e[0] + e[2];
                    l[n][1] += e[1] + e[3];
                    // weights to 16 bits (bf16 beside bf16 values, f16 beside E4M3 ones): the products with v
                    // and their sums stay in f32
                    pf[u][n][0] = movm(pack2<F8>(e[0], e[1]));
                    pf[u][n][1] = movm(pack2<F8>(e[2], e[3]));
                }
            }
            // O^T += V^T P^T
#pragma unroll
            for (int u = 0; u < C::NSUB; ++u) {
                if (u * 16 >= valid) break;
                const uint32_t vb = vt + u * 16 * C::ROWB;
                const int r = (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
#pragma unroll
                for (int k = 0; k < KS; k += 2) {
                    uint32_t a0[4], a1[4];
                    if (!F8) {
                        ldsm4t(a0, vb + chunk_at<C::BOXB>(r, 2 * k + c));
                        ldsm4t(a1, vb + chunk_at<C::BOXB>(r, 2 * k + 2 + c));
                    } else {
                        // a 16-bit element of the transposed load is dims 2g, 2g + 1 of one key: bytes are
                        // sorted to (dim 2g: two keys), (dim 2g + 1: two keys), rows g and g + 8 of the tile
                        uint32_t w[4];
                        ldsm4t(w, vb + chunk_at<C::BOXB>(r, k + c));
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = __byte_perm(w[i], 0, 0x3120);
                        a0[0] = cvt_e4m3x2(w[0]), a0[1] = cvt_e4m3x2(w[0] >> 16);
                        a0[2] = cvt_e4m3x2(w[2]), a0[3] = cvt_e4m3x2(w[2] >> 16);
                        a1[0] = cvt_e4m3x2(w[1]), a1[1] = cvt_e4m3x2(w[1] >> 16);
                        a1[2] = cvt_e4m3x2(w[3]), a1[3] = cvt_e4m3x2(w[3] >> 16);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma<F8>(o[n][k], a0, pf[u][n][0], pf[u][n][1]);
                        mma<F8>(o[n][k + 1], a1, pf[u][n][0], pf[u][n][1]);
                    }
                }
            }
            __syncwarp();
            if (++cstage == kStages) cstage = 0, cphase ^= 1;
            produce();
        }

        // ---- the segment's warps joined; out, or a partial result for the pair's last CTA ----
        const uint32_t c0 = start / quota, c1 = (start + units - 1) / quota;
        const bool whole = c0 == c1;
        float* slot = A.slots + ((uint64_t)blockIdx.x * 2 + (blockIdx.x == c0 ? 1 : 0)) * kSlotFloats;
        const float vscale = p.kv.v_scale ? __ldg(p.kv.v_scale + kh) : 1.f;
        constexpr int EPT = 8 * D / (kWarps * 32);  // output elements per thread: 4 or 2
        const int jh = tid * EPT / D, jd = tid * EPT % D;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n * 8 >= heads) break;
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], d);
                l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], d);
            }
            float* jw = join + warp * 8 * C::JROW;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = F8 ? k * 16 + 2 * g + (i >> 1) : k * 16 + g + (i >> 1) * 8;
                    jw[(2 * t4 + (i & 1)) * C::JROW + d] = o[n][k][i];
                }
            if (g == 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    stat[(warp * 8 + 2 * t4 + i) * 2] = m[n][i];
                    stat[(warp * 8 + 2 * t4 + i) * 2 + 1] = l[n][i];
                }
            }
            __syncthreads();
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, stat[(w * 8 + jh) * 2]);
            const float zz = mm == -INFINITY ? 0.f : mm;
            float acc[EPT], ll = 0.f;
#pragma unroll
            for (int i = 0; i < EPT; ++i) acc[i] = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = ex2(stat[(w * 8 + jh) * 2] - zz);
                ll = __fmaf_rn(f, stat[(w * 8 + jh) * 2 + 1], ll);
#pragma unroll
                for (int i = 0; i < EPT; ++i) acc[i] = __fmaf_rn(f, join[(w * 8 + jh) * C::JROW + jd + i], acc[i]);
            }
            if (whole) {
                if (n * 8 + jh < heads) {
                    const float r = ll > 0.f || ll != ll ? vscale / ll : 0.f;
                    uint32_t* dst = reinterpret_cast<uint32_t*>(
                        p.out + ((uint64_t)b * p.q_heads + hbase + n * 8 + jh) * D + jd);
#pragma unroll
                    for (int i = 0; i < EPT; i += 2) dst[i / 2] = pack2<false>(acc[i] * r, acc[i + 1] * r);
                }
            } else {
#pragma unroll
                for (int i = 0; i < EPT; ++i) slot[(n * 8 + jh) * D + jd + i] = acc[i];
                if (jd == 0) {
                    slot[kMaxTiles * 8 * 128 + (n * 8 + jh) * 2] = mm;
                    slot[kMaxTiles * 8 * 128 + (n * 8 + jh) * 2 + 1] = ll;
                }
            }
            __syncthreads();  // the join's room is free again
        }
        if (whole) continue;
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            const uint32_t before = atomicAdd(A.counters + c0, 1u);
            last_flag = before == c1 - c0;
            if (before == c1 - c0) A.counters[c0] = 0;  // as found, for the next call
        }
        __syncthreads();
        if (!last_flag) continue;
        __threadfence();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int h = n * 8 + jh;
            if (h >= heads) continue;
            const uint64_t step = 2 * kSlotFloats;
            const float* sl = A.slots + (uint64_t)c0 * step + kSlotFloats;  // the first CTA's second slot, then first slots
            float mm = -INFINITY, ll = 0.f, acc[EPT];
#pragma unroll
            for (int i = 0; i < EPT; ++i) acc[i] = 0.f;
            for (uint32_t c = c0; c <= c1; ++c) {
                const float* x = c == c0 ? sl : A.slots + (uint64_t)c * step;
                mm = fmaxf(mm, __ldcg(x + kMaxTiles * 8 * 128 + h * 2));
            }
            const float zz = mm == -INFINITY ? 0.f : mm;
#pragma unroll 4
            for (uint32_t c = c0; c <= c1; ++c) {
                const float* x = c == c0 ? sl : A.slots + (uint64_t)c * step;
                const float f = ex2(__ldcg(x + kMaxTiles * 8 * 128 + h * 2) - zz);
                ll = __fmaf_rn(f, __ldcg(x + kMaxTiles * 8 * 128 + h * 2 + 1), ll);
#pragma unroll
                for (int i = 0; i < EPT; i += 2) {
                    const float2 v = __ldcg(reinterpret_cast<const float2*>(x + h * D + jd + i));
                    acc[i] = __fmaf_rn(f, v.x, acc[i]);
                    acc[i + 1] = __fmaf_rn(f, v.y, acc[i + 1]);
                }
            }
            const float r = ll > 0.f || ll != ll ? vscale / ll : 0.f;
            uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + ((uint64_t)b * p.q_heads + hbase + h) * D + jd);
#pragma unroll
            for (int i = 0; i < EPT; i += 2) dst[i / 2] = pack2<false>(acc[i] * r, acc[i + 1] * r);
        }
    }
}

// The cache as a tensor map of 16-row boxes.
bool make_kv_map(CUtensorMap* map, const KvView& kv, const uint8_t* base, uint64_t page_stride) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return false;
    const uint64_t elt = kv.e4m3 ? 1 : 2, rowb = kv.head_dim * elt, boxb = rowb < 128 ? rowb : 128;
    const cuuint64_t dims[4] = {kv.head_dim, kv.page_size, kv.kv_heads, kv.pages};
    const cuuint64_t strides[3] = {rowb, rowb * kv.page_size, page_stride * elt};
    const cuuint32_t box[4] = {(cuuint32_t)(boxb / elt), 16, 1, 1};
    const cuuint32_t one[4] = {1, 1, 1, 1};
    return fn(map, kv.e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
              const_cast<uint8_t*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              boxb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t counter_bytes(int num_sms) { return ((size_t)num_sms * 4 + 255) / 256 * 256; }

template <int D, bool F8, int NT>
int launch(const DecodeArgs& a, int grid, cudaStream_t st) {
    using C = Cfg<D, F8, NT>;
    const size_t room = C::JOIN + kWarps * 8 * 2 * 4, prefix = (size_t)a.p.B * 4;
    const size_t most = 1024 + C::RING + (room > 4 * 4096 ? room : 4 * 4096);
    const size_t smem = 1024 + C::RING + (room > prefix ? room : prefix);
    static bool set = false;  // the library's lock is held
    if (!set) {
        if (cudaFuncSetAttribute(attn_decode_kernel<D, F8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)most) != cudaSuccess)
            return CZ_ELAUNCH;
        set = true;
    }
    attn_decode_kernel<D, F8, NT><<<grid, kWarps * 32, smem, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? CZ_OK : CZ_ELAUNCH;
}

}  // namespace

size_t attn_decode_workspace_bytes(int num_sms) {
    return counter_bytes(num_sms) + (size_t)num_sms * 2 * kSlotFloats * sizeof(float);
}

int attn_decode_launch(const AttnDecodeParams& p, int num_sms, cudaStream_t st) {
    DecodeArgs a{};
    a.p = p;
    a.group = p.q_heads / p.kv.kv_heads;
    const bool two = a.group > 8;
    a.tiles = two ? (a.group + 15) / 16 : 1;
    // the split's line and its parts' ends are counted in 32 bits
    const uint64_t units = ((uint64_t)p.table_width * p.kv.page_size + kUnit - 1) / kUnit + kMinUnits;
    if ((uint64_t)p.B * p.kv.kv_heads * a.tiles * units >= 0x7fffffffu) return CZ_ESHAPE;
    if (!make_kv_map(&a.kmap, p.kv, p.kv.k, p.kv.k_page) || !make_kv_map(&a.vmap, p.kv, p.kv.v, p.kv.v_page))
        return CZ_ESHAPE;
    a.counters = reinterpret_cast<uint32_t*>(p.workspace);
    a.slots = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.workspace) + counter_bytes(num_sms));
    const bool d128 = p.kv.head_dim == 128;
    if (p.kv.e4m3) {
        if (two) return d128 ? launch<128, true, 2>(a, num_sms, st) : launch<64, true, 2>(a, num_sms, st);
        return d128 ? launch<128, true, 1>(a, num_sms, st) : launch<64, true, 1>(a, num_sms, st);
    }
    if (two) return d128 ? launch<128, false, 2>(a, num_sms, st) : launch<64, false, 2>(a, num_sms, st);
    return d128 ? launch<128, false, 1>(a, num_sms, st) : launch<64, false, 1>(a, num_sms, st);
}

}  // namespace cz
