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
// Work split.  The caches of all (sequence, key/value head) pairs ("items") form one long
// line of steps (8 KB of keys and values each), cut into equal parts, one per warp, whatever the
// lengths are (read on the device, so a captured graph follows them).  A warp runs through its
// part alone: its own ring of TMA stages, its own running softmax, an item that lies whole in it
// written out at once, so short caches cost no barrier.  An item cut between warps leaves
// partial (o, m, l) in shared memory, joined at the block's end; one cut between blocks leaves
// a partial in the workspace, and the last block of the item to arrive joins them.  Both joins
// go in order along the line, so results do not depend on timing.  With few or short items the
// parts are laid so that none is cut between blocks, or as few as the idle blocks are worth.
//
// Measured: 96 sequences of up to 8,192 tokens, 32 heads on 4 of 128, 1.51 GB: 231-237 us, 6.39-6.55
// TB/s (a copy's rate is 6.46); one of 32,781 tokens 22.1-22.6 us (10.4 at that rate: some 5 us pass before the
// first keys arrive, some 5 in the joins); 97 tokens 5.7 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cz_common.cuh"
#include "cz_internal.h"

namespace cz {
namespace {

constexpr int kWarps = 8;
// 128 KB in flight per SM reach the card's rate; a third stage only lengthens the queue that the
// last blocks wait in (128 x 4,000 tokens: 171 us with 3, 163 us with 2).
constexpr int kStages = 2;
constexpr int kStageBytes = 8192;  // keys, then values, of one step
// With little work, an item of up to this many steps per warp stays in one block: up to there the join over
// the workspace costs more than the shorter loop gains (256 keys in bf16: 7.6 us in one block, 8.5 us in
// two; 512 keys: 9.6 us in one, 8.8 us in four).
constexpr int kShort = 2;
// What starting and ending an item costs a warp, in steps (48 ragged sequences on E4M3: 34.1, 32.5, 31.8 and
// 32.1 us with 1 to 4).
constexpr uint32_t kItemSteps = 3;
// What joins across blocks cost, in steps of a warp's loop (28 sequences of 61 tokens on 8 heads: 10.4 us cut
// anywhere, 7.0 us with four warps an item; 101 of 32 tokens: 10.9 and 7.7 us).
constexpr uint32_t kJoinSteps = 4;
constexpr int kMaxTiles = 2;       // 8-head column tiles per pass
constexpr int kBatch = 40;         // partials of other blocks joined at a time
constexpr int kSlotFloats = kMaxTiles * 8 * 128 + kMaxTiles * 8 * 2;  // o, then (m, l) per head

struct DecodeArgs {
    CUtensorMap kmap, vmap;  // page, head, column block, row, columns of the block (128 bytes at most)
    AttnDecodeParams p;
    uint32_t group, tiles;   // query heads per kv head; passes of NT * 8 of them
    float* slots;            // workspace: [grid][2][kSlotFloats]
    uint32_t* counters;      // workspace: [grid] arrivals at the item that begins in this block and goes on
    int box;                 // rows per TMA box: a step's, or 16 where pages are smaller or cut it
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void tma5d(uint32_t dst, const CUtensorMap* m, int row, int head, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(0), "r"(row), "r"(0), "r"(head), "r"(page), "r"(smem_u32(bar))
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
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t atom_add_acq_rel(uint32_t* p, uint32_t v) {
    uint32_t r;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(r) : "l"(p), "r"(v) : "memory");
    return r;
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
    const int n = ld_now(p.lens + b);
    const int most = (int)(p.table_width * p.kv.page_size);
    return n < 0 ? 0 : n > most ? most : n;
}

// The line: sequence by sequence, `items` stretches (kv heads x passes) of length() steps.
struct Line {
    int items;
    uint32_t quota;  // steps per warp
    uint32_t unit;   // items take whole units (0: their steps and kItemSteps)

    __device__ __forceinline__ uint32_t length(uint32_t n) const {
        return n == 0 ? 0 : unit ? (n + unit - 1) / unit * unit : n + kItemSteps;
    }
};

// Walks a warp's part [pos, end) of the line.
template <int TS>
struct Walk {
    uint32_t pos, end, off;  // place on the line; steps of the current item before it
    int b, item, len;
    uint32_t n, room;        // steps of an item of b; what they take on the line

    __device__ __forceinline__ void enter(const AttnDecodeParams& p, const Line& line, int bb) {
#pragma unroll 1
        for (b = bb; b < p.B; ++b) {
            len = seq_len(p, b);
            if (len > 0) break;
        }
        n = b < p.B ? (uint32_t)(len + TS - 1) / TS : 0;
        room = line.length(n);
    }
    // The next segment: keys [t0, t1) of (b, item), whose stretch begins at `start` on the line.
    // False at the part's end.
    __device__ __forceinline__ bool next(const AttnDecodeParams& p, const Line& line, int& sb, int& sitem, int& t0,
                                         int& t1, int& slen, uint32_t& start) {
#pragma unroll 1
        while (pos < end && b < p.B) {
            const uint32_t u0 = off, take = min(room - off, end - pos), u1 = min(u0 + take, n);
            sb = b;
            sitem = item;
            slen = len;
            t0 = (int)(u0 * TS);
            t1 = min(len, (int)(u1 * TS));
            start = pos - u0;
            pos += take;
            off += take;
            if (off == room) {
                off = 0;
                if (++item == line.items) {
                    item = 0;
                    enter(p, line, b + 1);
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
    static constexpr int JROW = D + 4;
    static constexpr int RING = kWarps * kStages * kStageBytes;
    // Weights go to f16 beside E4M3 values: 2^kShift above their maximum of 1, so that they stay normal down to
    // 2^-28 of it and vanish under 2^-38 only (unshifted, a hundred thousand keys of weight 2^-25 each would be
    // lost or doubled); bf16 has the range.  Partials are kept relative to 2^(m - kShift).
    static constexpr float kShift = F8 ? 14.f : 0.f;
    // a warp's partial of the item it starts in; that of the item it ends in goes into its ring
    static constexpr int PART = NT * 8 * JROW * 4;
    static_assert(PART <= kStages * kStageBytes, "a partial fits the ring");
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
    uint32_t* prefix = reinterpret_cast<uint32_t*>(base + C::RING);  // prologue: places before each sequence (one item's)
    __shared__ uint64_t full[kWarps][kStages];
    __shared__ uint32_t scan[kWarps][7];
    // partials of the items a warp starts in (0) and ends in (1): item (-1: none), whether its first and its last
    // keys are in it, place on the line and steps of the whole item
    struct Rec {
        int item, b, begins, ends;
        uint32_t start, steps;
    };
    __shared__ Rec recs[kWarps][2];
    __shared__ float2 stat[kWarps][2][NT * 8];  // (m, l)
    __shared__ int abort_flag, never;
    __shared__ uint32_t last_flag[2];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t4 = lane & 3;

    if (tid == 0) abort_flag = never = 0;
    if (lane < 2) recs[warp][lane].item = -1;
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], 1);
        fence_mbarrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tensormap(&A.kmap);
        prefetch_tensormap(&A.vmap);
    }

    __syncthreads();  // the flags are cleared before any warp's wait reads them
    pdl_wait();

    // ---- the line and this warp's part of it ----
    // of the sequences: steps and item costs; blocks with 1, 2 and 4 steps a warp; how many have keys; the longest
    Line line;
    line.items = (int)(p.kv.kv_heads * A.tiles);
    const uint32_t grid = gridDim.x, items = (uint32_t)line.items;
    uint32_t sum[6] = {0, 0, 0, 0, 0, 0};
    auto count = [&](int b) {
        const int l = seq_len(p, b);
        if (blockIdx.x == 0 && (warp == 0 || p.B > 32) && ld_now(p.lens + b) != l) atomicOr(p.err, kAttnErrIndex);
        const uint32_t n = (uint32_t)(l + C::TS - 1) / C::TS;
        sum[0] += n ? n + kItemSteps : 0;
        sum[1] += (n + kWarps - 1) / kWarps;
        sum[2] += (n + 2 * kWarps - 1) / (2 * kWarps);
        sum[3] += (n + 4 * kWarps - 1) / (4 * kWarps);
        sum[4] += n ? 1 : 0;
        sum[5] = max(sum[5], n);
        return n;
    };
    auto decide = [&]() {
        const uint32_t warps = grid * kWarps, longest = sum[5];
        line.quota = (sum[0] * items + warps - 1) / warps;
        line.unit = 0;
        if (sum[3] * items <= grid) {
            // little work, every item gets blocks of its own: the shortest loops that the blocks allow, but short items
            // in one block
            line.quota = longest <= kShort * kWarps ? max(1u, (longest + kWarps - 1) / kWarps)
                         : sum[1] * items <= grid   ? 1
                         : sum[2] * items <= grid   ? 2
                                                    : 4;
            line.unit = kWarps * line.quota;
        } else {
            // more items than blocks: several to a block, each on as many warps as that allows, unless the loops get
            // longer by more than the joins across blocks cost
            const uint32_t all = sum[4] * items;
            const uint32_t w = all * 4 <= warps ? 4 : all * 2 <= warps ? 2 : 1;
            const uint32_t q = (longest + w - 1) / w;
            if (all * w <= warps && q <= line.quota + kJoinSteps) {
                line.quota = q;
                line.unit = w * q;
            }
        }
    };
    auto reduce = [&]() {
#pragma unroll
        for (int i = 0; i < 5; ++i) sum[i] = __reduce_add_sync(0xffffffffu, sum[i]);
        sum[5] = __reduce_max_sync(0xffffffffu, sum[5]);
    };
    auto scan32 = [&](uint32_t v) {  // inclusive sums over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        return v;
    };
    uint32_t total, begin;  // begin: where the line's sequence `lo` starts
    uint32_t bquota;        // a block's part
    int lo = 0;             // the last sequence that begins at or before this warp's part (empty ones are skipped later)
    if (p.B <= 32) {        // every warp for itself
        const uint32_t n = lane < p.B ? count(lane) : 0;
        reduce();
        decide();
        bquota = line.quota * kWarps;
        const uint32_t mine = line.length(n), inc = scan32(mine);
        total = __shfl_sync(0xffffffffu, inc, 31) * items;
        const uint32_t pos = min(total, blockIdx.x * bquota + warp * line.quota);
        const unsigned at = __ballot_sync(0xffffffffu, lane < p.B && (inc - mine) * items <= pos);
        lo = 31 - __clz(at);
        begin = __shfl_sync(0xffffffffu, inc - mine, lo) * items;
    } else {
        const int per = (p.B + kWarps * 32 - 1) / (kWarps * 32);
#pragma unroll 1
        for (int i = 0; i < per; ++i)
            if (tid * per + i < p.B) count(tid * per + i);
        reduce();
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < 6; ++i) scan[warp][i] = sum[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 6; ++i) sum[i] = lane < kWarps ? scan[lane][i] : 0;
        reduce();
        decide();
        bquota = line.quota * kWarps;
        uint32_t mine = 0;
#pragma unroll 1
        for (int i = 0; i < per; ++i) {
            const int b = tid * per + i;
            if (b < p.B) mine += line.length((uint32_t)(seq_len(p, b) + C::TS - 1) / C::TS);
        }
        const uint32_t inc = scan32(mine);
        if (lane == 31) scan[warp][6] = inc;
        __syncthreads();
        uint32_t place = inc - mine;
        total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t v = scan[w][6];
            if (w < warp) place += v;
            total += v;
        }
        total *= items;
#pragma unroll 1
        for (int i = 0; i < per; ++i) {
            const int b = tid * per + i;
            if (b >= p.B) break;
            prefix[b] = place;
            place += line.length((uint32_t)(seq_len(p, b) + C::TS - 1) / C::TS);
        }
        __syncthreads();
        const uint32_t pos = min(total, blockIdx.x * bquota + warp * line.quota);
        int hi = p.B;
#pragma unroll 1
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (prefix[mid] * items <= pos) lo = mid;
            else hi = mid;
        }
        begin = prefix[lo] * items;
        __syncthreads();  // the prefix's room becomes the partials'
    }
    // a sequence with nothing cached: zeros
#pragma unroll 1
    for (int b = blockIdx.x; b < p.B; b += grid) {
        if (seq_len(p, b) != 0) continue;
        uint4* o = reinterpret_cast<uint4*>(p.out + (uint64_t)b * p.q_heads * D);
#pragma unroll 1
        for (uint32_t i = tid; i < p.q_heads * D / 8; i += kWarps * 32) o[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    if (blockIdx.x * bquota >= total) return;
    Walk<C::TS> wc;
    wc.pos = min(total, blockIdx.x * bquota + warp * line.quota);
    wc.end = min(total, wc.pos + line.quota);
    wc.b = p.B;
    wc.off = 0;
    wc.item = 0;
    if (wc.pos < total) {
        wc.enter(p, line, lo);
        const uint32_t in = wc.pos - begin;
        wc.item = (int)(in / wc.room);
        wc.off = in % wc.room;
    }

    // ---- producer side: batches of this warp's steps, page numbers one batch ahead ----
    constexpr int SPB = 32 / C::NSUB;  // steps per batch: a lane looks up one 16-key sub-tile
    struct Batch {
        int kh, tok, t1, steps, page, row;  // first key, segment end, steps, this lane's page and row in it
    };
    Walk<C::TS> wp = wc;
    int pb = 0, pitem = 0, pt0 = 0, pt1 = 0;  // the producer's segment: what is left of it
    bool pmore = true;
    Batch cur, nxt;
    cur.steps = nxt.steps = 0;
    int bstep = 0, pstage = 0;
    uint8_t* ring = base + warp * kStages * kStageBytes;
    // One step's copies.  (Called from one place, like both Walk::next: the code of an item's whole round
    // has to stay in the instruction caches.)
    auto produce = [&]() {
#pragma unroll 1
        while (bstep == cur.steps && (pmore || nxt.steps)) {
            cur = nxt;
            bstep = 0;
            nxt.steps = 0;
            if (pt0 >= pt1) {
                int len;
                uint32_t st;
                pmore = wp.next(p, line, pb, pitem, pt0, pt1, len, st);
            }
            if (pmore) {
                nxt.kh = pitem / (int)A.tiles;
                nxt.tok = pt0;
                nxt.t1 = pt1;
                nxt.steps = min(SPB, (pt1 - pt0 + C::TS - 1) / C::TS);
                const uint32_t tk = pt0 + lane * 16;
                const uint32_t idx = tk / p.kv.page_size;
                nxt.row = (int)(tk - idx * p.kv.page_size);
                nxt.page = (int)tk < pt1 ? ld_now(p.table + (uint64_t)pb * p.table_stride + idx) : 0;
                pt0 += SPB * C::TS;
            }
        }
        if (bstep == cur.steps) return;
        const int tok = cur.tok + bstep * C::TS;
        const int subs = min(C::NSUB, (cur.t1 - tok + 15) / 16);
        uint64_t* bar = &full[warp][pstage];
        const uint32_t dst = smem_u32(ring + pstage * kStageBytes);
        const int skip = A.box / 16;  // sub-tiles per box
        if (lane == 0) mbar_arrive_expect_tx(bar, (subs + skip - 1) / skip * skip * 16 * C::ROWB * 2);
#pragma unroll 1
        for (int s = 0; s < subs; s += skip) {
            int page = __shfl_sync(0xffffffffu, cur.page, bstep * C::NSUB + s);
            const int row = __shfl_sync(0xffffffffu, cur.row, bstep * C::NSUB + s);
            if (lane == 0) {
                if ((uint32_t)page >= p.kv.pages) {  // not followed
                    atomicOr(p.err, kAttnErrIndex);
                    page = 0;
                }
                tma5d(dst + s * 16 * C::ROWB, &A.kmap, row, cur.kh, page, bar);
                tma5d(dst + s * 16 * C::ROWB + kStageBytes / 2, &A.vmap, row, cur.kh, page, bar);
            }
        }
        ++bstep;
        pstage = pstage + 1 == kStages ? 0 : pstage + 1;
    };
    int credit = kStages;  // stages free to fill
    __syncwarp();

    // ---- consumer side ----
    int cstage = 0;
    uint32_t cphase = 0;
    int b, item, t0, t1, len;
    uint32_t start;
#pragma unroll 1
    while (wc.next(p, line, b, item, t0, t1, len, start)) {
        const int kh = item / (int)A.tiles, head0 = (item % (int)A.tiles) * NT * 8;
        const int heads = min(NT * 8, (int)A.group - head0);  // of this pass
        const uint64_t hbase = (uint64_t)kh * A.group + head0;
        const float ks = p.kv.k_scale ? ld_now(p.kv.k_scale + kh) : 1.f;

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
                            used ? ld_now(reinterpret_cast<const uint32_t*>(qr + k * 16 + j * 8 + t4 * 2)) : 0u;
                ct[n][0] = ct[n][1] = p.scale * 1.4426950408889634f;
            } else {
                // the four bytes a lane gets of a key chunk are dims 4 t4 .. 4 t4 + 3: so here too
                uint2 rq[KS];
                uint32_t big = 0;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    rq[k] = used ? ld_now(reinterpret_cast<const uint2*>(qr + k * 16 + t4 * 4)) : make_uint2(0u, 0u);
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

#pragma unroll 1
        for (int tok = t0;; tok += C::TS) {
#pragma unroll 1
            for (; credit > 0; --credit) produce();
            if (tok >= t1) break;
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
#pragma unroll 1
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
                const float z0 = mx[0] == -INFINITY ? 0.f : mx[0] - C::kShift, z1 = mx[1] == -INFINITY ? 0.f : mx[1] - C::kShift;
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
            ++credit;
        }

        // ---- the segment's end ----
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], d);
                l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], d);
            }
        if (t0 == 0 && t1 == len) {  // the whole item: out
            const float vscale = p.kv.v_scale ? ld_now(p.kv.v_scale + kh) : 1.f;
            uint16_t* out = p.out + ((uint64_t)b * p.q_heads + hbase) * D;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float r0 = l[n][0] > 0.f || l[n][0] != l[n][0] ? vscale / l[n][0] : 0.f;
                const float r1 = l[n][1] > 0.f || l[n][1] != l[n][1] ? vscale / l[n][1] : 0.f;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const float* c = o[n][k];
                    if (F8) {  // dims 16 k + 2 g, + 1 of heads 2 t4 and 2 t4 + 1
                        const int h = n * 8 + 2 * t4;
                        uint16_t* d = out + (uint64_t)h * D + k * 16 + 2 * g;
                        if (h < heads) *reinterpret_cast<uint32_t*>(d) = pack2<false>(c[0] * r0, c[2] * r0);
                        if (h + 1 < heads) *reinterpret_cast<uint32_t*>(d + D) = pack2<false>(c[1] * r1, c[3] * r1);
                    } else {  // two heads of a dim -> two dims of a head
                        const uint32_t lo = movm(pack2<false>(c[0] * r0, c[1] * r1));
                        const uint32_t hi = movm(pack2<false>(c[2] * r0, c[3] * r1));
                        uint16_t* d = out + (uint64_t)(n * 8 + g) * D + k * 16 + 2 * t4;
                        if (n * 8 + g < heads) {
                            *reinterpret_cast<uint32_t*>(d) = lo;
                            *reinterpret_cast<uint32_t*>(d + 8) = hi;
                        }
                    }
                }
            }
        } else {
            const int which = t0 == 0;  // an item begun here is the part's last: the ring is free for it
            float* jw = reinterpret_cast<float*>(which ? ring : base + C::RING + warp * C::PART);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int d = F8 ? k * 16 + 2 * g + (i >> 1) : k * 16 + g + (i >> 1) * 8;
                        jw[(n * 8 + 2 * t4 + (i & 1)) * C::JROW + d] = o[n][k][i];
                    }
                if (g == 0) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        stat[warp][which][n * 8 + 2 * t4 + i] = make_float2(m[n][i] - C::kShift, l[n][i]);
                }
            }
            if (lane == 0)
                recs[warp][which] = Rec{item, b, t0 == 0, t1 == len, start, (uint32_t)(len + C::TS - 1) / C::TS};
        }
    }

    // ---- items cut between this block's warps, or between blocks ----
    __syncthreads();
    constexpr int EPT = 4;  // a warp a head, 4 dims a lane (half of the lanes for 64)
    const int jh = warp, jd = lane * EPT;
    const bool on = jd < D;
    auto finish = [&](const Rec& r, int n, float* acc, float ll) {
        const int kh = r.item / (int)A.tiles, h = (r.item % (int)A.tiles) * NT * 8 + n * 8 + jh;
        if (h >= (int)A.group || !on) return;
        const float vscale = p.kv.v_scale ? ld_now(p.kv.v_scale + kh) : 1.f;
        const float f = ll > 0.f || ll != ll ? vscale / ll : 0.f;
        uint32_t* dst = reinterpret_cast<uint32_t*>(
            p.out + ((uint64_t)r.b * p.q_heads + (uint64_t)kh * A.group + h) * D + jd);
#pragma unroll
        for (int i = 0; i < EPT; i += 2) dst[i / 2] = pack2<false>(acc[i] * f, acc[i + 1] * f);
    };
    // lane x looks after record x (warp x / 2, kind x % 2): an item's records follow one another, the
    // first of them one that begins it, unless it came from the block before
    const Rec& mine = recs[(lane >> 1) & 7][lane & 1];
    const bool has = lane < 2 * kWarps && mine.item >= 0;
    const uint32_t have = __ballot_sync(0xffffffffu, has), begs = __ballot_sync(0xffffffffu, has && mine.begins);
    const uint32_t fins = __ballot_sync(0xffffffffu, has && mine.ends);
    int open_left = -1, open_right = -1;  // first records of the items that go on in other blocks: before, or only after
#pragma unroll 1
    for (uint32_t left = have; left;) {
        const int x = __ffs(left) - 1;
        const uint32_t later = begs & left & ~(1u << x);
        const uint32_t group = left & (later ? (later & (0u - later)) - 1 : 0xffffffffu);
        left &= ~group;
        const bool begins = begs >> x & 1, done = begins && (fins & group);
        if (!done) (begins ? open_right : open_left) = x;
        float* slot = A.slots + ((uint64_t)blockIdx.x * 2 + begins) * kSlotFloats;
#pragma unroll 1
        for (int n = 0; n < NT; ++n) {
            const bool in = lane < 2 * kWarps && (group >> lane & 1);
            const float2 ml = in ? stat[(lane >> 1) & 7][lane & 1][n * 8 + jh] : make_float2(-INFINITY, 0.f);
            const float mm = warp_max(ml.x), zz = mm == -INFINITY ? 0.f : mm;
            const float f = ex2(ml.x - zz), ll = warp_sum(f * ml.y);
            float acc[EPT];
#pragma unroll
            for (int i = 0; i < EPT; ++i) acc[i] = 0.f;
#pragma unroll
            for (int z = 0; z < 2 * kWarps; ++z) {
                const float fz = __shfl_sync(0xffffffffu, f, z);
                if ((group >> z & 1) && on) {
                    const float* v = reinterpret_cast<const float*>(z & 1 ? base + (z >> 1) * kStages * kStageBytes
                                                                          : base + C::RING + (z >> 1) * C::PART) +
                                     (n * 8 + jh) * C::JROW + jd;
#pragma unroll
                    for (int i = 0; i < EPT; ++i) acc[i] = __fmaf_rn(fz, v[i], acc[i]);
                }
            }
            if (done) {
                finish(recs[x >> 1][x & 1], n, acc, ll);
            } else {
#pragma unroll
                for (int i = 0; i < EPT; ++i)
                    if (on) slot[(n * 8 + jh) * D + jd + i] = acc[i];
                if (jd == 0) *(reinterpret_cast<float2*>(slot + kMaxTiles * 8 * 128) + n * 8 + jh) = make_float2(mm, ll);
            }
        }
    }
    if (open_left < 0 && open_right < 0) return;
    __syncthreads();  // the partials are written; then one release / acquire each
    if (tid < 64 && lane == 0) {
        const int x = tid ? open_right : open_left;
        uint32_t last = 0;
        if (x >= 0) {
            const Rec& r = recs[x >> 1][x & 1];
            const uint32_t c0 = r.start / bquota, c1 = (r.start + r.steps - 1) / bquota;
            last = atom_add_acq_rel(A.counters + c0, 1u) == c1 - c0;
            if (last) A.counters[c0] = 0;  // as found, for the next call
        }
        last_flag[tid >> 5] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
        if (!last_flag[side]) continue;
        const int x = side ? open_right : open_left;
        const Rec& r = recs[x >> 1][x & 1];
        const uint32_t c0 = r.start / bquota, c1 = (r.start + r.steps - 1) / bquota;
        // The item's partials in order.  Up to kBatch of them are fetched at once, each thread's own pieces into
        // shared memory that is free by now (fetched one by one they would cost a trip to L2 each; held in
        // registers, unrolled code that runs once and cold).
        static_assert(kBatch * 8 * D * 4 <= C::RING + kWarps * C::PART, "a batch fits");
        const int parts = (int)(c1 - c0) + 1;
        float* own = reinterpret_cast<float*>(base) + jh * D + jd;
#pragma unroll 1
        for (int n = 0; n < NT; ++n) {
            const int h = n * 8 + jh;
            float acc[EPT], mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int i = 0; i < EPT; ++i) acc[i] = 0.f;
            auto part = [&](int q) { return A.slots + ((uint64_t)(c0 + q) * 2 + (q == 0 ? 1 : 0)) * kSlotFloats; };
            auto stats = [&](int q) {
                return q < parts ? __ldcg(reinterpret_cast<const float2*>(part(q) + kMaxTiles * 8 * 128) + h)
                                 : make_float2(-INFINITY, 0.f);
            };
#pragma unroll 1
            for (int c = 0; c < parts; c += kBatch) {
                const int cnt = min(kBatch, parts - c);
#pragma unroll 1
                for (int j = 0; on && j < cnt; ++j) cp_async16(own + j * 8 * D, part(c + j) + h * D + jd);
                asm volatile("cp.async.commit_group;" ::: "memory");
                // (m, l) of parts c + lane and c + 32 + lane
                const float2 s0 = stats(c + lane), s1 = lane < kBatch - 32 ? stats(c + 32 + lane) : make_float2(-INFINITY, 0.f);
                const float top = fmaxf(mm, warp_max(fmaxf(s0.x, s1.x))), zz = top == -INFINITY ? 0.f : top;
                const float a = ex2(mm - zz), f0 = ex2(s0.x - zz), f1 = ex2(s1.x - zz);
                mm = top;
                ll = __fmaf_rn(ll, a, warp_sum(__fmaf_rn(f0, s0.y, f1 * s1.y)));
#pragma unroll
                for (int i = 0; i < EPT; ++i) acc[i] *= a;
                asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll 4
                for (int j = 0; j < cnt; ++j) {
                    const float f = __shfl_sync(0xffffffffu, j < 32 ? f0 : f1, j & 31);
                    const float* v = own + j * 8 * D;
#pragma unroll
                    for (int i = 0; i < EPT; ++i)
                        if (on) acc[i] = __fmaf_rn(f, v[i], acc[i]);
                }
            }
            finish(r, n, acc, ll);
        }
    }
}

// The cache as a tensor map: [page][head][128-byte column block][row][columns], boxes of `rows` rows
// of all column blocks, each block's rows together in shared memory.
bool make_kv_map(CUtensorMap* map, const KvView& kv, const uint8_t* base, uint64_t page_stride, uint32_t rows) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return false;
    const uint64_t elt = kv.e4m3 ? 1 : 2, rowb = kv.head_dim * elt, boxb = rowb < 128 ? rowb : 128;
    const cuuint64_t dims[5] = {boxb / elt, kv.page_size, rowb / boxb, kv.kv_heads, kv.pages};
    const cuuint64_t strides[4] = {rowb, boxb, rowb * kv.page_size, page_stride * elt};
    const cuuint32_t box[5] = {(cuuint32_t)(boxb / elt), rows, (cuuint32_t)(rowb / boxb), 1, 1};
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    return fn(map, kv.e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
              const_cast<uint8_t*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              boxb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t counter_bytes(int num_sms) { return ((size_t)num_sms * 4 + 255) / 256 * 256; }

template <int D, bool F8, int NT>
int launch(DecodeArgs& a, int grid, cudaStream_t st) {
    using C = Cfg<D, F8, NT>;
    a.box = a.p.kv.page_size % C::TS == 0 ? C::TS : 16;
    if (!make_kv_map(&a.kmap, a.p.kv, a.p.kv.k, a.p.kv.k_page, a.box) ||
        !make_kv_map(&a.vmap, a.p.kv, a.p.kv.v, a.p.kv.v_page, a.box))
        return CZ_ESHAPE;
    // behind the rings, one after the other: the prefix [B], the partials
    const size_t parts = kWarps * C::PART, prefix = (size_t)a.p.B * 4;
    const size_t smem = 1024 + C::RING + (parts > prefix ? parts : prefix);
    constexpr size_t most = 227 * 1024 - 4096;  // beside the static variables
    if (smem > most) return CZ_ESHAPE;
    static uint32_t set = 0;  // the library's lock is held
    if (set != init_serial) {
        if (cudaFuncSetAttribute(attn_decode_kernel<D, F8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)most) != cudaSuccess)
            return CZ_ELAUNCH;
        set = init_serial;
    }
    return launch_early(attn_decode_kernel<D, F8, NT>, grid, kWarps * 32, smem, st, a) ? CZ_OK : CZ_ELAUNCH;
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
    // the line and its parts' ends are counted in 32 bits; a step is 16 keys or more
    const uint64_t steps = (uint64_t)p.table_width * p.kv.page_size / 16 + kItemSteps + kWarps * 4;
    if ((uint64_t)p.B * p.kv.kv_heads * a.tiles * steps >= 0x7fff0000u) return CZ_ESHAPE;
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
