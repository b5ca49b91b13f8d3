// Causal attention over packed prompts: query i of sequence b (nq queries, nk keys,
// aligned at their ends) sees the keys j <= i + nk - nq;
//   out = sum_j p_j v_j,  p = softmax_j(scale q . k_j),  zeros when it sees none,
// over tiles of 128 keys with a running maximum m and sum l (f32):
//   S = Q K^T,  P = 2^(c S - c m),  l += rowsum P,  O += P V,  c = scale log2(e).
//
// Bound by the tensor pipe (4 D flops per visible pair) with the exponentials (one per
// pair and head, 16 a clock and SM) close behind.  Both products run on tcgen05 with
// their accumulators in TMEM: S and O of two 128-row query tiles fill its 512 columns, so
// that one tile's softmax runs under the other's products; P replaces S in place as
// bf16 and is the second product's A operand straight from TMEM.
//
// A query tile packs the G query heads of a key/value head: row = token * G + head, 128 / G
// tokens.  Keys and values are read once for all of them, a short prompt still fills
// the tile (16 tokens of 8 heads), and the diagonal wastes at most 16 of 128 keys there.
//
// One block per SM runs through pairs of query tiles (single ones where that takes the busiest block less: 927 tokens
// of 8 heads on one, 21.7 -> 16.2 us), the longest first and in turn from either end, so that the blocks
// end together; the next pair's queries, keys and first products go out
// while the last one's results are written.  Warps: 0-3 and 4-7 softmax of query tile 0 and 1 (a
// thread a row), 8 TMA loads, 9 MMA issue, 10 picks the pairs, 11 clears what lies behind the last
// values.
//
// Measured: one prompt of 8,192 tokens, 32 heads on 4 of 128: 430 us, 1,280 TFLOP/s (0.78 of the
// measured bf16 rate; 490 us back to back, under the power cap).  What is left is the way from a
// tile's scores to its weights, some 1,600 cycles of load, maximum and exponentials on which the
// next product waits, against 1,084 of the other tile's products; half of the exponentials taken out
// gave 385 us.  Tried and slower: a quarter, a third or an eighth of them on the FMA pipe (441, 449,
// 446 us against 433), two threads a row (601 us: registers), no halves (the same).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cz_common.cuh"
#include "cz_internal.h"

namespace cz {
namespace {

constexpr int kThreads = 384;
constexpr int kKeys = 128;     // keys per tile
constexpr uint32_t kTmemCols = 512;
// A row's old maximum stays in use until a new one is more than this many powers of two
// above it: P and l then grow to at most 2^8, far inside f32 and bf16, and most tiles
// rescale nothing.  The result does not depend on it (o and l share the factor).
constexpr float kSlack = 8.f;
// P = 2^(c S - c m) is one FMA with c m rounded, which moves a tile's weights by up to 2^-13 of themselves where c m is
// this large (and past 2^31 the rounding alone overflows the exponential).  Beyond it, which trained weights do not
// reach, m is taken off the scores in TMEM first and they are loaded again.  The code for it costs the others 0.2 of
// 6.0 us on a prompt of 77 tokens, 1-2 % on eleven packed ones, nothing on 8,192 tokens (subtracted in registers, or as a
// second form of the loop behind a branch: 0.2 us, 2-4 % and 2 %).
constexpr float kPlain = 4096.f;

struct PrefillArgs {
    CUtensorMap qmap, kmap, vmap;  // [rows][heads][D] in boxes of 64 columns
    AttnPrefillParams p;
    int group, pack, tokens;       // query heads per kv head; heads and tokens of a query tile
    int step;                      // tokens of a block's turn: two query tiles', or one's (then the second is empty)
    int htiles;                    // passes over a group's heads
    uint32_t sms;
};

template <int D>
struct Cfg {
    static constexpr int NX = D / 64;                  // 128-byte column blocks
    static constexpr int QBYTES = 128 * D * 2;
    static constexpr int KVBYTES = kKeys * D * 2;
    static constexpr int OBYTES = 8 * 32 * 128;        // the epilogue's turning room: 64 columns of a warp's rows
    static constexpr int ROOM = 227 * 1024 - 2048 - 2 * QBYTES - OBYTES;
    static constexpr int STAGES = ROOM / KVBYTES > 8 ? 8 : ROOM / KVBYTES;
    static constexpr int SMEM = 1024 + 2 * QBYTES + STAGES * KVBYTES + OBYTES;
    static constexpr uint32_t OCOL = 256;              // O of tile i at OCOL + i * 128, S of tile i at i * 128
};

struct Pair {
    int q0, nq, k0, nk, tile, head;  // sequence, pair of query tiles in it (tile < 0: no more), kv head and pass
};

struct Bars {
    uint64_t ifull[2], iempty[2];  // the picked pairs
    uint64_t qfull[2], qfree[2], full[8], empty[8], sfull[2], pready[2][2], odone[2], vask, vclean, drain;
    Pair pairs[2];
    uint32_t tmem;
    int abort, never;
};

// A value that is the same in every lane, as one the compiler knows to be.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void tma3d(uint32_t dst, const CUtensorMap* m, int x, int head, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(head), "r"(row), "r"(smem_u32(bar))
        : "memory");
}
// Shared-memory operand descriptors, 128-byte swizzle: K-major rows of 128 bytes (8-row
// groups 1024 bytes apart), or MN-major (V: keys are rows of 64 dims; 8-key groups 1024 bytes
// apart, the next 64 dims `chunk` bytes on).
__device__ __forceinline__ uint64_t desc_k(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t a, uint32_t chunk) {
    return (uint64_t)((a >> 4) & 0x3FFF) | ((uint64_t)(chunk >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16, bf16 x bf16 -> f32; bmn: B is MN-major.
__host__ __device__ constexpr uint32_t idesc(int M, int N, bool bmn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (bmn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
// The issuing warp runs converged and one elected lane issues: with warp-uniform operands the
// descriptors stay in uniform registers (issued from a divergent branch, a product cost some 100 cycles
// more than it took the tensor pipe).
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.u32 p, %4, 0;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.u32 p, %4, 0;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile(
        "{\n.reg .pred e;\nelect.sync _|e, 0xffffffff;\n"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void ld32(uint32_t* r, uint32_t a) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void ld16(uint32_t* r, uint32_t a) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void st16(uint32_t a, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(
            r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(a)
        : "memory");
}
typedef unsigned long long f2;  // two f32 in a register pair
__device__ __forceinline__ f2 pair(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(f2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Maximum of three, NaN if one is NaN.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// A bounded wait without calls (setmaxnreg and calls do not go together).
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, const volatile int* abort) {
#pragma unroll 1
    for (uint32_t it = 0; it < CZ_SPIN_LIMIT; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 15) == 15 && *abort) return false;
    }
    return false;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// A sequence's bounds; false (and reported) when they leave the buffers.
__device__ __forceinline__ bool bounds(const AttnPrefillParams& p, int b, int& q0, int& nq, int& k0, int& nk) {
    q0 = ld_now(p.cu_q + b);
    k0 = ld_now(p.cu_k + b);
    const int q1 = ld_now(p.cu_q + b + 1), k1 = ld_now(p.cu_k + b + 1);
    nq = q1 - q0;
    nk = k1 - k0;
    if (q0 < 0 || q1 < q0 || q1 > p.Tq || k0 < 0 || k1 < k0 || k1 > p.Tk) {
        nq = nk = 0;
        return false;
    }
    return true;
}
// How many of a sequence's query tile pairs (of `step` tokens) reach key x or a later one; all of
// them for x <= 0.  The pair's reach is its last token's, as if the last pair were full.
__device__ __forceinline__ int reach(int nq, int nk, int step, int x) {
    const int n = (nq + step - 1) / step;
    const int y = x - (nk - nq);  // first pair i with (i + 1) step >= y
    if (x <= 0 || y <= step) return n;
    return max(0, n - ((y + step - 1) / step - 1));
}

// One warp: the query tile pair of rank `rank`, longest reach first.  own: this lane's sequence, kept by the
// caller from pick to pick (the first 32; more are read again each time).
struct Bounds {
    int q0, nq, k0, nk;
};
// Order is by the reach in multiples of this many keys: finer than a tile, and few halvings.
constexpr int kGrain = 32;
__device__ __forceinline__ Pair pick(const AttnPrefillParams& p, int step, int rank, const Bounds& own, bool sorted) {
    const int lane = threadIdx.x & 31;
    auto get = [&](int b, int& q0, int& nq, int& k0, int& nk) {
        if (b < 32) q0 = own.q0, nq = own.nq, k0 = own.k0, nk = own.nk;
        else bounds(p, b, q0, nq, k0, nk);
    };
    auto count = [&](int x) {
        int c = 0;
#pragma unroll 1
        for (int b = lane; b < p.B; b += 32) {
            int q0, nq, k0, nk;
            get(b, q0, nq, k0, nk);
            c += reach(nq, nk, step, x * kGrain);
        }
        return (int)__reduce_add_sync(0xffffffffu, (unsigned)c);
    };
    int tile = -1, q0 = 0, nq = 0, k0 = 0, nk = 0;
    if (p.B == 1) {
        q0 = uniform(own.q0), nq = uniform(own.nq), k0 = uniform(own.k0), nk = uniform(own.nk);
        const int n = (nq + step - 1) / step;
        tile = rank < n ? n - 1 - rank : -1;
    } else {
        if (count(0) > rank) {
            int lo = 0, hi = 0x3fffffff / kGrain;  // count(lo) > rank >= count(hi); unsorted: all at once
            if (sorted) {
                int top = 0;  // past every reach
#pragma unroll 1
                for (int b = lane; b < p.B; b += 32) {
                    get(b, q0, nq, k0, nk);
                    top = max(top, nk + step);
                }
                hi = (int)__reduce_max_sync(0xffffffffu, (unsigned)top) / kGrain + 1;
#pragma unroll 1
                while (hi - lo > 1) {
                    const int mid = lo + (hi - lo) / 2;
                    if (count(mid) > rank) lo = mid;
                    else hi = mid;
                }
            }
            int left = sorted ? rank - count(hi) : rank;  // which of the pairs that reach lo but not hi
            for (int b0 = 0; b0 < p.B; b0 += 32) {
                const int b = b0 + lane;
                int c = 0;
                q0 = nq = k0 = nk = 0;
                if (b < p.B) {
                    get(b, q0, nq, k0, nk);
                    c = reach(nq, nk, step, lo * kGrain) - (sorted ? reach(nq, nk, step, hi * kGrain) : 0);
                }
                int inc = c;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += v;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, left < inc);
                if (hit) {
                    const int src = __ffs(hit) - 1;
                    const int n = (nq + step - 1) / step;
                    const int t = n - reach(nq, nk, step, lo * kGrain) + (left - (inc - c));
                    tile = __shfl_sync(0xffffffffu, t, src);
                    q0 = __shfl_sync(0xffffffffu, q0, src);
                    nq = __shfl_sync(0xffffffffu, nq, src);
                    k0 = __shfl_sync(0xffffffffu, k0, src);
                    nk = __shfl_sync(0xffffffffu, nk, src);
                    break;
                }
                left -= __shfl_sync(0xffffffffu, inc, 31);
            }
        }
    }
    return Pair{q0, nq, k0, nk, tile, 0};
}

// A pair's key tiles, per query tile: up to its last token's limit.
struct Work {
    int n0, n1, most, tok0, tok1;
    // keys of the last tile that belong to the sequence; products past them are left out, and the rows that
    // fill up the last 16 (a neighbour's, of any value) are cleared first
    int last_keys;
    bool unclean;

    __device__ __forceinline__ Work(const Pair& w, int tokens, int step) {
        tok0 = w.tile * step;
        tok1 = step > tokens ? tok0 + tokens : w.nq;
        const int a = min(w.nq, tok0 + tokens) - 1 + w.nk - w.nq, b = min(w.nq, tok1 + tokens) - 1 + w.nk - w.nq;
        n0 = tok0 >= w.nq || a < 0 ? 0 : a / kKeys + 1;
        n1 = tok1 >= w.nq || b < 0 ? 0 : b / kKeys + 1;
        most = max(n0, n1);
        last_keys = most > 0 ? min(kKeys, w.nk - (most - 1) * kKeys) : 0;
        unclean = last_keys & 15;
    }
    __device__ __forceinline__ int n(int i) const { return i ? n1 : n0; }
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1) attn_prefill_kernel(const __grid_constant__ PrefillArgs A) {
    using C = Cfg<D>;
    const AttnPrefillParams& p = A.p;
    extern __shared__ uint8_t raw[];
    uint8_t* sq = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    uint8_t* skv = sq + 2 * C::QBYTES;
    __shared__ Bars B;
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (warp == 8 && lane == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.ifull[i], 1);
            mbar_init(&B.iempty[i], 11);  // loads, products, 8 softmax warps, the clearing warp
            mbar_init(&B.qfull[i], 1);
            mbar_init(&B.qfree[i], 1);
            mbar_init(&B.sfull[i], 1);
            mbar_init(&B.pready[i][0], 4);
            mbar_init(&B.pready[i][1], 4);
            mbar_init(&B.odone[i], 1);
        }
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&B.full[i], 1);
            mbar_init(&B.empty[i], 1);
        }
        mbar_init(&B.vask, 1);
        mbar_init(&B.vclean, 1);
        mbar_init(&B.drain, 1);
        B.abort = B.never = 0;
        fence_mbarrier_init();
        prefetch_tensormap(&A.qmap);
        prefetch_tensormap(&A.kmap);
        prefetch_tensormap(&A.vmap);
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    pdl_wait();
    __syncthreads();
    fence_after();
    const uint32_t tmem = (uint32_t)uniform((int)B.tmem);
    volatile int* abort = &B.abort;

    auto gave_up = [&]() {
        *abort = 1;
        atomicOr(p.err, kAttnErrWait);
    };
    // The t-th pair of this block, as the picking warp hands it out; false when there are no more.
    auto next_pair = [&](int t, Pair& w) {
        const int at = t & 1;
        const bool ok = __all_sync(0xffffffffu, wait_bar(&B.ifull[at], (t >> 1) & 1, abort));
        if (!ok) {
            gave_up();
            return false;
        }
        const Pair& x = B.pairs[at];
        w.q0 = uniform(x.q0);
        w.nq = uniform(x.nq);
        w.k0 = uniform(x.k0);
        w.nk = uniform(x.nk);
        w.tile = uniform(x.tile);
        w.head = uniform(x.head);
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.iempty[at]);
        return w.tile >= 0;
    };

    // registers: 2 x 208 + 88 = 3 x 168, what the block was launched with
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8) {
            // ---------------- loads ----------------
            const uint32_t qbytes = (uint32_t)(A.tokens * A.pack) * 128 * C::NX;
            int issued = 0, qused[2] = {0, 0};
            bool ok = true;
            Pair w;
#pragma unroll 1
            for (int t = 0; ok && next_pair(t, w); ++t) {
                const Work k(w, A.tokens, A.step);
                const int kh = w.head / A.htiles, head = kh * A.group + (w.head % A.htiles) * A.pack;
                auto load_q = [&](int i) {
                    if (k.n(i) == 0) return true;
                    if (qused[i] && !wait_bar(&B.qfree[i], (qused[i] - 1) & 1, abort)) return false;
                    ++qused[i];
                    mbar_arrive_expect_tx(&B.qfull[i], qbytes);
#pragma unroll
                    for (int x = 0; x < C::NX; ++x)
                        tma3d(smem_u32(sq + i * C::QBYTES + x * 128 * 128), &A.qmap, x * 64, head,
                              w.q0 + (i ? k.tok1 : k.tok0), &B.qfull[i]);
                    return true;
                };
                auto load_kv = [&](const CUtensorMap* m, int j) {
                    const int s = issued % C::STAGES;
                    if (issued >= C::STAGES && !wait_bar(&B.empty[s], ((issued / C::STAGES) & 1) ^ 1, abort)) return false;
                    mbar_arrive_expect_tx(&B.full[s], C::KVBYTES);
#pragma unroll
                    for (int x = 0; x < C::NX; ++x)
                        tma3d(smem_u32(skv + s * C::KVBYTES + x * kKeys * 128), m, x * 64, kh, w.k0 + j * kKeys, &B.full[s]);
                    ++issued;
                    return true;
                };
                if (k.most > 0 && lane == 0) {
                    ok = load_kv(&A.kmap, 0) && load_q(0) && load_q(1) && load_kv(&A.vmap, 0);
#pragma unroll 1
                    for (int j = 1; j < k.most && ok; ++j) ok = load_kv(&A.kmap, j) && load_kv(&A.vmap, j);
                    if (!ok) gave_up();
                }
                ok = uniform(ok);
            }
            // no copy stays in flight behind the block's end (all have landed unless a wait gave up)
            if (lane == 0) {
                for (int i = max(0, issued - C::STAGES); i < issued; ++i)
                    if (!wait_bar(&B.full[i % C::STAGES], (i / C::STAGES) & 1, &B.never)) gave_up();
                for (int i = 0; i < 2; ++i)
                    if (qused[i] && !wait_bar(&B.qfull[i], (qused[i] - 1) & 1, &B.never)) gave_up();
            }
            __syncwarp();
        } else if (warp == 9) {
            // ---------------- products ----------------
            constexpr uint32_t IDS = idesc(128, kKeys, false), IDO = idesc(128, D, true);
            const uint64_t dq = desc_k(smem_u32(sq)), dk = desc_k(smem_u32(skv));
            const uint64_t dv = desc_mn(smem_u32(skv), kKeys * 128);
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                const bool ok = __all_sync(0xffffffffu, wait_bar(bar, parity, abort));
                if (!ok) gave_up();
                return ok;
            };
            // the ring's uses in order: K_0, V_0, K_1, V_1, ... of one pair after the other
            int ustage = 0;
            uint32_t uphase = 0, qphase[2] = {0, 0}, pphase[2] = {0, 0}, vphase = 0;
            auto wait_kv = [&]() { return wait(&B.full[ustage], uphase); };
            auto next_kv = [&]() {
                const int st = ustage;
                if (++ustage == C::STAGES) ustage = 0, uphase ^= 1;
                return st;
            };
            auto qk = [&](int i, int st, bool last) {  // S_i = Q_i K^T
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (k / 4) * (128 * 128 / 16) + (k % 4) * 2;
                    mma_ss(tmem + i * 128, dq + (uint32_t)(i * C::QBYTES / 16 + off),
                           dk + (uint32_t)(st * C::KVBYTES / 16 + off), IDS, k > 0);
                }
                commit(&B.sfull[i]);
                if (last) commit(&B.qfree[i]);
            };
            bool ok = true;
            Pair w;
#pragma unroll 1
            for (int t = 0; ok && next_pair(t, w); ++t) {
                const Work work(w, A.tokens, A.step);
                if (work.most == 0) continue;
                ok = wait_kv();
                int kst = next_kv();
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (ok && work.n(i) > 0) {
                        ok = wait(&B.qfull[i], qphase[i]);
                        qphase[i] ^= 1;
                        if (ok) qk(i, kst, work.n(i) == 1);
                    }
                if (ok) commit(&B.empty[kst]);
#pragma unroll 1
                for (int j = 0; j < work.most && ok; ++j) {
                    const bool more = j + 1 < work.most;
                    const int ksteps = more ? kKeys / 16 : (work.last_keys + 15) / 16;
                    ok = wait_kv();
                    if (!ok) break;
                    bool ask = work.unclean && !more;
                    if (ask && lane == 0) mbar_arrive(&B.vask);
                    __syncwarp();
                    const int vst = next_kv();
                    bool kwait = more;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (j >= work.n(i) || !ok) continue;
                        auto pv = [&](int k) {
                            if (k < ksteps)
                                mma_ts(tmem + C::OCOL + i * 128, tmem + i * 128 + k * 8,
                                       dv + (uint32_t)((vst * C::KVBYTES + k * 2048) / 16), IDO, j > 0 || k > 0);
                        };
                        // the first 64 keys' products run under the other weights' exponentials
                        ok = wait(&B.pready[i][0], pphase[i]) && (!ask || wait(&B.vclean, vphase));
                        if (!ok) continue;
                        if (ask) vphase ^= 1;
                        ask = false;
                        fence_after();
#pragma unroll
                        for (int k = 0; k < 4; ++k) pv(k);
                        ok = wait(&B.pready[i][1], pphase[i]);
                        if (!ok) continue;
                        pphase[i] ^= 1;
                        fence_after();
#pragma unroll
                        for (int k = 4; k < 8; ++k) pv(k);
                        if (j + 1 == work.n(i)) {
                            commit(&B.odone[i]);
                        } else {
                            if (kwait) {
                                ok = wait_kv();
                                kst = next_kv();
                                kwait = false;
                            }
                            // into S_i: in order behind the product that reads P_i from it
                            if (ok) qk(i, kst, j + 2 == work.n(i));
                        }
                    }
                    if (!ok) break;
                    commit(&B.empty[vst]);
                    if (more) commit(&B.empty[kst]);
                }
            }
            // every product has finished before TMEM is given back
            commit(&B.drain);
            if (!wait_bar(&B.drain, 0, &B.never)) gave_up();
            __syncwarp();
        } else if (warp == 10) {
            // ---------------- the block's pairs, in turn from either end of each round ----------------
            const int heads = (int)p.kv_heads * A.htiles;
            const bool sorted = gridDim.x == A.sms;  // (fewer blocks: a turn each, in any order)
            Bounds own = {0, 0, 0, 0};
            if (lane < p.B && !bounds(p, lane, own.q0, own.nq, own.k0, own.nk)) atomicOr(p.err, kAttnErrIndex);
            if (blockIdx.x == 0) {
                Bounds x;
#pragma unroll 1
                for (int b = lane + 32; b < p.B; b += 32)
                    if (!bounds(p, b, x.q0, x.nq, x.k0, x.nk)) atomicOr(p.err, kAttnErrIndex);
            }
#pragma unroll 1
            for (int t = 0;; ++t) {
                const int at = t & 1;
                if (t >= 2 && !__all_sync(0xffffffffu, wait_bar(&B.iempty[at], ((t >> 1) & 1) ^ 1, abort))) {
                    gave_up();
                    break;
                }
                const uint32_t item = t * gridDim.x + (t & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                Pair w = pick(p, A.step, (int)(item / heads), own, sorted);
                w.head = (int)(item % heads);
                if (lane == 0) {
                    B.pairs[at] = w;
                    mbar_arrive(&B.ifull[at]);
                }
                if (w.tile < 0) break;
            }
        } else {
            // ---------------- what lies behind the last values ----------------
            int uses = 0;
            uint32_t phase = 0;
            Pair w;
#pragma unroll 1
            for (int t = 0; next_pair(t, w); ++t) {
                const Work k(w, A.tokens, A.step);
                uses += 2 * k.most;
                if (!k.unclean) continue;
                if (!__all_sync(0xffffffffu, wait_bar(&B.vask, phase, abort))) {
                    gave_up();
                    break;
                }
                phase ^= 1;
                uint8_t* v = skv + ((uses - 1) % C::STAGES) * C::KVBYTES;
                for (int i = lane; i < (16 - (k.last_keys & 15)) * 8 * C::NX; i += 32) {
                    const int r = k.last_keys + i / (8 * C::NX), c = i % (8 * C::NX);
                    *reinterpret_cast<uint4*>(v + (c >> 3) * kKeys * 128 + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.vclean);
            }
        }
    } else {
        // ---------------- softmax: a thread a row ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int i = warp >> 2;
        const int r = (warp & 3) * 32 + lane;
        const int lt = r / A.pack, lh = r % A.pack;
        const uint32_t quad = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t sa = tmem + quad + i * 128, oa = tmem + quad + C::OCOL + i * 128;
        const float c = p.scale * 1.4426950408889634f;
        uint32_t sphase = 0, ophase = 0;
        bool ok = true;
        Pair w;
#pragma unroll 1
        for (int turn = 0; ok && next_pair(turn, w); ++turn) {
            const Work work(w, A.tokens, A.step);
            const int tok = i ? work.tok1 : work.tok0, tiles = work.n(i);
            const int kh = w.head / A.htiles, head0 = (w.head % A.htiles) * A.pack;  // first query head of the group's pass
            const int t = tok + lt;
            const bool live = lt < A.tokens && t < w.nq && head0 + lh < A.group;
            const int lim0 = tok + w.nk - w.nq;  // the tile's first token's limit
            const int lim = live ? t + w.nk - w.nq : 0x7fffffff;
            float m = -INFINITY, l = 0.f;
            bool big = false;  // some row's maximum is past kPlain
#pragma unroll 1
            for (int j = 0; j < tiles; ++j) {
                ok = __all_sync(0xffffffffu, wait_bar(&B.sfull[i], sphase, abort));
                if (!ok) {
                    gave_up();
                    break;
                }
                sphase ^= 1;
                fence_after();
                uint32_t sv[kKeys];
                float mc = 0.f;
#pragma unroll 1
                for (bool again = false;; again = true) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) ld32(sv + x * 32, sa + x * 32);
                    wait_ld();
                    if (j * kKeys + kKeys - 1 > lim0) {
                        const int cut = lim - j * kKeys;  // columns past it are not seen
#pragma unroll
                        for (int x = 0; x < kKeys; ++x)
                            if (x > cut) sv[x] = 0xff800000u;
                    }
                    if (again) break;
                    float mx[4] = {m, m, m, m};
#pragma unroll
                    for (int x = 0; x < kKeys; x += 8)
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            mx[y] = max3(mx[y], __uint_as_float(sv[x + 2 * y]), __uint_as_float(sv[x + 2 * y + 1]));
                    const float top = max3(mx[0], mx[1], max3(mx[2], mx[2], mx[3]));
                    if (j == 0) {
                        m = top;
                        big = __any_sync(0xffffffffu, live && fabsf(m * c) > kPlain);
                    } else if (__any_sync(0xffffffffu, live && !((top - m) * c <= kSlack))) {
                        // the products into O behind this tile's S have finished: S's completion covers them
                        const float a = top == m ? 1.f : ex2((m - top) * c);
                        m = top;
                        big = __any_sync(0xffffffffu, live && fabsf(m * c) > kPlain);
                        l *= a;
#pragma unroll 1
                        for (int x = 0; x < D / 16; ++x) {
                            uint32_t o[16];
                            ld16(o, oa + x * 16);
                            wait_ld();
#pragma unroll
                            for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * a);
                            st16(oa + x * 16, o);
                        }
                    }
                    mc = m == -INFINITY ? 0.f : m * c;
                    if (!big) break;
                    const float less = fabsf(mc) > kPlain ? m : 0.f;
#pragma unroll 1
                    for (int x = 0; x < kKeys / 16; ++x) {
                        uint32_t t[16];
                        ld16(t, sa + x * 16);
                        wait_ld();
#pragma unroll
                        for (int y = 0; y < 16; ++y) t[y] = __float_as_uint(__uint_as_float(t[y]) - less);
                        st16(sa + x * 16, t);
                    }
                    wait_st();
                    if (less != 0.f) mc = 0.f;
                }
                const f2 cc = pair(c, c), mm = pair(-mc, -mc);
                f2 sum0 = 0, sum1 = 0;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t pk[16];
#pragma unroll
                    for (int y = 0; y < 16; ++y) {
                        const f2 t = fma2(pair(__uint_as_float(sv[x * 32 + 2 * y]), __uint_as_float(sv[x * 32 + 2 * y + 1])), cc, mm);
                        float e0, e1;
                        unpair(t, e0, e1);
                        e0 = ex2(e0);
                        e1 = ex2(e1);
                        if (y & 1) sum1 = add2(sum1, pair(e0, e1));
                        else sum0 = add2(sum0, pair(e0, e1));
                        pk[y] = pack_bf16(e0, e1);  // the second product's operand; its sums stay in f32
                    }
                    st16(sa + x * 16, pk);  // over columns that are in registers by now
                    if (x & 1) {
                        wait_st();
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&B.pready[i][x >> 1]);
                    }
                }
                float e0, e1;
                unpair(add2(sum0, sum1), e0, e1);
                l += e0 + e1;
            }
            if (ok && tiles > 0) {
                ok = __all_sync(0xffffffffu, wait_bar(&B.odone[i], ophase, abort));
                if (!ok) gave_up();
                ophase ^= 1;
                fence_after();
            }
            if (ok) {
                const float inv = m == -INFINITY ? 0.f : 1.f / l;  // no key seen: zeros
                // A thread has a row, whose 16-byte pieces would go to 32 lines in one store: turned in shared
                // memory (64 columns at a time, pieces swizzled by the row), a store covers four whole lines.
                uint8_t* room = skv + C::STAGES * C::KVBYTES + warp * 32 * 128;
                const unsigned long long row =
                    live ? ((unsigned long long)(w.q0 + t) * p.q_heads + (unsigned)(kh * A.group + head0 + lh)) * D : ~0ull;
#pragma unroll
                for (int x = 0; x < D / 64; ++x) {
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        uint32_t o[32];
                        if (tiles > 0) {
                            ld32(o, oa + x * 64 + y * 32);
                            wait_ld();
                        }
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            uint32_t v[4];
#pragma unroll
                            for (int u = 0; u < 4; ++u)
                                v[u] = inv == 0.f ? 0u
                                                  : pack_bf16(__uint_as_float(o[z * 8 + 2 * u]) * inv,
                                                              __uint_as_float(o[z * 8 + 2 * u + 1]) * inv);
                            *reinterpret_cast<uint4*>(room + lane * 128 + (((y * 4 + z) ^ (lane & 7)) << 4)) =
                                make_uint4(v[0], v[1], v[2], v[3]);
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        const int r4 = y * 4 + (lane >> 3), piece = lane & 7;
                        const unsigned long long at = __shfl_sync(0xffffffffu, row, r4);
                        const uint4 v = *reinterpret_cast<const uint4*>(room + r4 * 128 + ((piece ^ (r4 & 7)) << 4));
                        if (at != ~0ull) *reinterpret_cast<uint4*>(p.out + at + x * 64 + piece * 8) = v;
                    }
                    __syncwarp();
                }
            }
            fence_before();  // O is read before the next pair's weights are announced, and its products overwrite it
        }
    }
    __syncthreads();
    if (warp == 9)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

bool make_map(CUtensorMap* map, const uint16_t* base, uint64_t rows, uint64_t heads, uint64_t dim, uint64_t stride,
              uint32_t box_heads, uint32_t box_rows) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[3] = {dim, heads, rows};
    const cuuint64_t strides[2] = {dim * 2, stride * 2};
    const cuuint32_t box[3] = {64, box_heads, box_rows};
    const cuuint32_t one[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t*>(base), dims, strides, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// One prompt in turns of `step` tokens: what the busiest block's turns take, in hundredths of a pair's time on a key
// tile.  A single query tile takes 0.94 of that (0.9 with heads of 64), a further turn 1.5 of it to begin and end.
uint64_t busiest(const AttnPrefillParams& p, int step, bool pair, int64_t heads, int num_sms) {
    const uint64_t tile = pair ? 100 : p.head_dim == 64 ? 90 : 94;
    const int64_t n = ((int64_t)p.Tq + step - 1) / step, turns = n * heads;
    uint64_t most = 0;
    for (int64_t x = 0; x < num_sms && x < turns; ++x) {
        uint64_t sum = 0;
        for (int64_t t = 0;; ++t) {  // as the picking warp goes: longest first, in turn from either end
            const int64_t item = t * num_sms + (t & 1 ? num_sms - 1 - x : x);
            if (item >= turns) break;
            const int64_t end = (n - item / heads) * step;  // the turn's last query's keys
            const int64_t keys = (end < p.Tq ? end : p.Tq) + (int64_t)p.Tk - p.Tq;
            sum += (t ? 150 : 0) + (keys > 0 ? (uint64_t)(keys + kKeys - 1) / kKeys * tile : 0);
        }
        if (sum > most) most = sum;
    }
    return most;
}

template <int D>
int launch(const PrefillArgs& a, uint32_t grid, cudaStream_t st) {
    static uint32_t set = 0;  // the library's lock is held
    if (set != init_serial) {
        if (cudaFuncSetAttribute(attn_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 Cfg<D>::SMEM) != cudaSuccess)
            return CZ_ELAUNCH;
        set = init_serial;
    }
    return launch_early(attn_prefill_kernel<D>, grid, kThreads, Cfg<D>::SMEM, st, a) ? CZ_OK : CZ_ELAUNCH;
}

}  // namespace

int attn_prefill_launch(const AttnPrefillParams& p, int num_sms, cudaStream_t st) {
    PrefillArgs a{};
    a.p = p;
    a.group = (int)(p.q_heads / p.kv_heads);
    a.htiles = (a.group + 127) / 128;
    a.pack = (a.group + a.htiles - 1) / a.htiles;
    a.tokens = 128 / a.pack;
    // Turns at most.  One query tile each where that still leaves SMs idle.  One prompt whose pairs do: by the key tiles
    // of the block that gets most, single against pairs (`busiest`).  Measured: 8 heads on 1 of 64, 2,400 tokens 32.6
    // against 36.1 us, 4,600 59.7 against 64.5, but 3,000 after 3,000 keys 91.0 against 83.7; 12 on 2 of 128, 2,000
    // tokens 31.0 against 32.8, but 2,500 after 2,500 keys 96.6 against 73.5; 32 on 4 of 128, 600 tokens 13.9 against
    // 14.7, 900 18.8 against 18.4, but 1,100 23.3 against 21.7, 700 after 4,000 keys 111.1 against 67.5.  Several prompts
    // of more single tiles than SMs take pairs (their lengths are on the device): 2 of 350 tokens 12.1 against 15.6.
    const uint64_t heads = (uint64_t)p.kv_heads * a.htiles;
    const uint64_t single = ((uint64_t)p.Tq / a.tokens + p.B) * heads;
    const uint64_t pairs = ((uint64_t)p.Tq / (2 * a.tokens) + p.B) * heads;
    const uint64_t sms = (uint64_t)num_sms;
    const auto most = [&](int step, bool pair) { return busiest(p, step, pair, (int64_t)heads, num_sms); };
    const bool one = single <= sms || (p.B == 1 && pairs <= sms && most(a.tokens, false) < most(2 * a.tokens, true));
    a.step = one ? a.tokens : 2 * a.tokens;
    const uint64_t turns = ((uint64_t)p.Tq / a.step + p.B) * heads;
    if (turns > 0x3fffffffu) return CZ_ESHAPE;
    a.sms = (uint32_t)num_sms;
    const uint32_t grid = turns < (uint64_t)num_sms ? (uint32_t)turns : (uint32_t)num_sms;
    if (!make_map(&a.qmap, p.q, p.Tq, p.q_heads, p.head_dim, p.q_stride, a.pack, a.tokens)) return CZ_ESHAPE;
    if (p.Tk == 0) {  // nothing is loaded then: the kernel checks the bounds and writes the sequences' zeros
        a.kmap = a.vmap = a.qmap;
    } else if (!make_map(&a.kmap, p.k, p.Tk, p.kv_heads, p.head_dim, p.k_stride, 1, kKeys) ||
               !make_map(&a.vmap, p.v, p.Tk, p.kv_heads, p.head_dim, p.v_stride, 1, kKeys)) {
        return CZ_ESHAPE;
    }
    return p.head_dim == 128 ? launch<128>(a, grid, st) : launch<64>(a, grid, st);
}

}  // namespace cz
