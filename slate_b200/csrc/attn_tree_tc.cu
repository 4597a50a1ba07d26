// attn_tree_tc.cu -- tree attention for many rows on the tcgen05 tensor cores
// (f16 and 8-bit caches, head_dim 64 and 128; attn_tree.cu has the formula, the
// split of f32 values into f16 pairs and the few-row kernels).
//
// One CTA an SM.  A tile of 128 rows (nodes x group) stays: q as f16 hi and lo in
// tensor memory.  The cache streams past in tiles of 128 tokens:
//   S = Qhi K^T + Qlo K^T           128 x 128, in tensor memory, f32
//   P = exp(S - max), hi and lo     written over S, the next product's A operand
//   D += Phi V + Plo V              128 x head_dim, in tensor memory
//   O += D, D = 0                   in registers, every RUN tiles or when a maximum grew by 2^LAG
// S has two buffers: while the softmax warps work on tile j, the tensor cores run P V of
// tile j - 1 and Q K^T of tile j + 1.
// Warps 0-7: softmax; two threads share a row, each with half of the tile's tokens (they
// exchange the row's maximum) and of O's dims.  Four threads a row hid no more of the latency
// and left each too few registers.  Warps 8-14 bring K and V page by page in turn into the
// operands' swizzled layout (f16: 16-byte asynchronous copies; 8 bits: through registers, two
// pages ahead, widened to f16 on the way).  Warp 15 issues the products.
// q comes and O leaves a row at a time through the tiles' shared memory (a thread that read or wrote
// its own row moved a sector an element: 15.5 us for one tile a CTA against 21.8).
// SPLIT, up to 64 rows: lanes 64-127 would idle, and the softmax of a tile is what the next waits for;
// so they hold the rows again, each lane takes half of a tile's tokens (P is 0 for the others), and
// a row's two lanes are joined like two CTAs' parts (8 x 16 nodes of f16: 51 us against 54, at
// head_dim 64 44 against 47.5, of 8 bits 60 against 64).
// What bounds it.  256 rows and more over long contexts (4 sequences of 64 nodes, 64 heads over
// 8, 32000 tokens of 8 bits: 438 us, 413 TFLOP/s of the formula, 827 with both halves): the softmax's
// issue slots (59 % busy), two passes over S with an exponential and a split a score, next to tensor cores that
// are busy about half of the time.  Few rows (8 sequences of 16 nodes, 32 heads over 8, 8000 tokens
// of f16: 51 us, 3.1 TB/s): the loads within the tiles, then what a CTA does before the first tile
// and after the last, some 20 us of the call.  8 bits with as few rows (60 us, 1.4 TB/s): widening K and V to f16
// through registers, with two buffers, for products of which half are padding.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "sb_internal.h"
#include "sb_kernels.h"
#include "sb_kv.h"
#include "sb_pdl.h"
#include "sb_tree.h"

using namespace sb_tree;

namespace {

constexpr int MR = 128, KT = 128;
constexpr int PARTS = 2;                      // threads that share a row
constexpr int NSW = 4 * PARTS, NPW = 7, NTHREADS = 32 * (NSW + NPW + 1);
constexpr uint64_t WAIT_NS = 2000000000ull;
constexpr int SCB = 8;                        // tiles whose scales and flags are kept: NB + 3 are in use
// The maximum that p is taken against may lag behind the true one by 2^LAG: only then are O and
// the sum rescaled.  p carries 2^(15 - LAG), so that it stays below f16's end all the same.
constexpr int LAG = 8;
// 8 bits: as long as a range's v scales lie within 2^SPAN (and below 2^TALL), p v's factor in f16 is set
// by the largest of them, for all rows alike: a row's top token then keeps 31 - SPAN bits, and the sum l takes the
// same factor.  From the first tile on where they do not, each row has its own, by the tokens that it sees and
// their p, and l none (see `wide`): 4 x 64 nodes over 32000 tokens 774 us instead of 438, 8 x 16 over 8000 75 instead
// of 60.  Scales that spread like exp(normal / 2) stay within 2^7.
constexpr int SPAN = 10, TALL = 40;
// Tiles that D may add up before it is drained (a power of two).  The tensor cores cut each
// step's sum off: 8 tiles, 128 steps, cost 1e-6 of the output at worst, one tile 1e-7.
constexpr int RUN = 8;

template <int KV, int HD>
struct TcShape {
    // K and V tiles in shared memory, of each: the 8-bit producers go through registers and
    // the first-level cache, which a third pair would leave little of (256 rows over 32000 tokens took 550 us with
    // three, 490 with two, when this was chosen); f16 keeps more copies in flight with three (64 rows 66 us, with two 76)
    static constexpr int NB = KV == SLATE_KV_Q8 ? 2 : 3;
    static constexpr int TB = KT * HD * 2;                 // a K or V tile in f16
    static constexpr int SC = SCB * 2 * KT * 4;
    static constexpr int SMEM = 2 * NB * TB + SC + 1024;
    // q and O pass through the tiles; f16: behind K and all but the last page of V of a CTA's first
    // tile, which come in meanwhile
    static constexpr int STAGE = KV == SLATE_KV_Q8 ? 0 : 2 * NB * TB - MR * (HD + 1) * 4;
    static_assert(KV == SLATE_KV_Q8 ? MR * (HD + 1) * 4 <= 2 * NB * TB : STAGE >= (NB + 1) * TB - 16 * 128, "");
};

struct Yes {
    static constexpr bool value = true;
};
struct No {
    static constexpr bool value = false;
};

template <int NB>
struct Bars {
    uint64_t kfull[NB], kfree[NB], vfull[NB], vfree[NB], sfull[2], pfull[2], dfull[2];
};

__device__ __forceinline__ uint64_t gtimer() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t c) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(c));
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    // the thread may sleep up to 2 us in the instruction: a spin would take the softmax's issue slots
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}\n"
                 : "=r"(ok) : "r"(su32(b)), "r"(parity), "r"(2000) : "memory");
    return ok != 0;
}
// Bounded: false, and the CTA's fail word set, after WAIT_NS or once another warp failed.
__device__ __forceinline__ bool bar_wait_slow(uint64_t* b, uint32_t parity, volatile int* fail) {
    const uint64_t t0 = gtimer();
    for (uint32_t n = 1;; ++n) {
        if (bar_try(b, parity)) return true;
        if ((n & 31) == 0) {
            if (*fail) return false;
            if (gtimer() - t0 > WAIT_NS) {
                *fail = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile int* fail) {
    return bar_try(b, parity) || bar_wait_slow(b, parity, fail);
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 128-byte swizzle, 8-row groups 1024 bytes apart.  K-major operands (q, K: the product
// runs along a row) ignore lbo; for the MN-major V (the product runs along the rows) lbo is
// the step from 64 dims to the next.
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
                 "r"(acc));
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar))
                 : "memory");
}
// 16 columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_ld(uint32_t a, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), 
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), 
                 "=r"(r[15])
                 : "r"(a));
}
__device__ __forceinline__ void tmem_st(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(a),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), 
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void softmax_sync() {
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(32 * NSW) : "memory");
}
// Byte of 16-byte chunk ch (8 f16) of row r in an operand of 128 rows: 64 columns a
// 16 KB block, rows of 128 bytes, chunks exchanged by the row's low bits.
__device__ __forceinline__ uint32_t op_at(int r, int ch) {
    return (uint32_t)((ch >> 3) * 16384 + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
}

// The CTA's segments: each a run of tiles of one item.  In shared memory, advanced by one
// thread: the roles have no registers to spare for it.
struct Segs {
    int64_t at, stop, seq_before;
    int s, seg, unit;                   // unit: in tokens, a multiple of KT
    Seq sq;
    int nt, kvh, r_base, n_rows, end, tok0;
    bool whole;
    __device__ __forceinline__ bool next(const slate_kv_cache_t& c, const slate_tree_t& tr, int G) {
        if (at >= stop) return false;
        while (at >= seq_before + seq_units(sq, c.n_kv_heads)) {
            seq_before += seq_units(sq, c.n_kv_heads);
            sq = seq_of(c, tr, ++s, G, MR, unit);
        }
        int u0;
        const int item = item_of(at - seq_before, sq.units, u0), nu = (int)min((int64_t)sq.units, u0 + (stop - at)) - u0;
        kvh = item / sq.tiles;
        r_base = (item % sq.tiles) * MR;
        n_rows = min(MR, sq.n * G - r_base);
        end = sq.ctx + sq.n;
        tok0 = u0 * unit;
        nt = (min(end - tok0, nu * unit) + KT - 1) / KT;
        whole = nu == sq.units;
        at += nu;
        ++seg;
        return true;
    }
};

template <int KV, int HD, bool SPLIT>
__global__ void __launch_bounds__(NTHREADS, 1) attn_tree_tc(
    const slate_kv_cache_t c, int layer, const slate_tree_t tr, int nq, float* __restrict__ out,
    int ld_out, const float* __restrict__ q, int ld_q, float scale, float* __restrict__ ws) {
    using S = TcShape<KV, HD>;
    constexpr bool Q8 = KV == SLATE_KV_Q8;
    constexpr int KS = HD / 16, NB = S::NB;
    extern __shared__ unsigned char smem_raw[];
    // by an offset, so that the compiler still knows it for shared memory
    unsigned char* smem = smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u);
    unsigned char* skv = smem;                                  // NB of K, NB of V
    float* ssc = (float*)(skv + 2 * NB * S::TB);                      // [SCB][K, V][KT]
    __shared__ Bars<NB> bars;
    __shared__ Segs sg;
    __shared__ int more_s;
    __shared__ PlanBuf buf;
    __shared__ uint32_t tmem_s;
    __shared__ __align__(8) uint8_t gone_s[SCB][8];                // per page: the table has none
    __shared__ uint16_t odd_s[SCB][8];                             // per page: tokens whose v is not finite
    __shared__ uint2 vends_s[SCB];                                 // bits of the tile's largest v scale; 0 - those of the
                                                                   // smallest (0: it has none)
    __shared__ float part_max[2][PARTS][MR];      // [tile parity][part][row]
    __shared__ float part_top[Q8 ? 2 : 1][PARTS][Q8 ? MR : 1];     // alike, of score + exponent of the v scale
    __shared__ int need_s[4];                     // tile % 4: some row's maximum grew beyond LAG
    __shared__ int fail_s;
    sb_grid_wait();
    sb_grid_release();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nkv = c.n_kv_heads, G = nq / nkv;
    Start st_;
    int unit = KT;
    if (!plan_start(c, tr, G, MR, unit, TC_SLACK, gridDim.x, buf, st_)) return;
    if (tid == 0) {
        nan_words(ws, HD)[blockIdx.x] = 0;
        for (int i = 0; i < NB; ++i) {
            bar_init(&bars.kfull[i], 8);          // pages
            bar_init(&bars.vfull[i], 8);
            bar_init(&bars.kfree[i], 1);
            bar_init(&bars.vfree[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&bars.sfull[i], 1);
            bar_init(&bars.pfull[i], 32 * NSW);
            bar_init(&bars.dfull[i], 1);
        }
        for (int i = 0; i < 4; ++i) need_s[i] = 0;
        for (int i = 0; i < SCB; ++i) vends_s[i] = make_uint2(0, 0);
        fail_s = 0;
        sg.at = st_.at;
        sg.stop = st_.stop;
        sg.seg = -1;
        sg.unit = unit;
        sg.s = st_.sq.s;
        sg.seq_before = st_.seq_before;
        sg.sq = st_.sq;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == NSW + NPW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&tmem_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_before();
    }
    __syncthreads();
    tc_after();
    const uint32_t tmem = tmem_s;
    // Every role walks the same segments; four barriers of the CTA a segment: the last one has
    // left the buffers, the next is known, q is there, every product is done and the half rows'
    // sums are there.
    const auto next_segment = [&]() {
        __syncthreads();
        if (tid == 0) more_s = sg.next(c, tr, G);
        __syncthreads();
        return more_s != 0;
    };
    // tensor memory: S / P of even and odd tiles, D, q's high halves, q's low halves
    const auto sS = [&](int b) { return tmem + 128u * b; };
    const uint32_t sD = tmem + 256, sQ = tmem + 384;
    // Tiles before this segment.  Tile t of them all uses S / P t % 2, K and V buffer t % NB,
    // scales t % SCB, and each barrier's phase is how often its buffer was used before.
    uint32_t tb = 0;
    const auto phase2 = [](uint32_t t) { return t >> 1 & 1; };
    const auto phaseN = [](uint32_t t) { return t / NB & 1; };
    volatile int* fail = &fail_s;

    if (warp < NSW) {
        // no spills: with 227 KB of shared memory the first-level cache is too small to hold them
        asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
        while (next_segment()) {
            const Seq& sq_ = sg.sq;
            const int nt = sg.nt, kvh = sg.kvh, r_base = sg.r_base, n_rows = sg.n_rows, tok0 = sg.tok0;
            // ================= softmax: thread = row, part h of the tile's tokens and of O's dims
            // SPLIT: lanes 64-127 hold rows 0-63 again; a row's two lanes take half of the tokens each and
            // are joined at the segment's end
            constexpr int HO = HD / PARTS, TQ = KT / PARTS / (SPLIT ? 2 : 1), RMASK = SPLIT ? 63 : 127;
            const int h = warp >> 2, r = tid & 127, rq = r & RMASK;     // lane; row
            const auto toff = [&]() { return TQ * h + (SPLIT ? r & 64 : 0); };     // the thread's first token of a tile
            const bool live = ((warp & 3) * 32 & RMASK) < n_rows;       // of the warp
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            // ---- q, each row divided by a power of two, so that its halves have their bits down to 2^-18 of its
            // ---- maximum; scale's sign joins q
            // ---- (a row at a time through the K and V tiles, which nobody else uses yet: a thread that
            // read its own row would ask for a sector an element)
            float O[HO];
            {
                float* stage = (float*)(skv + S::STAGE);
                for (int i0 = warp; i0 < n_rows; i0 += 4 * NSW) {
                    float x[4][HD / 32];               // four rows in flight
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int rr = r_base + min(i0 + u * NSW, n_rows - 1);
                        const float* src = q + (size_t)(sq_.r0 + rr / G) * ld_q + (size_t)(kvh * G + rr % G) * HD + lane;
#pragma unroll
                        for (int k = 0; k < HD / 32; ++k) x[u][k] = src[32 * k];
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int k = 0; k < HD / 32; ++k)
                            if (i0 + u * NSW < n_rows) stage[(i0 + u * NSW) * (HD + 1) + lane + 32 * k] = x[u][k];
                }
                softmax_sync();
                const float* x = stage + min(rq, n_rows - 1) * (HD + 1) + HO * h;
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < HO; ++i) {
                    O[i] = x[i];
                    top = max(top, __float_as_uint(O[i]) & 0x7fffffffu);
                }
                part_max[0][h][r] = __uint_as_float(top);
            }
            softmax_sync();
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < PARTS; ++i) top = max(top, __float_as_uint(part_max[0][i][r]));
            const int qe = min(max((int)(top >> 23) - 127, -112), 126) - 14;   // the largest becomes 2^14 to 2^15
            const float rs = fabsf(scale) * 1.4426950408889634f * __int_as_float((127 + qe) << 23);
            {
                const float inv = copysignf(__int_as_float((127 - qe) << 23), scale);
#pragma unroll
                for (int i = 0; i < HO; i += 16) {
                    uint32_t hl[16];                   // 8 pairs' high halves, then their low halves
#pragma unroll
                    for (int e = 0; e < 16; e += 2) split_f16(O[i + e] * inv, O[i + e + 1] * inv, hl[e / 2], hl[8 + e / 2]);
                    tmem_st(sQ + lanes + HO * h + i, hl);
                }
                tmem_st_wait();
                tc_before();
            }
#pragma unroll
            for (int i = 0; i < HO; ++i) O[i] = 0.f;
            __syncthreads();
            tc_after();
            const uint64_t mk = rq < n_rows ? __ldg(tr.mask + sq_.r0 + (r_base + rq) / G) : 0;
            float m = -INFINITY, l = 0.f;              // m: what p is taken against, in log2 units
            // 8 bits: O is in units of 2^(m + a - (15 - LAG)); 2^a is above every v scale so far, and l's units are
            // the same; once `wide`, a is the row's own and l's units are 2^(m - (15 - LAG))
            float a = -80.f;
            uint32_t vlow = 0u - 0x7f7fffffu;          // 0 - the bits of the smallest v scale so far
            bool wide = false;
            bool ok = true;
            const auto scales = [&](int j) { return ssc + (tb + j) % SCB * (2 * KT) + toff(); };
            const auto s_part = [&](int j) { return sS((tb + j) & 1) + lanes + toff(); };
            const auto first_token = [&](int j) { return tok0 + j * KT + toff(); };
            const auto wait_s = [&](int j) {
                ok = ok && __all_sync(FULL, bar_wait(&bars.sfull[(tb + j) & 1], phase2(tb + j), fail));
                tc_after();
            };
            // The product of tile j is done.  Not waited for every tile: its barrier (of the tile's parity)
            // is at most one phase ahead, since the tile after next needs this thread's p.
            const auto wait_d = [&](int j) {
                ok = ok && __all_sync(FULL, bar_wait(&bars.dfull[(tb + j) & 1], phase2(tb + j), fail));
                tc_after();
            };
            // 2^exponent is above |x|, and 2^(exponent - 1) not (0: -126, infinity and NaN: 129)
            const auto exponent = [](float x) { return (int)(__float_as_uint(x) >> 23 & 255) - 126; };
            // every row sees every token of the thread's part of tile j
            const auto seen_by_all = [&](int j) {
                const uint8_t* gone = &gone_s[(tb + j) % SCB][toff() / 16];
                return (SPLIT ? *(const uint16_t*)gone : *(const uint32_t*)gone) == 0 && first_token(j) + TQ <= sq_.ctx;
            };
            // which of the part's 32 tokens from t the row sees
            const auto seen = [&](int j, int t) {
                const uint8_t* gone = &gone_s[(tb + j) % SCB][toff() / 16 + t / 16];
                uint32_t v = 0xffffffffu;
                if (gone[0]) v &= 0xffff0000u;
                if (gone[1]) v &= 0x0000ffffu;
                const int x = first_token(j) + t - sq_.ctx;            // < 0: tokens of the context first
                if (x + 32 > 0) {
                    const uint64_t all = mk & (sq_.n == 64 ? ~0ull : (1ull << sq_.n) - 1);
                    v &= x >= 0 ? (x < 64 ? (uint32_t)(all >> x) : 0u) : (uint32_t)(all << -x) | ((1u << -x) - 1);
                }
                return v;
            };
            // the largest of 16 scores (8 bits: times the tokens' scales; top: of score + exponent of the v scale)
            const auto max16 = [&](auto all, const uint32_t (&x)[16], const float* ks, uint32_t v, float mx, float& top) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    float y[4] = {__uint_as_float(x[i]), __uint_as_float(x[i + 1]), __uint_as_float(x[i + 2]),
                                  __uint_as_float(x[i + 3])};
                    if (Q8) {
                        const float4 k4 = *(const float4*)(ks + i);
                        const float2 y0 = __fmul2_rn(make_float2(y[0], y[1]), make_float2(k4.x, k4.y));
                        const float2 y1 = __fmul2_rn(make_float2(y[2], y[3]), make_float2(k4.z, k4.w));
                        y[0] = y0.x, y[1] = y0.y, y[2] = y1.x, y[3] = y1.y;
                    }
                    if (!all.value)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!(v >> (i + e) & 1)) y[e] = -INFINITY;
                    if (Q8 && !all.value && wide) {
                        const float4 v4 = *(const float4*)(ks + KT + i);
                        const float vv[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaf(y[e], rs, (float)max(exponent(vv[e]), -80)));
                    }
                    mx = fmaxf(fmaxf(mx, fmaxf(y[0], y[1])), fmaxf(y[2], y[3]));
                }
                return mx;
            };
            // 16 scores to p, as 8 pairs' high halves and then their low halves
            const auto p16 = [&](auto all, const uint32_t (&x)[16], uint32_t (&pk)[16], const float* ks, uint32_t v,
                                 float2 rs2, float2 nb2, float2& sum, float2 pf, float2 vf) {
                float4 k4, v4;
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float2 y = make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                    if (Q8 && i % 4 == 0) {
                        k4 = *(const float4*)(ks + i);
                        v4 = *(const float4*)(ks + KT + i);
                    }
                    if (Q8) y = __fmul2_rn(y, i % 4 ? make_float2(k4.z, k4.w) : make_float2(k4.x, k4.y));
                    y = __ffma2_rn(y, rs2, nb2);
                    float2 p = make_float2(ex2(y.x), ex2(y.y));
                    if (!all.value) {
                        if (!(v >> i & 1)) p.x = 0.f;
                        if (!(v >> (i + 1) & 1)) p.y = 0.f;
                    }
                    sum = __fadd2_rn(sum, p);
                    if (Q8) {
                        float2 z = i % 4 ? make_float2(v4.z, v4.w) : make_float2(v4.x, v4.y);
                        if (!all.value) {
                            p = __fmul2_rn(p, pf);
                            z = __fmul2_rn(z, vf);
                        }
                        p = __fmul2_rn(p, z);
                        if (!all.value) {                              // 0 stays 0 whatever the scale
                            if (!(v >> i & 1)) p.x = 0.f;
                            if (!(v >> (i + 1) & 1)) p.y = 0.f;
                        }
                    }
                    split_f16(p.x, p.y, pk[i / 2], pk[8 + i / 2]);
                }
            };
            const auto tile_max = [&](auto all, int j, float& top) {
                float mx = -INFINITY;
#pragma unroll
                for (int cc = 0; cc < TQ / 16; ++cc) {
                    uint32_t x[16];
                    tmem_ld(s_part(j) + 16 * cc, x);
                    const uint32_t v = all.value ? 0xffffffffu : seen(j, 16 * cc & ~31) >> (16 * cc & 31);
                    tmem_ld_wait();
                    mx = max16(all, x, scales(j) + 16 * cc, v, mx, top);
                }
                return mx;
            };
            // p of tile j, written over the S that it came from, and its sum
            const auto tile_p = [&](auto all, int j) {
                const float base = (m == -INFINITY ? 0.f : m) - ((float)(15 - LAG) - (Q8 && !wide ? a : 0.f));
                // the row's own factor 2^-a: with p alone where it is above 1, else half with v's scale, so that
                // neither overflows
                const float f = Q8 && !all.value && wide ? ex2(a < 0.f ? -a : -0.5f * a) : 1.f;
                const float2 pf = make_float2(f, f), vf = a < 0.f ? make_float2(1.f, 1.f) : pf;
                const float2 rs2 = make_float2(rs, rs), nb2 = make_float2(-base, -base);
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
                for (int cc = 0; cc < TQ / 16; ++cc) {                 // 16 tokens: one step of the product
                    uint32_t x[16], pk[16];
                    tmem_ld(s_part(j) + 16 * cc, x);
                    const uint32_t v = all.value ? 0xffffffffu : seen(j, 16 * cc & ~31) >> (16 * cc & 31);
                    tmem_ld_wait();
                    p16(all, x, pk, scales(j) + 16 * cc, v, rs2, nb2, sum, pf, vf);
                    tmem_st(s_part(j) + 16 * cc, pk);
                }
                return sum.x + sum.y;
            };
            // the part's maximum of tile j for the row's other threads, and whether anything has to be
            // rescaled for it; a barrier
            const auto publish = [&](int j, float mx, float top, float high) {
                const uint32_t t = tb + j;
                if (ok && live) {
                    part_max[t & 1][h][r] = mx;
                    if (Q8 && wide) part_top[Q8 ? t & 1 : 0][h][Q8 ? r : 0] = top;
                    if (mx * rs > m + (float)LAG || (Q8 && (wide ? top > m + a + (float)LAG : high > a))) need_s[t & 3] = 1;
                }
                softmax_sync();
                if (tid == 0) {
                    need_s[(t + 2) & 3] = 0;
                    // (before the producers come to that tile, whose K follows the scores of tile t + 2)
                    if (Q8) vends_s[(t + 4) % SCB] = make_uint2(0, 0);
                }
            };
            const auto add_d = [&]() {                 // O += D
#pragma unroll
                for (int cc = 0; cc < HO / 16; ++cc) {
                    uint32_t d[16];
                    tmem_ld(sD + lanes + HO * h + 16 * cc, d);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; ++i) O[16 * cc + i] += __uint_as_float(d[i]);
                }
            };
            for (int j = 0; j < nt; ++j) {             // to the end even after a failed wait: the barriers count
                const uint32_t t = tb + j;
                wait_s(j);
                float high = a;
                if (Q8 && !wide) {                     // (alike in every thread)
                    const uint2 v = vends_s[t % SCB];
                    vlow = max(vlow, v.y);
                    high = fmaxf(a, (float)((int)(v.x >> 23) - 126));
                    if (high > (float)TALL || high - (float)(int)((0u - vlow) >> 23) > (float)(SPAN - 126)) {
                        wide = true;
                        l *= ex2(a);
                    }
                }
                const bool all = seen_by_all(j) && !wide;
                float mx = -INFINITY, top = -INFINITY;
                if (ok && live) mx = all ? tile_max(Yes{}, j, top) : tile_max(No{}, j, top);
                publish(j, mx, top, high);
                const bool need = need_s[t & 3];
                if (j > 0 && (need || j % RUN == 0)) {
                    wait_d(j - 1);
                    if (ok && live) add_d();
                }
                if (need && ok && live) {
                    mx = fmaxf(part_max[t & 1][0][r], part_max[t & 1][1][r]);
                    const float mn = fmaxf(m, mx == -INFINITY ? -INFINITY : mx * rs);
                    float corr = mn == -INFINITY ? 1.f : ex2(m - mn);
                    const float before = m;
                    m = mn;
                    if (Q8 && wide) {
                        l *= corr;
                        top = fmaxf(part_top[Q8 ? t & 1 : 0][0][Q8 ? r : 0], part_top[Q8 ? t & 1 : 0][1][Q8 ? r : 0]);
                        if (mn != -INFINITY) {
                            top = fmaxf(before + a, top);
                            corr = ex2(before + a - top);
                            a = top - mn;
                        }
                    } else {
                        if (Q8) {
                            corr *= ex2(a - high);
                            a = high;
                        }
                        l *= corr;
                    }
#pragma unroll
                    for (int i = 0; i < HO; ++i) O[i] *= corr;
                }
                if (SPLIT && ok && live) {             // nothing of the other lane's tokens
                    const uint32_t zero[16] = {};
                    const uint32_t other = sS(t & 1) + lanes + (toff() ^ 64);
                    tmem_st(other, zero);
                    tmem_st(other + 16, zero);
                }
                if (ok && live) {
                    l += all ? tile_p(Yes{}, j) : tile_p(No{}, j);
                    tmem_st_wait();
                }
                tc_before();
                bar_arrive(&bars.pfull[t & 1]);
            }
            wait_d(nt - 1);
            if (ok && live) {
                add_d();
                // f16: infinities and NaN were taken out of the v that only some rows see (the last 64
                // tokens at most); a row that sees one becomes NaN, to be computed by the formula
                if (!Q8)
                    for (int j = max(nt - 2, 0); j < nt; ++j) {
                        const int x0 = tok0 + j * KT - sq_.ctx;
                        if (x0 + KT <= 0) continue;
                        for (int w = 0; w < 8; ++w) {
                            const int x = x0 + 16 * w;                 // 16 tokens from node x
                            if (SPLIT && (w >> 2) != (r >> 6)) continue;       // the other lane's tokens
                            if (x > -16 && x < sq_.n && (odd_s[(tb + j) % SCB][w] & (uint32_t)(x >= 0 ? mk >> x : mk << -x))) l = NAN;
                        }
                    }
            }
            tb += nt;
            if (Q8 && wide) {                          // l in O's units again
                const float f = ex2(-0.5f * a);
                l = l * f * f;
            }
            if (live) part_max[0][h][r] = l;
            __syncthreads();                           // every product is done: q and the scales are free
            bool nan = false;
            if constexpr (SPLIT) {
                const float bad = *fail ? NAN : 0.f;   // a wait ran out: no number may pass for a result
                if (rq < n_rows) {
                    // l and o carry the same power of two; that of another part may differ
                    if (h == 0) part_max[1][0][r] = Q8 ? m + a : m;
                    else part_max[1][1][r] = part_max[0][0][r] + part_max[0][1][r] + bad;
                    float* x = (float*)(skv + S::STAGE) + r * (HD + 1) + HO * h;
#pragma unroll
                    for (int i = 0; i < HO; ++i) x[i] = O[i] + bad;
                }
                softmax_sync();
                for (int i = warp; i < n_rows; i += NSW) {             // a row at a time, its two lanes joined
                    const int rr = r_base + i;
                    float* o = sg.whole ? out + (size_t)(sq_.r0 + rr / G) * ld_out + (size_t)(kvh * G + rr % G) * HD
                                        : ws + ((size_t)(2 * blockIdx.x + (sg.seg ? 1 : 0)) * MR + i) * (HD + 2) + 2;
                    const float* x = (const float*)(skv + S::STAGE) + i * (HD + 1) + lane;
                    const float ma = part_max[1][0][i], mb = part_max[1][0][i + 64], M = fmaxf(ma, mb);
                    float fa = ma == -INFINITY ? 1.f : ex2(ma - M), fb = mb == -INFINITY ? 1.f : ex2(mb - M);
                    const float L = fmaf(part_max[1][1][i], fa, part_max[1][1][i + 64] * fb);
                    if (sg.whole) {
                        const float inv = L == 0.f ? 0.f : 1.f / L;
                        fa *= inv;
                        fb *= inv;
                    } else if (lane == 0) {
                        o[-2] = M;
                        o[-1] = L;
                    }
#pragma unroll
                    for (int k = 0; k < HD / 32; ++k) {
                        const float y = fmaf(x[32 * k], fa, x[64 * (HD + 1) + 32 * k] * fb);
                        o[lane + 32 * k] = y;
                        nan |= y != y;
                    }
                }
            } else {
                if (r < n_rows) {
                    float L = part_max[0][0][r];
#pragma unroll
                    for (int i = 1; i < PARTS; ++i) L += part_max[0][i][r];
                    const float bad = *fail ? NAN : 0.f;
                    if (!sg.whole && h == 0) {
                        float* o = ws + ((size_t)(2 * blockIdx.x + (sg.seg ? 1 : 0)) * MR + r) * (HD + 2);
                        o[0] = Q8 ? m + a : m;
                        o[1] = L + bad;
                    }
                    const float f = (sg.whole ? (L == 0.f ? 0.f : 1.f / L) : 1.f);
                    float* x = (float*)(skv + S::STAGE) + r * (HD + 1) + HO * h;
#pragma unroll
                    for (int i = 0; i < HO; ++i) x[i] = O[i] * f + bad;
                }
                softmax_sync();
                for (int i = warp; i < n_rows; i += NSW) {             // through the tiles again, a row at a time
                    const int rr = r_base + i;
                    float* o = sg.whole ? out + (size_t)(sq_.r0 + rr / G) * ld_out + (size_t)(kvh * G + rr % G) * HD
                                        : ws + ((size_t)(2 * blockIdx.x + (sg.seg ? 1 : 0)) * MR + i) * (HD + 2) + 2;
#pragma unroll
                    for (int k = 0; k < HD / 32; ++k) {
                        const float y = ((const float*)(skv + S::STAGE))[i * (HD + 1) + lane + 32 * k];
                        o[lane + 32 * k] = y;
                        nan |= y != y;
                    }
                }
            }
            if (nan) nan_words(ws, HD)[blockIdx.x] = 1;
            if (*fail) break;
        }
    } else {
    // (256 x 144 + 256 x 112 registers are the 512 x 128 that the block starts with)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    if (warp == NSW + NPW) {
        // ================= products: f32 accumulate, M = 128, N = 128 (scores) or HD (p v);
        // V is MN-major (bit 16)
        constexpr uint32_t idq = 1u << 4 | (uint32_t)(KT >> 3) << 17 | (uint32_t)(MR >> 4) << 24;
        constexpr uint32_t idv = 1u << 4 | 1u << 16 | (uint32_t)(HD >> 3) << 17 | (uint32_t)(MR >> 4) << 24;
        while (next_segment()) {
            __syncthreads();
            if (lane == 0) {
                bool ok = true;
                const auto pv = [&](uint32_t t) {
                    const int b = t & 1, vb_ = t % NB;
                    ok = ok && bar_wait(&bars.vfull[vb_], phaseN(t), fail) && bar_wait(&bars.pfull[b], phase2(t), fail);
                    if (!ok) return;
                    // D begins anew where the softmax has added it to O
                    const bool anew = need_s[t & 3] || (t - tb) % RUN == 0;
                    fence_async();
                    tc_after();
                    const uint32_t vb = su32(skv) + (NB + vb_) * S::TB;
#pragma unroll
                    for (int k = 0; k < KT / 16; ++k) {
                        const uint64_t bd = desc(vb + 2048 * k, 16384);
                        mma_ts(sD, sS(b) + 16 * k + 8, bd, idv, k > 0 || !anew);
                        mma_ts(sD, sS(b) + 16 * k, bd, idv, 1);
                    }
                    commit(&bars.vfree[vb_]);
                    commit(&bars.dfull[b]);
                };
                const uint32_t nt = sg.nt;
                for (uint32_t t = tb; t < tb + nt && ok; ++t) {
                    const int b = t & 1, kb_ = t % NB;
                    ok = bar_wait(&bars.kfull[kb_], phaseN(t), fail);
                    if (!ok) break;
                    // K was written through the generic proxy and is read through the async one.  The
                    // fence stands here, behind the barrier: in the producers it would wait for the loads
                    // that they keep in flight.
                    fence_async();
                    tc_after();
                    const uint32_t kb = su32(skv) + kb_ * S::TB;
#pragma unroll
                    for (int h = 1; h >= 0; --h)       // lo first: the small products enter a small sum
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            const uint32_t o = (uint32_t)(k >> 2) * 16384 + 32 * (k & 3);
                            mma_ts(sS(b), sQ + 16 * k + 8 * h, desc(kb + o, 16), idq, h == 0 || k > 0);
                        }
                    commit(&bars.kfree[kb_]);
                    commit(&bars.sfull[b]);
                    if (t > tb) pv(t - 1);
                }
                if (ok) pv(tb + nt - 1);
                tb += nt;
            }
            __syncwarp();
            __syncthreads();
            if (*fail) break;
        }
    } else {
        // ================= K and V: job n is page n % 8 of K (n / 8 even) or V of tile n / 16;
        // warp 8 + w takes jobs w, w + 7, ...
        const int w = warp - NSW;
        while (next_segment()) {
            const int nt = sg.nt, kvh = sg.kvh, tok0 = sg.tok0, end = sg.end, ctx = sg.sq.ctx, slot = sg.sq.slot;
            if (!Q8 && tb) __syncthreads();
            bool ok = true;
            const int njobs = 16 * nt;
            const size_t kv_step = (size_t)nkv * sb_kv_block_bytes(KV, HD), page_step = 2 * kv_step;
            const unsigned char* pool = sb_kv_block(c, layer, 0, 0, kvh);
            const int32_t* pages = c.page_table + (size_t)max(slot, 0) * c.max_pages;
            const int n_pages = (int)c.n_pages, last = slot >= 0 && slot < c.n_slots ? min(c.max_pages, (end + 15) / 16) : 0;
            const auto page_of = [&](int n) {
                const int i = (tok0 + (n >> 4) * KT) / 16 + (n & 7);
                const int p = n < njobs && i < last ? __ldg(pages + i) : -1;
                return p < n_pages ? p : -1;
            };
            // the operand buffer is free once the product NB tiles back has read it
            const auto wait_free = [&](int n) {
                const uint32_t t = tb + (n >> 4);
                if (ok && t >= NB)
                    ok = __all_sync(FULL, bar_wait(n & 8 ? &bars.vfree[t % NB] : &bars.kfree[t % NB], phaseN(t - NB), fail));
            };
            const auto arrive = [&](int n) {           // the proxy fence is the product warp's
                __syncwarp();
                const uint32_t b = (tb + (n >> 4)) % NB;
                if (lane == 0) bar_arrive(n & 8 ? &bars.vfull[b] : &bars.kfull[b]);
            };
            if constexpr (Q8) {
                // Lane: 16 dims k of token t (and every TS-th after it), widened to chunks 2 k and 2 k + 1.
                // Eight lanes in turn hold four k of two tokens: their chunks differ by the tokens' low
                // bit, so that a store meets no bank twice.
                constexpr int U = HD / 16, TS = 32 / U, NP = 16 / TS;
                const int lt = lane / 4 % TS, lk = lane % 4 + 4 * (lane / 4 / TS);
                const uint32_t to[2] = {op_at(lt, 2 * lk), op_at(lt + TS, 2 * lk) - TS * 128};
                struct Raw {
                    uint4 x[NP];
                    int page, next;                    // of the set's next job: its address is known in time
                };
                const auto fetch = [&](Raw& r, int n) {
                    const int page = r.page = r.next;
                    r.next = page_of(n + 2 * NPW);
                    const unsigned char* blk = pool + max(page, 0) * page_step + ((n & 8) ? kv_step : 0);
#pragma unroll
                    for (int i = 0; i < NP; ++i)
                        r.x[i] = page < 0 ? make_uint4(0, 0, 0, 0)
                                          : __ldg((const uint4*)(blk + SB_Q8_SCALES) + (lt + TS * i) * U + lk);
                };
                const auto put = [&](const Raw& r, int n) {
                    float4 k4 = make_float4(0.f, 0.f, 0.f, 0.f), v4 = k4;      // both scales of 4 tokens
                    if (!(n & 8) && r.page >= 0 && lane < 4) {
                        const unsigned char* blk = pool + r.page * page_step;
                        k4 = __ldg((const float4*)blk + lane);
                        v4 = __ldg((const float4*)(blk + kv_step) + lane);
                    }
                    wait_free(n);
                    if (!ok) return;
                    const int j = n >> 4, pg = n & 7;
                    const uint32_t sc_ = (tb + j) % SCB;
                    unsigned char* dst = skv + (((n & 8) ? NB : 0) + (tb + j) % NB) * S::TB + pg * 2048;
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const uint4 v = r.x[i];
                        const uint4 a = make_uint4(i8_f16<0x4140>(v.x), i8_f16<0x4342>(v.x), i8_f16<0x4140>(v.y), i8_f16<0x4342>(v.y));
                        const uint4 z = make_uint4(i8_f16<0x4140>(v.z), i8_f16<0x4342>(v.z), i8_f16<0x4140>(v.w), i8_f16<0x4342>(v.w));
                        *(uint4*)(dst + to[i & 1] + TS * i * 128) = a;
                        *(uint4*)(dst + (to[i & 1] ^ 16) + TS * i * 128) = z;
                    }
                    if (!(n & 8)) {                    // before kfull: the softmax reads them after the scores
                        if (lane < 4) {
                            float* sc = ssc + sc_ * 2 * KT + 16 * pg + 4 * lane;
                            *(float4*)sc = make_float4(no_inf(k4.x), no_inf(k4.y), no_inf(k4.z), no_inf(k4.w));
                            *(float4*)(sc + KT) = v4;
                            uint32_t b[4] = {__float_as_uint(v4.x), __float_as_uint(v4.y), __float_as_uint(v4.z), __float_as_uint(v4.w)};
                            const int t = tok0 + j * KT + 16 * pg + 4 * lane;
                            if (t + 4 > ctx)           // what only some rows see, or none, and is no number: not looked at
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (t + i >= end || (t + i >= ctx && b[i] >= 0x7f800000u)) b[i] = 0;
                            atomicMax(&vends_s[sc_].x, max(max(b[0], b[1]), max(b[2], b[3])));
                            atomicMax(&vends_s[sc_].y, max(max(0u - b[0], 0u - b[1]), max(0u - b[2], 0u - b[3])));
                        }
                        if (lane == 0) {
                            gone_s[sc_][pg] = r.page < 0;
                        }
                    }
                    arrive(n);
                };
                // two pages in flight, in registers of their own: the wait for one is not a wait for
                // the other
                Raw a, z;
                a.next = page_of(w);
                z.next = page_of(w + NPW);
                fetch(a, w);
                fetch(z, w + NPW);
                __syncthreads();                       // q has left the tiles
                for (int n = w; n < njobs && ok; n += 2 * NPW) {
                    put(a, n);
                    fetch(a, n + 2 * NPW);
                    if (n + NPW < njobs) put(z, n + NPW);
                    fetch(z, n + 3 * NPW);
                }
            } else {
                constexpr int CPT = HD / 8, TS = 32 / CPT, NP = 16 / TS;       // chunks a token; tokens a step
                constexpr int DEPTH = 2;
                const auto land = [&](int n) {         // job n has arrived
                    const int j = n >> 4, pg = n & 7, t0 = tok0 + j * KT + 16 * pg;
                    if ((n & 8) && tok0 + j * KT + KT > ctx) {
                        // v that only some rows see: its infinities and NaN leave the tile
                        uint32_t odd = 0;
                        unsigned char* dst = skv + (NB + (tb + j) % NB) * S::TB + pg * 2048;
                        for (int i = 0; i < NP; ++i) {
                            const int t = lane / CPT + TS * i;
                            if (t0 + t < ctx) continue;
                            uint32_t* v = (uint32_t*)(dst + op_at(t, lane % CPT));
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t x = v[k];
                                uint32_t keep = 0xffffffffu;
                                if ((x & 0x7c00u) == 0x7c00u) keep &= 0xffff0000u;
                                if ((x & 0x7c000000u) == 0x7c000000u) keep &= 0x0000ffffu;
                                if (keep != 0xffffffffu) {
                                    v[k] = x & keep;
                                    odd |= 1u << t;
                                }
                            }
                        }
                        odd = __reduce_or_sync(FULL, odd);
                        if (lane == 0) odd_s[(tb + j) % SCB][pg] = (uint16_t)odd;
                    }
                    arrive(n);
                };
                // Lane i holds the page of the warp's job i, of 32 jobs and the 32 after them: no job waits
                // for its page's number.
                const auto pages_of = [&](int first) { return page_of(w + NPW * (first + lane)); };
                int window = pages_of(0), window2 = pages_of(32), job = 0;
                bool q_gone = tb > 0;
                for (int n = w; n < njobs && ok; n += NPW, ++job) {
                    const int j = n >> 4, pg = n & 7, t0 = tok0 + j * KT + 16 * pg;
                    if (job && (job & 31) == 0) {
                        window = window2;
                        window2 = pages_of(job + 32);
                    }
                    const int page = __shfl_sync(FULL, window, job & 31);
                    if (!q_gone && n >= 15) {
                        q_gone = true;
                        __syncthreads();
                    }
                    wait_free(n);
                    if (!ok) break;
                    const uint32_t dst = su32(skv) + (((n & 8) ? NB : 0) + (tb + j) % NB) * S::TB + pg * 2048;
                    const unsigned char* src = pool + max(page, 0) * page_step + ((n & 8) ? kv_step : 0) + 16 * lane;
#pragma unroll
                    for (int i = 0; i < NP; ++i)
                        cp16(dst + op_at(lane / CPT + TS * i, lane % CPT), src + 512 * i,
                             page >= 0 && t0 + lane / CPT + TS * i < end);
                    if (lane == 0 && !(n & 8)) gone_s[(tb + j) % SCB][pg] = page < 0;
                    cp_commit();
                    // DEPTH jobs stay in flight; what a job waits for lies at least 33 jobs back, so the
                    // ones still to land cannot be in its way
                    if (n >= DEPTH * NPW) {
                        cp_wait<DEPTH>();
                        land(n - DEPTH * NPW);
                    }
                }
                if (!q_gone) __syncthreads();
                const int mine = (njobs - w + NPW - 1) / NPW;      // the last of the warp's jobs
                cp_wait<0>();
                for (int i = max(mine - DEPTH, 0); i < mine && ok; ++i) land(w + i * NPW);
            }
            tb += nt;
            __syncthreads();
            if (*fail) break;
        }
    }
    }
    __syncthreads();
    if (*fail) {
        // products and copies in flight end before the CTA does; then, what this CTA owed and
        // did not do: NaN, whole or in part, which attn_tree_join has computed by the formula
        if (tid == 0) nan_words(ws, HD)[blockIdx.x] = 1;
        for (const uint64_t t0 = gtimer(); gtimer() - t0 < WAIT_NS / 100;) {}
        while (next_segment()) {
            for (int e = tid; e < sg.n_rows * (HD + 2); e += NTHREADS) {
                const int r = e / (HD + 2), d = e % (HD + 2), row = sg.r_base + r;
                if (!sg.whole) ws[((size_t)(2 * blockIdx.x + 1) * MR + r) * (HD + 2) + d] = NAN;
                else if (d < HD) out[(size_t)(sg.sq.r0 + row / G) * ld_out + (size_t)(sg.kvh * G + row % G) * HD + d] = NAN;
            }
        }
    }
    if (warp == NSW + NPW) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int KV, int HD, bool SPLIT>
int launch(const slate_kv_cache_t& c, int layer, const slate_tree_t& tr, int nq, float* out, int ld_out,
           const float* q, int ld_q, float scale, float* ws, cudaStream_t st) {
    const auto k = attn_tree_tc<KV, HD, SPLIT>;
    static unsigned long long ready = 0;
    const cudaError_t may = sb_allow_smem((const void*)k, TcShape<KV, HD>::SMEM, &ready);
    if (may != cudaSuccess) return sb_cuda_check(may, "attention_tree shared memory");
    return sb_cuda_check(sb_launch_pdl(k, dim3(SMS), dim3(NTHREADS), TcShape<KV, HD>::SMEM, st, c, layer, tr, nq,
                                       out, ld_out, q, ld_q, scale, ws),
                         "attention_tree");
}

}  // namespace

int sb_tree::attend_tc(const slate_kv_cache_t& c, int layer, const slate_tree_t& tr, int nq, float* out, int ld_out,
                       const float* q, int ld_q, float scale, float* ws, cudaStream_t st) {
    const auto by_rows = [&](auto kv, auto hd) {
        constexpr int KV = decltype(kv)::value, HD = decltype(hd)::value;
        return tr.max_nodes * (nq / c.n_kv_heads) <= 64 ? launch<KV, HD, true> : launch<KV, HD, false>;
    };
    const auto by_hd = [&](auto kv) {
        return c.head_dim == 64 ? by_rows(kv, std::integral_constant<int, 64>{}) : by_rows(kv, std::integral_constant<int, 128>{});
    };
    const auto f = c.kv_dtype == SLATE_KV_F16 ? by_hd(std::integral_constant<int, SLATE_KV_F16>{})
                                              : by_hd(std::integral_constant<int, SLATE_KV_Q8>{});
    return f(c, layer, tr, nq, out, ld_out, q, ld_q, scale, ws, st);
}
