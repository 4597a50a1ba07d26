// attn_tree_tc.cu -- tree attention for many rows on the tcgen05 tensor cores
// (f16 and 8-bit caches, head_dim 64 and 128; attn_tree.cu has the formula, the
// split of f32 values into f16 pairs and the few-row kernels).
//
// One CTA an SM.  A tile of 128 rows (nodes x group) stays: q as f16 hi and lo in
// shared memory.  The cache streams past in tiles of 128 tokens:
//   S = Qhi K^T + Qlo K^T           128 x 128, in tensor memory, f32
//   P = exp(S - max), hi and lo     written over S, the next product's A operand
//   D = Phi V + Plo V               128 x head_dim, in tensor memory
//   O = O corr + D                  in registers, one FMA an element
// S and D have two buffers each: while the softmax warps work on tile j, the tensor cores
// run P V of tile j - 1 and Q K^T of tile j + 1.  D is drained every tile because an
// accumulator carried over a long context in the tensor cores would truncate at every step.
// Warps 0-3, 4-7: softmax of a tile's first and second 64 tokens, a thread a row (the two
// exchange the row's maximum), and the first and second half of O's dims.  Warps 8-14 bring
// K and V page by page in turn into the operands' swizzled layout (f16: 16-byte asynchronous
// copies; 8 bits: through registers, two pages ahead, widened to f16 on the way).  Warp 15
// issues the products.
// What bounds it: the tensor cores, 2 x the plain formula's products for the two
// halves, from 64 rows up; the exponentials and splits take nearly as many issue slots.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "sb_internal.h"
#include "sb_kernels.h"
#include "sb_kv.h"
#include "sb_pdl.h"
#include "sb_tree.h"

using namespace sb_tree;

namespace {

constexpr int MR = 128, KT = 128, NTHREADS = 512, NPW = 7;
constexpr uint64_t WAIT_NS = 2000000000ull;
constexpr int SCB = 4;                        // tiles whose scales and flags are kept

template <int KV, int HD>
struct TcShape {
    static constexpr int QB = MR * HD * 2;                 // one half of q
    static constexpr int TB = KT * HD * 2;                 // a K or V tile in f16
    static constexpr int SC = SCB * 2 * KT * 4;
    static constexpr int SMEM = 2 * QB + 4 * TB + SC + 1024;
};

struct Yes {
    static constexpr bool value = true;
};
struct No {
    static constexpr bool value = false;
};

struct Bars {
    uint64_t kfull[2], kfree[2], vfull[2], vfree[2], sfull[2], pfull[2], dfull[2];
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
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(acc));
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
// 32 or 16 columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_ld(uint32_t a, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), 
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), 
                 "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), 
                 "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), 
                 "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(a));
}
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
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// Byte of 16-byte chunk ch (8 f16) of row r in an operand of 128 rows: 64 columns a
// 16 KB block, rows of 128 bytes, chunks exchanged by the row's low bits.
__device__ __forceinline__ uint32_t op_at(int r, int ch) {
    return (uint32_t)((ch >> 3) * 16384 + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
}

// The CTA's segments: each a run of tiles of one item.  In shared memory, advanced by one
// thread: the roles have no registers to spare for it.
struct Segs {
    int64_t at, stop, seq_before;
    int s, seg;
    Seq sq;
    int u0, nt, kvh, r_base, n_rows, end, tok0;
    bool whole;
    __device__ __forceinline__ bool next(const slate_kv_cache_t& c, const slate_tree_t& tr, int G) {
        if (at >= stop) return false;
        while (at >= seq_before + seq_units(sq, c.n_kv_heads)) {
            seq_before += seq_units(sq, c.n_kv_heads);
            sq = seq_of(c, tr, ++s, G, MR, KT);
        }
        const uint32_t rel = (uint32_t)(at - seq_before);
        const int item = (int)(rel / (uint32_t)sq.units);
        u0 = (int)(rel % (uint32_t)sq.units);
        nt = (int)min((int64_t)sq.units, u0 + (stop - at)) - u0;
        kvh = item / sq.tiles;
        r_base = (item % sq.tiles) * MR;
        n_rows = min(MR, sq.n * G - r_base);
        end = sq.ctx + sq.n;
        tok0 = u0 * KT;
        whole = nt == sq.units;
        at += nt;
        ++seg;
        return true;
    }
};

template <int KV, int HD>
__global__ void __launch_bounds__(NTHREADS, 1) attn_tree_tc(
    const slate_kv_cache_t c, int layer, const slate_tree_t tr, int nq, float* __restrict__ out,
    int ld_out, const float* __restrict__ q, int ld_q, float scale, float* __restrict__ ws) {
    using S = TcShape<KV, HD>;
    constexpr bool Q8 = KV == SLATE_KV_Q8;
    constexpr int KS = HD / 16;
    extern __shared__ unsigned char smem_raw[];
    // by an offset, so that the compiler still knows it for shared memory
    unsigned char* smem = smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u);
    unsigned char* sq = smem;                                   // [hi, lo]
    unsigned char* skv = sq + 2 * S::QB;                        // [K0, K1, V0, V1]
    float* ssc = (float*)(skv + 4 * S::TB);                      // [SCB][K, V][KT]
    __shared__ Bars bars;
    __shared__ Segs sg;
    __shared__ int more_s;
    __shared__ PlanBuf buf;
    __shared__ uint32_t tmem_s;
    __shared__ __align__(8) uint8_t gone_s[SCB][8];                // per page: the table has none
    __shared__ uint16_t odd_s[SCB][8];                             // per page: tokens whose v is not finite
    __shared__ __align__(16) float vmax_s[SCB][8];                 // per page: largest v scale
    __shared__ float rowscale[MR], half_max[2][2][MR];          // [tile parity][half][row]
    __shared__ int fail_s;
    sb_grid_release();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nkv = c.n_kv_heads, G = nq / nkv;
    int64_t before;
    const int64_t total = plan_total(c, tr, G, MR, KT, buf, before);
    const Cut cut(total, gridDim.x);
    if ((int)blockIdx.x >= cut.C) return;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&bars.kfull[i], 8);          // pages
            bar_init(&bars.vfull[i], 8);
            bar_init(&bars.kfree[i], 1);
            bar_init(&bars.vfree[i], 1);
            bar_init(&bars.sfull[i], 1);
            bar_init(&bars.pfull[i], 256);
            bar_init(&bars.dfull[i], 1);
        }
        fail_s = 0;
        sg.at = cut.first(blockIdx.x);
        sg.stop = cut.first(blockIdx.x + 1);
        sg.seg = -1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&tmem_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_before();
    }
    int64_t seq_before;
    const int s0 = plan_find(c, tr, G, MR, KT, buf, before, cut.first(blockIdx.x), seq_before);     // a barrier
    tc_after();
    const uint32_t tmem = tmem_s;
    if (tid == 0) {
        sg.s = s0;
        sg.seq_before = seq_before;
        sg.sq = seq_of(c, tr, s0, G, MR, KT);
    }
    // Every role walks the same segments; four barriers of the CTA a segment: the last one has
    // left the buffers, the next is known, q is there, every product is done and the half rows'
    // sums are there.
    const auto next_segment = [&]() {
        __syncthreads();
        if (tid == 0) more_s = sg.next(c, tr, G);
        __syncthreads();
        return more_s != 0;
    };
    const auto sS = [&](int b) { return tmem + 128u * b; };
    const auto sD = [&](int b) { return tmem + 256u + 128u * b; };
    uint32_t nuse[2] = {0, 0};                  // tiles done in each buffer by this role: barrier phases
    volatile int* fail = &fail_s;

    if (warp < 8) {
        // no spills: with 227 KB of shared memory the first-level cache is too small to hold them
        asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        while (next_segment()) {
            const Seq& sq_ = sg.sq;
            const int nt = sg.nt, kvh = sg.kvh, r_base = sg.r_base, n_rows = sg.n_rows, tok0 = sg.tok0;
        // ---- q, each row divided by the power of two below its maximum; scale's sign joins q
        for (int r = warp; r < MR; r += 8) {
            const int row = r_base + r;
            const bool live = r < n_rows;
            const float* x = q + (size_t)(sq_.r0 + (live ? row / G : 0)) * ld_q +
                             (size_t)(kvh * G + (live ? row % G : 0)) * HD;
            constexpr int E = HD / 32;
            float v[E];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                v[i] = live ? x[lane * E + i] : 0.f;
                top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
            }
            top = __reduce_max_sync(FULL, top);
            const int e = min(max((int)(top >> 23) - 127, -100), 100);
            const float inv = copysignf(__int_as_float((127 - e) << 23), scale);
            if (lane == 0) rowscale[r] = fabsf(scale) * 1.4426950408889634f * __int_as_float((127 + e) << 23);
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                uint32_t hi, lo;
                split_f16(v[i] * inv, v[i + 1] * inv, hi, lo);
                const int d = lane * E + i;
                const uint32_t o = op_at(r, d / 8) + 2 * (d & 7);
                *(uint32_t*)(sq + o) = hi;
                *(uint32_t*)(sq + S::QB + o) = lo;
            }
        }
        fence_async();
        __syncthreads();
            // ================= softmax: thread = row, half h of the tile's tokens and of O's dims
            constexpr int HO = HD / 2;
            const int h = warp >> 2, r = tid & 127;
            const bool live = (warp & 3) * 32 < n_rows;                 // of the warp
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            const float rs = rowscale[r];
            const uint64_t mk = r < n_rows ? __ldg(tr.mask + sq_.r0 + (r_base + r) / G) : 0;
            float m = -INFINITY, l = 0.f, corr = 0.f;
            int vexp = -80, vlast = -80;
            float O[HO];
#pragma unroll
            for (int i = 0; i < HO; ++i) O[i] = 0.f;
            bool ok = true;
            // O = O corr + D of tile j (its buffer's last one)
            const auto drain = [&](int j) {
                const int b = j & 1;
                ok = ok && __all_sync(FULL, bar_wait(&bars.dfull[b], (nuse[b] - 1) & 1, fail));
                if (!ok || !live) return;
                tc_after();
                const float2 c2 = make_float2(corr, corr);
#pragma unroll
                for (int cc = 0; cc < HO / 32; ++cc) {
                    uint32_t d[32];
                    tmem_ld(sD(b) + lanes + HO * h + 32 * cc, d);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 x = __ffma2_rn(make_float2(O[32 * cc + i], O[32 * cc + i + 1]), c2,
                                                    make_float2(__uint_as_float(d[i]), __uint_as_float(d[i + 1])));
                        O[32 * cc + i] = x.x;
                        O[32 * cc + i + 1] = x.y;
                    }
                }
                // f16: infinities and NaN were taken out of the v that only some rows see; the
                // rows that see them get them here
                const int t0 = tok0 + j * KT;
                if (!Q8 && t0 + KT > sq_.ctx) {
                    for (int w = 0; w < 8; ++w)
                        for (uint32_t rest = odd_s[j % SCB][w]; rest; rest &= rest - 1) {
                            const int t = t0 + 16 * w + __ffs(rest) - 1, x = t - sq_.ctx;
                            const int page = sb_kv_page(c, sq_.slot, t);
                            if (page < 0 || x < 0 || x >= sq_.n || !(mk >> x & 1)) continue;
                            const __half* v = (const __half*)sb_kv_block(c, layer, page, 1, kvh) + (t & 15) * HD + HO * h;
#pragma unroll
                            for (int i = 0; i < HO; ++i) {
                                const float y = __half2float(v[i]);
                                if (!(fabsf(y) < INFINITY)) O[i] += y;
                            }
                        }
                }
            };
            for (int j = 0; j < nt; ++j) {             // to the end even after a failed wait: the barriers count
                const int b = j & 1;
                ok = ok && __all_sync(FULL, bar_wait(&bars.sfull[b], nuse[b] & 1, fail));
                tc_after();
                const bool work = ok && live;
                const float* ks = ssc + (j % SCB) * 2 * KT + 64 * h;
                const float* vs = ks + KT;
                const int t0 = tok0 + j * KT + 64 * h;                 // the half's first token
                const uint32_t gone4 = *(const uint32_t*)&gone_s[j % SCB][4 * h];    // a byte a page
                const uint32_t sp = sS(b) + lanes + 64 * h;
                // which of the half's 32 tokens from t the row sees
                const auto seen = [&](int t) {
                    uint32_t v = 0xffffffffu;
                    if (gone4 >> (t / 2) & 1) v &= 0xffff0000u;
                    if (gone4 >> (t / 2 + 8) & 1) v &= 0x0000ffffu;
                    const int x = t0 + t - sq_.ctx;                    // < 0: tokens of the context first
                    if (x + 32 > 0) {
                        const uint64_t all = mk & (sq_.n == 64 ? ~0ull : (1ull << sq_.n) - 1);
                        v &= x >= 0 ? (x < 64 ? (uint32_t)(all >> x) : 0u) : (uint32_t)(all << -x) | ((1u << -x) - 1);
                    }
                    return v;
                };
                // Two passes over the half of S, 32 tokens at a time: the maximum; then p, its halves
                // written over the S that they came from.  `all`: every row sees every token.
                const auto tile_max = [&](auto all) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int cc = 0; cc < 2; ++cc) {
                        uint32_t x[32];
                        tmem_ld(sp + 32 * cc, x);
                        const uint32_t v = all.value ? 0xffffffffu : seen(32 * cc);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            float y[4] = {__uint_as_float(x[i]), __uint_as_float(x[i + 1]), __uint_as_float(x[i + 2]),
                                          __uint_as_float(x[i + 3])};
                            if (Q8) {
                                const float4 k4 = *(const float4*)(ks + 32 * cc + i);
                                const float2 y0 = __fmul2_rn(make_float2(y[0], y[1]), make_float2(k4.x, k4.y));
                                const float2 y1 = __fmul2_rn(make_float2(y[2], y[3]), make_float2(k4.z, k4.w));
                                y[0] = y0.x, y[1] = y0.y, y[2] = y1.x, y[3] = y1.y;
                            }
                            if (!all.value)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (!(v >> (i + e) & 1)) y[e] = -INFINITY;
                            mx = fmaxf(fmaxf(mx, fmaxf(y[0], y[1])), fmaxf(y[2], y[3]));
                        }
                    }
                    return mx;
                };
                const auto tile_p = [&](auto all, float base) {
                    float2 sum = make_float2(0.f, 0.f);
                    const float2 rs2 = make_float2(rs, rs), nb2 = make_float2(-base, -base);
#pragma unroll 1
                    for (int cc = 0; cc < 4; ++cc) {                   // 16 tokens: one step of the product
                        uint32_t x[16], pk[16];                        // pk: hi of 8 pairs, then lo
                        tmem_ld(sp + 16 * cc, x);
                        const uint32_t v = all.value ? 0xffffffffu : seen(16 * cc & ~31) >> (16 * cc & 31);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float2 y = make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                            if (Q8) y = __fmul2_rn(y, *(const float2*)(ks + 16 * cc + i));
                            y = __ffma2_rn(y, rs2, nb2);
                            float2 p = make_float2(ex2(y.x), ex2(y.y));
                            if (!all.value) {
                                if (!(v >> i & 1)) p.x = 0.f;
                                if (!(v >> (i + 1) & 1)) p.y = 0.f;
                            }
                            sum = __fadd2_rn(sum, p);
                            if (Q8) {
                                p = __fmul2_rn(p, *(const float2*)(vs + 16 * cc + i));
                                if (!all.value) {                      // 0 stays 0 whatever the scale
                                    if (!(v >> i & 1)) p.x = 0.f;
                                    if (!(v >> (i + 1) & 1)) p.y = 0.f;
                                }
                            }
                            split_f16(p.x, p.y, pk[i / 2], pk[8 + i / 2]);
                        }
                        tmem_st(sp + 16 * cc, pk);
                    }
                    return sum.x + sum.y;
                };
                const bool all = !gone4 && t0 + 64 <= sq_.ctx;
                if (work) half_max[b][h][r] = all ? tile_max(Yes{}) : tile_max(No{});
                softmax_sync();
                float ncorr = 0.f;
                if (work) {
                    const float mx = fmaxf(half_max[b][0][r], half_max[b][1][r]);
                    // the row's scores in log2 units; f16: p carries 2^15 itself
                    const float top = mx == -INFINITY ? -INFINITY : mx * rs;
                    const float mn = fmaxf(m, top);
                    // p carries 2^up; 8 bits: 2^15 over a power of two above every v scale so far, so that
                    // p vscale keeps f16's range
                    int up = 15;
                    if (Q8) {
                        const float4 a = *(const float4*)vmax_s[j % SCB], z = *(const float4*)(vmax_s[j % SCB] + 4);
                        const float vm = fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(z.x, z.y), fmaxf(z.z, z.w)));
                        vexp = max(vexp, min(max((int)(__float_as_uint(vm) >> 23) - 126, -80), 126));
                        up -= vexp;
                    }
                    const float base = (mn == -INFINITY ? 0.f : mn) - (float)up;
                    ncorr = ex2(m - (mn == -INFINITY ? 0.f : mn));
                    m = mn;
                    const float ls = all ? tile_p(Yes{}, base) : tile_p(No{}, base);
                    if (Q8) ncorr *= ex2((float)(vlast - vexp));       // l and o carry 2^up alike
                    vlast = vexp;
                    l = fmaf(l, ncorr, ls);
                    tmem_st_wait();
                }
                tc_before();
                bar_arrive(&bars.pfull[b]);
                if (j > 0) drain(j - 1);
                corr = ncorr;
                ++nuse[b];
            }
            drain(nt - 1);
            if (live) half_max[0][h][r] = l;
            __syncthreads();                           // every product is done: q and the scales are free
            if (r < n_rows) {
                const float L = half_max[0][0][r] + half_max[0][1][r];
                const float bad = *fail ? NAN : 0.f;   // a wait ran out: no number may pass for a result
                const int row = r_base + r;
                float* o = sg.whole ? out + (size_t)(sq_.r0 + row / G) * ld_out + (size_t)(kvh * G + row % G) * HD + HO * h
                                    : ws + ((size_t)(2 * blockIdx.x + (sg.seg ? 1 : 0)) * MR + r) * (HD + 2) + 2 + HO * h;
                if (!sg.whole && h == 0) {
                    o[-2] = Q8 ? m + (float)vexp : m;  // 2^up of another part may differ
                    o[-1] = L + bad;
                }
                const float f = (sg.whole ? (L == 0.f ? 0.f : 1.f / L) : 1.f); // l and o carry the same power of two
#pragma unroll
                for (int i = 0; i < HO; i += 2) {
                    const float2 y = make_float2(O[i] * f + bad, O[i + 1] * f + bad);
                    if (sg.whole) {
                        o[i] = y.x;
                        o[i + 1] = y.y;
                    } else {
                        *(float2*)(o + i) = y;
                    }
                }
            }
            if (*fail) break;
        }
    } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 15) {
        // ================= products: f32 accumulate, M = 128, N = 128 (scores) or HD (p v);
        // V is MN-major (bit 16)
        constexpr uint32_t idq = 1u << 4 | (uint32_t)(KT >> 3) << 17 | (uint32_t)(MR >> 4) << 24;
        constexpr uint32_t idv = 1u << 4 | 1u << 16 | (uint32_t)(HD >> 3) << 17 | (uint32_t)(MR >> 4) << 24;
        while (next_segment()) {
            __syncthreads();
            if (lane == 0) {
                bool ok = true;
                uint32_t npv[2] = {nuse[0], nuse[1]};
                const auto pv = [&](int j) {
                    const int b = j & 1;
                    const uint32_t ph = npv[b]++ & 1;
                    ok = ok && bar_wait(&bars.vfull[b], ph, fail) && bar_wait(&bars.pfull[b], ph, fail);
                    if (!ok) return;
                    tc_after();
                    const uint32_t vb = su32(skv) + (2 + b) * S::TB;
#pragma unroll
                    for (int k = 0; k < KT / 16; ++k) {
                        const uint64_t bd = desc(vb + 2048 * k, 16384);
                        mma_ts(sD(b), sS(b) + 16 * k + 8, bd, idv, k > 0);
                        mma_ts(sD(b), sS(b) + 16 * k, bd, idv, 1);
                    }
                    commit(&bars.vfree[b]);
                    commit(&bars.dfull[b]);
                };
                for (int j = 0; j < sg.nt && ok; ++j) {
                    const int b = j & 1;
                    ok = bar_wait(&bars.kfull[b], nuse[b]++ & 1, fail);
                    if (!ok) break;
                    tc_after();
                    const uint32_t aq = su32(sq), kb = su32(skv) + b * S::TB;
#pragma unroll
                    for (int h = 1; h >= 0; --h)       // lo first: the small products enter a small sum
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            const uint32_t o = (uint32_t)(k >> 2) * 16384 + 32 * (k & 3);
                            mma_ss(sS(b), desc(aq + h * S::QB + o, 16), desc(kb + o, 16), idq, h == 0 || k > 0);
                        }
                    commit(&bars.kfree[b]);
                    commit(&bars.sfull[b]);
                    if (j > 0) pv(j - 1);
                }
                if (ok) pv(sg.nt - 1);
            }
            __syncwarp();
            __syncthreads();
            if (*fail) break;
        }
    } else {
        // ================= K and V: job n is page n % 8 of K (n / 8 even) or V of tile n / 16;
        // warp 8 + w takes jobs w, w + 7, ...
        const int w = warp - 8;
        uint32_t used[2] = {0, 0};                     // tiles before this segment, in each buffer
        while (next_segment()) {
            const int nt = sg.nt, kvh = sg.kvh, tok0 = sg.tok0, end = sg.end, ctx = sg.sq.ctx, slot = sg.sq.slot;
            __syncthreads();
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
            // the operand buffer is free once the product two tiles back has read it
            const auto wait_free = [&](int n) {
                const int j = n >> 4, b = j & 1;
                const uint32_t use = used[b] + (j >> 1);
                if (ok && use > 0)
                    ok = __all_sync(FULL, bar_wait(n & 8 ? &bars.vfree[b] : &bars.kfree[b], (use - 1) & 1, fail));
            };
            const auto arrive = [&](int n) {
                fence_async();
                __syncwarp();
                if (lane == 0) bar_arrive(n & 8 ? &bars.vfull[(n >> 4) & 1] : &bars.kfull[(n >> 4) & 1]);
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
                    float4 ks, vs;                     // K jobs, lanes 0-3: both scales of 4 tokens
                    int page;
                };
                const auto fetch = [&](Raw& r, int n) {
                    const int page = r.page = page_of(n);
                    r.ks = r.vs = make_float4(0.f, 0.f, 0.f, 0.f);
                    const unsigned char* blk = pool + max(page, 0) * page_step + ((n & 8) ? kv_step : 0);
#pragma unroll
                    for (int i = 0; i < NP; ++i)
                        r.x[i] = page < 0 ? make_uint4(0, 0, 0, 0)
                                          : __ldg((const uint4*)(blk + SB_Q8_SCALES) + (lt + TS * i) * U + lk);
                    if (page >= 0 && !(n & 8) && lane < 4) {
                        r.ks = __ldg((const float4*)blk + lane);
                        r.vs = __ldg((const float4*)(blk + kv_step) + lane);
                    }
                };
                const auto put = [&](const Raw& r, int n) {
                    wait_free(n);
                    if (!ok) return;
                    const int j = n >> 4, pg = n & 7;
                    unsigned char* dst = skv + (((n & 8) ? 2 : 0) + (j & 1)) * S::TB + pg * 2048;
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const uint4 v = r.x[i];
                        const uint4 a = make_uint4(i8_f16<0x4140>(v.x), i8_f16<0x4342>(v.x), i8_f16<0x4140>(v.y), i8_f16<0x4342>(v.y));
                        const uint4 z = make_uint4(i8_f16<0x4140>(v.z), i8_f16<0x4342>(v.z), i8_f16<0x4140>(v.w), i8_f16<0x4342>(v.w));
                        *(uint4*)(dst + to[i & 1] + TS * i * 128) = a;
                        *(uint4*)(dst + (to[i & 1] ^ 16) + TS * i * 128) = z;
                    }
                    if (!(n & 8)) {                    // before kfull: the softmax reads them after the scores
                        float vm = 0.f;
                        if (lane < 4) {
                            float* sc = ssc + (j % SCB) * 2 * KT + 16 * pg + 4 * lane;
                            *(float4*)sc = r.ks;
                            *(float4*)(sc + KT) = r.vs;
                            const int t = tok0 + j * KT + 16 * pg + 4 * lane;
                            const float vv[4] = {r.vs.x, r.vs.y, r.vs.z, r.vs.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (t + i < end && vv[i] < INFINITY) vm = fmaxf(vm, vv[i]);
                        }
                        vm = fmaxf(vm, __shfl_xor_sync(FULL, vm, 1));
                        vm = fmaxf(vm, __shfl_xor_sync(FULL, vm, 2));
                        if (lane == 0) {
                            vmax_s[j % SCB][pg] = vm;
                            gone_s[j % SCB][pg] = r.page < 0;
                        }
                    }
                    arrive(n);
                };
                // two pages in flight, in registers of their own: the wait for one is not a wait for
                // the other
                Raw a, z;
                fetch(a, w);
                fetch(z, w + NPW);
                for (int n = w; n < njobs && ok; n += 2 * NPW) {
                    put(a, n);
                    fetch(a, n + 2 * NPW);
                    if (n + NPW < njobs) put(z, n + NPW);
                    fetch(z, n + 3 * NPW);
                }
            } else {
                constexpr int CPT = HD / 8, TS = 32 / CPT, NP = 16 / TS;       // chunks a token; tokens a step
                const auto land = [&](int n) {         // job n has arrived
                    const int j = n >> 4, pg = n & 7, t0 = tok0 + j * KT + 16 * pg;
                    if ((n & 8) && tok0 + j * KT + KT > ctx) {
                        // v that only some rows see: its infinities and NaN leave the tile
                        uint32_t odd = 0;
                        unsigned char* dst = skv + (2 + (j & 1)) * S::TB + pg * 2048;
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
                        if (lane == 0) odd_s[j % SCB][pg] = (uint16_t)odd;
                    }
                    arrive(n);
                };
                int page = page_of(w);
                for (int n = w; n < njobs && ok; n += NPW) {
                    const int j = n >> 4, pg = n & 7, t0 = tok0 + j * KT + 16 * pg;
                    const int next = page_of(n + NPW);
                    wait_free(n);
                    if (!ok) break;
                    const uint32_t dst = su32(skv) + (((n & 8) ? 2 : 0) + (j & 1)) * S::TB + pg * 2048;
                    const unsigned char* src = pool + max(page, 0) * page_step + ((n & 8) ? kv_step : 0) + 16 * lane;
#pragma unroll
                    for (int i = 0; i < NP; ++i)
                        cp16(dst + op_at(lane / CPT + TS * i, lane % CPT), src + 512 * i,
                             page >= 0 && t0 + lane / CPT + TS * i < end);
                    if (lane == 0 && !(n & 8)) gone_s[j % SCB][pg] = page < 0;
                    cp_commit();
                    page = next;
                    // two jobs stay in flight; what a job waits for lies at least 17 jobs back, so the
                    // ones still to land cannot be in its way
                    if (n >= 2 * NPW) {
                        cp_wait<2>();
                        land(n - 2 * NPW);
                    }
                }
                const int mine = (njobs - w + NPW - 1) / NPW;      // the last two of the warp's jobs
                if (ok && mine >= 2) {
                    cp_wait<1>();
                    land(w + (mine - 2) * NPW);
                }
                cp_wait<0>();
                if (ok && mine >= 1) land(w + (mine - 1) * NPW);
            }
            used[0] += (nt + 1) / 2;
            used[1] += nt / 2;
            __syncthreads();
            if (*fail) break;
        }
    }
    }
    __syncthreads();
    if (*fail) {
        // products and copies in flight end before the CTA does; then, what this CTA owed and
        // did not do: NaN, whole or in part
        for (const uint64_t t0 = gtimer(); gtimer() - t0 < WAIT_NS / 100;) {}
        while (next_segment()) {
            for (int e = tid; e < sg.n_rows * (HD + 2); e += NTHREADS) {
                const int r = e / (HD + 2), d = e % (HD + 2), row = sg.r_base + r;
                if (!sg.whole) ws[((size_t)(2 * blockIdx.x + 1) * MR + r) * (HD + 2) + d] = NAN;
                else if (d < HD) out[(size_t)(sg.sq.r0 + row / G) * ld_out + (size_t)(sg.kvh * G + row % G) * HD + d] = NAN;
            }
        }
    }
    if (warp == 15) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int KV, int HD>
int launch(const slate_kv_cache_t& c, int layer, const slate_tree_t& tr, int nq, float* out, int ld_out,
           const float* q, int ld_q, float scale, float* ws, cudaStream_t st) {
    const auto k = attn_tree_tc<KV, HD>;
    static const cudaError_t ready =
        cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<KV, HD>::SMEM);
    if (ready != cudaSuccess) return sb_cuda_check(ready, "attention_tree shared memory");
    k<<<SMS, NTHREADS, TcShape<KV, HD>::SMEM, st>>>(c, layer, tr, nq, out, ld_out, q, ld_q, scale, ws);
    return sb_cuda_check(cudaGetLastError(), "attention_tree");
}

}  // namespace

int sb_tree::attend_tc(const slate_kv_cache_t& c, int layer, const slate_tree_t& tr, int nq, float* out, int ld_out,
                       const float* q, int ld_q, float scale, float* ws, cudaStream_t st) {
    const auto f = c.kv_dtype == SLATE_KV_F16 ? (c.head_dim == 64 ? launch<SLATE_KV_F16, 64> : launch<SLATE_KV_F16, 128>)
                                              : (c.head_dim == 64 ? launch<SLATE_KV_Q8, 64> : launch<SLATE_KV_Q8, 128>);
    return f(c, layer, tr, nq, out, ld_out, q, ld_q, scale, ws, st);
}
