// attn_tree.cu -- attention of token-tree nodes over the paged cache
// (slate_cuda_attention_tree): for row i of a sequence, kv head h and each query
// head of its group
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - max_j),
// over j < ctx (the context) and the nodes j that bit j - ctx of the row's mask
// names.
//
// The M = nodes * group rows that share a kv head are one matrix product with the
// cache: attn_tree_mma (head_dim 64 and 128) reads the cache once for up to 32 of
// them (16 at head_dim 128 on f16 and 8 bits, where attn_tree_tc takes the others) and multiplies on the tensor
// cores; attn_tree_rows takes any head_dim.
//
// f32-level products from 16-bit operands.  f16 and 8-bit cache: k and v are
// exact in f16 (8 bits: the integer; its scale joins the score, or p).  q and p
// are split into f16 hi + lo, so two products carry
// what f32 would.  To stay clear of f16's ends each q row is first divided by the
// power of two that leaves its largest element at 2^14 or more, and p (at most 1) multiplied by 2^15: an
// element down to 2^-18 of the largest keeps 22 bits, a smaller one is off by 2^-40 of the largest at most.
// 8 bits, up to 16 rows: q as integers of four 8-bit digits, each element off by 2^-24 of itself and 2^-31 of the
// row's largest.  f32 cache: tf32 hi + lo of
// both sides (22 bits whatever the size), three products, lo lo left out: 2^-22 of a product.  The running sums stay in
// f32 registers: every tile's
// product is formed from zero and added by one FMA with the rescale, because a
// tensor-core accumulator carried over thousands of tokens would truncate each time.
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

// Any head_dim: one CTA per (row, query head), its four warps take pages in
// turn.  A page's scores are formed first, then its maximum joins the running
// one and its sum of p v is formed by itself before it joins the running sum,
// which keeps the f32 sums of long contexts two levels deep.  Keys that the row
// does not see are skipped, so nothing they hold can reach it.  Each row reads the
// cache by itself: the head_dims that no common model has.
constexpr int NW = 4;
__global__ void __launch_bounds__(32 * NW, 8) attn_tree_rows(
    const slate_kv_cache_t c, int layer, const slate_tree_t tr, int nq, float* __restrict__ out,
    int ld_out, const float* __restrict__ q, int ld_q, float scale) {
    __shared__ float sm[NW], sl[NW], so[NW][256];
    sb_grid_wait();
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, hd = c.head_dim;
    const int row = blockIdx.x, h = blockIdx.y, kvh = h / (nq / c.n_kv_heads);
    // the row's sequence: the last s with row_off[s] <= row
    int lo = 0, hi = tr.n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (tr.row_off[mid] <= row) lo = mid;
        else hi = mid;
    }
    const int r0 = max(tr.row_off[lo], 0), slot = tr.slot[lo];
    const int ctx = min(max(tr.ctx[lo], 0), c.max_pages * SB_PAGE_TOKENS);
    const int n = min(max(min(tr.row_off[lo + 1], tr.rows) - r0, 0), tr.max_nodes);
    if (row < r0 || row >= r0 + n) return;               // of no sequence, or beyond max_nodes: left as it is
    const uint64_t mask = tr.mask[row];
    const int end = ctx + n;
    float qv[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        qv[i] = d < hd ? q[(size_t)row * ld_q + (size_t)h * hd + d] * scale : 0.f;
        o[i] = 0.f;
    }
    for (int pg = warp; pg * SB_PAGE_TOKENS < end; pg += NW) {
        const int page = sb_kv_page(c, slot, pg * SB_PAGE_TOKENS);
        if (page < 0) continue;
        const unsigned char* kb = sb_kv_block(c, layer, page, 0, kvh);
        const unsigned char* vb = sb_kv_block(c, layer, page, 1, kvh);
        float sc = -INFINITY;                            // lane t: the score of token t
        for (int t = 0; t < SB_PAGE_TOKENS; ++t) {
            const int j = pg * SB_PAGE_TOKENS + t;
            if (j >= end || (j >= ctx && !(mask >> (j - ctx) & 1))) continue;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane + 32 * i < hd) s = fmaf(qv[i], kv_element(kb, c.kv_dtype, t * hd + lane + 32 * i), s);
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(FULL, s, x);
            if (c.kv_dtype == SLATE_KV_Q8) s *= no_inf(((const float*)kb)[t]);
            if (lane == t) sc = s;
        }
        float mx = sc;
        for (int x = 16; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, x));
        // a NaN score reaches the sums through p below (fmaxf passes it by)
        const bool any = __any_sync(FULL, sc != -INFINITY);
        if (!any) continue;
        const float mn = fmaxf(m, mx), corr = m == -INFINITY ? 0.f : expf(m - mn);
        const float p = sc == -INFINITY ? 0.f : expf(sc - mn);
        float ps = p, po[8];
        for (int x = 16; x; x >>= 1) ps += __shfl_xor_sync(FULL, ps, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) po[i] = 0.f;
        for (int t = 0; t < SB_PAGE_TOKENS; ++t) {
            const int j = pg * SB_PAGE_TOKENS + t;
            if (j >= end || (j >= ctx && !(mask >> (j - ctx) & 1))) continue;
            float pt = __shfl_sync(FULL, p, t);
            if (c.kv_dtype == SLATE_KV_Q8) pt *= ((const float*)vb)[t];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane + 32 * i < hd)
                    po[i] = fmaf(pt, kv_element(vb, c.kv_dtype, t * hd + lane + 32 * i), po[i]);
        }
        l = fmaf(l, corr, ps);
        m = mn;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = fmaf(o[i], corr, po[i]);
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) so[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w]);
    // a warp that saw no key has l = 0 and o = 0
    for (int w = 0; w < NW; ++w) L += sl[w] * (sm[w] == -INFINITY ? 1.f : expf(sm[w] - M));
    bool nan = false;
    for (int d = tid; d < hd; d += 32 * NW) {
        float O = 0.f;
        for (int w = 0; w < NW; ++w) O += so[w][d] * (sm[w] == -INFINITY ? 1.f : expf(sm[w] - M));
        O = L == 0.f ? 0.f : O / L;
        nan |= O != O;
        out[(size_t)row * ld_out + (size_t)h * hd + d] = O;
    }
    if (__syncthreads_or(nan) && warp == 0)
        row_by_formula<8>(row_job(c, layer, kvh, slot, ctx, n, mask), q + (size_t)row * ld_q + (size_t)h * hd, scale,
                       out + (size_t)row * ld_out + (size_t)h * hd);
}

// ------------------------------------------------------------ tensor-core path
constexpr int UNIT = 64;
constexpr int MW = 4;                       // warps a CTA
constexpr float DIG = 127.f * 0x1p24f;      // four digits to base 256 stay within 8 bits each

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
                 "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_i8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 "
                 "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 "
                 "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo in tf32 (the low 13 bits cut off)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
// KT tokens of K and V a tile and warp, ~8 KB, in a ring of NS tiles for each warp
// (the ring and q fit CPS times into an SM's shared memory).  A row's 16-byte chunks are
// exchanged by XOR with a function of the row, so that neither ldmatrix (8 rows, one
// chunk each) nor the f32 reads (4 or 8 rows) meet in a bank.
template <int KV, int HD, int MODE>
struct Shape {
    // (f32: a unit's arithmetic takes longer than what a second range costs; with 0, 1 and 4: 16 x 7 nodes over 700
    // tokens 31.2, 29.0 and 28.9 us, over 1501 42.6, 42.6 and 44.4, over 3000 64.3, 64.4 and 71.2, 5 x 1 over 6000
    // at head_dim 128 41.8, 39.8 and 39.8)
    static constexpr int SLACK = KV == SLATE_KV_F32 ? 1 : 4;
    static constexpr int RB = KV == SLATE_KV_F32 ? 4 * HD : KV == SLATE_KV_F16 ? 2 * HD : HD;
    static constexpr int KT = RB == 512 ? 8 : RB == 256 ? 16 : 32;
    static constexpr int CPR = RB / 16;
    static constexpr int TB = 2 * KT * RB + (KV == SLATE_KV_Q8 ? 8 * KT : 0);
    static constexpr int MT = MODE == 2 ? 2 : 1;
    static constexpr int MR = MODE == 0 ? 8 : 16 * MT;              // rows a tile
    // 8 bits and up to 16 rows: scores from integer products, q in four 8-bit digits
    static constexpr bool I8 = KV == SLATE_KV_Q8 && MODE < 2;
    static constexpr int KS = I8 ? HD / 32 : KV == SLATE_KV_F32 ? HD / 8 : HD / 16;    // k steps of a score
    static constexpr int HL = I8 ? 2 * MODE + 2 : MODE == 0 ? 1 : 2;    // A operands a k step
    static constexpr int QB = MT * KS * HL * 512;
    // CTAs an SM: three where 168 registers a thread do (64 sequences of one node over 4096 tokens 57
    // us, with two 62; head_dim 128 spilled with three, 93 against 84)
    static constexpr int CPS = KV == SLATE_KV_Q8 && HD == 64 && MODE == 0 ? 3 : 2;
    static_assert(CPS * MR <= TC_ROWS && CPS * SMS <= MAX_CTAS, "workspace");
    static constexpr int NS0 = ((CPS == 3 ? 74 : 112) * 1024 - QB) / (MW * TB);
    static constexpr int NS = NS0 > 6 ? 6 : NS0;
    static constexpr int MERGE = MW * MR * (HD + 2) * 4;
    static constexpr int RING = MW * NS * TB > MERGE ? MW * NS * TB : MERGE;
    static constexpr int SMEM = QB + RING + MR * 16;
};
template <int KV, int RB>
__device__ __forceinline__ uint32_t swz(int row, int chunk) {
    if (KV == SLATE_KV_F32)      // rows 0,2,4,6 (or 1,3,5,7) of one dim, rows 2i and 2i + 1 of 4 chunks
        return row * RB + ((chunk ^ ((row & 6) ^ ((row & 1) << 2))) << 4);
    if (RB == 64) {              // two rows a 128-byte line
        const int line = row >> 1, pos = (row & 1) * 4 + chunk;
        return line * 128 + ((pos ^ (line & 3)) << 4);
    }
    return row * RB + ((chunk ^ (row & 7)) << 4);
}

// A CTA of four warps, each with its own ring of tiles.  What bounds it: HBM for up to 8 rows of f16 and f32 (64
// sequences of one node over 4096 tokens, 32 heads over 8 of 128: 129 and 243 us, 6.2 and 6.6 TB/s).  8 bits: neither
// HBM (60 % busy) nor the issue slots (54 %), but the latency between a warp's own instructions, two warps a
// scheduler at 253 registers (the same call: 85 us, 4.9 TB/s).  f32 with 32
// rows: the three tf32 products and the latency between them, again two warps a scheduler:
// 16 x 7 nodes over 1501 tokens, 32 heads over 8 of 64: 42.5 us, 1.8 TB/s (12000
// tokens: 179 us, 3.3 TB/s).  One node over 700 tokens: 8.9 us, two launches and five dependent
// reads.
// Partial of one cut item: [MR][HD + 2]: (max in log2 units, sum, o) rows.
template <int KV, int HD, int MODE>
__global__ void __launch_bounds__(32 * MW, Shape<KV, HD, MODE>::CPS) attn_tree_mma(
    const slate_kv_cache_t c, int layer, const slate_tree_t tr, int nq, float* __restrict__ out,
    int ld_out, const float* __restrict__ q, int ld_q, float scale, float* __restrict__ ws) {
    using S = Shape<KV, HD, MODE>;
    constexpr int KT = S::KT, RB = S::RB, TB = S::TB, NS = S::NS, MT = S::MT, MR = S::MR, KS = S::KS;
    constexpr int NTK = KT / 8;                       // 8-token score tiles
    constexpr int NTD = HD / 8;                       // 8-dim output tiles
    constexpr int RI = MODE == 0 ? 1 : 2 * MT;        // rows a lane
    extern __shared__ __align__(128) unsigned char smem[];
    uint4* sq = (uint4*)smem;                         // [MT][KS][HL][32 lanes] A fragments
    unsigned char* ring = smem + S::QB;
    float* rowscale = (float*)(smem + S::QB + S::RING);        // [MR]
    uint64_t* rowmask = (uint64_t*)(rowscale + 2 * ((MR + 1) / 2));   // [MR]
    __shared__ PlanBuf buf;
    sb_grid_wait();
    sb_grid_release();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int nkv = c.n_kv_heads, G = nq / nkv;
    Start st_;
    int unit = UNIT;
    if (!plan_start(c, tr, G, MR, unit, S::SLACK, gridDim.x, buf, st_)) return;
    if (tid == 0) nan_words(ws, HD)[blockIdx.x] = 0;
    int64_t at = st_.at, seq_before = st_.seq_before;
    const int64_t stop = st_.stop;
    Seq sq_ = st_.sq;
    int s = sq_.s;
    const size_t page_blk = sb_kv_block_bytes(KV, HD);
    unsigned char* myring = ring + (size_t)warp * NS * TB;
    const uint32_t myring_s = su32(myring);

    for (int seg = 0; at < stop; ++seg) {
        while (at >= seq_before + seq_units(sq_, nkv)) {
            seq_before += seq_units(sq_, nkv);
            sq_ = seq_of(c, tr, ++s, G, MR, unit);
        }
        int u0;
        const int item = item_of(at - seq_before, sq_.units, u0);
        const int u1 = (int)min((int64_t)sq_.units, u0 + (stop - at));
        const int kvh = item / sq_.tiles, r_base = (item % sq_.tiles) * MR;
        const int n_rows = min(MR, sq_.n * G - r_base);
        const int end = sq_.ctx + sq_.n, tok0 = u0 * unit, tok1 = min(end, u1 * unit);
        at += u1 - u0;

        // ---- q as A fragments, each row divided by a power of two
        __syncthreads();                               // the last segment's merge is read
        if (tid < MR) rowmask[tid] = tid < n_rows ? __ldg(tr.mask + sq_.r0 + (r_base + tid) / G) : 0;
        float qv[MR / MW][HD / 32];                    // all of the warp's rows before any is used
#pragma unroll
        for (int k = 0; k < MR / MW; ++k) {
            const int row = r_base + min(warp + k * MW, n_rows - 1);
            const float* x = q + (size_t)(sq_.r0 + row / G) * ld_q + (size_t)(kvh * G + row % G) * HD + lane * (HD / 32);
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) qv[k][i] = x[i];
        }
#pragma unroll
        for (int k = 0; k < MR / MW; ++k) {
            const int r = warp + k * MW;
            float(&v)[HD / 32] = qv[k];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
            }
            top = __reduce_max_sync(FULL, top);
            // exponent of the maximum, kept where 2^-e and 2^e are normal numbers
            constexpr int UP = KV == SLATE_KV_F32 || S::I8 ? 0 : 14;
            const int e = min(max((int)(top >> 23) - 127, UP - 126), 126) - UP;
            const float inv = __int_as_float((127 - e) << 23);
            if (lane == 0) rowscale[r] = scale * 1.4426950408889634f * __int_as_float((127 + e) << 23);
            if constexpr (S::I8) {
                // q / 2^(e + 1) (below 1) times DIG as an integer of four digits to base 256, each in
                // -128 .. 127: an element is off by 2^-24 of itself (the factor 127) and 2^-31 of the row's largest.
                // Dims 32 ks + 16 hi + 4 t + b are byte b of register 2 hi (+ 1: row + 8)
                // of lane (row % 8, t).  Up to 8 rows: an operand holds a digit in its rows 0-7 and the next lower
                // one in rows 8-15; else an operand a digit.
                // (a maximum of 2^127 and more has no digits: by the formula)
                if (lane == 0) rowscale[r] = top < 0x7f000000u ? rowscale[r] * (2.f / DIG) : NAN;
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    const int d = lane * (HD / 32) + i, v0 = __float2int_rn(v[i] * inv * (0.5f * DIG));
                    const int d0 = (int8_t)v0, v1 = (v0 - d0) >> 8, d1 = (int8_t)v1, v2 = (v1 - d1) >> 8, d2 = (int8_t)v2;
                    const int digit[4] = {(v2 - d2) >> 8, d2, d1, d0};
                    const int reg = (d >> 4 & 1) * 2, at = ((r & 7) * 4 + (d >> 2 & 3)) * 16 + (d & 3);
                    int8_t* f8 = (int8_t*)(sq + (size_t)(d / 32) * S::HL * 32);
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const int op = MODE == 0 ? h / 2 : h, up8 = MODE == 0 ? h % 2 : r >> 3 & 1;
                        f8[512 * op + at + 4 * (reg + up8)] = (int8_t)digit[h];
                    }
                }
            } else {
            // element d of row r in the fragments: rows r % 16 < 8 in registers 0 and 2
            const int mt = r / 16, rg = r & 7, up = MODE == 0 ? 0 : (r >> 3) & 1;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                const int d = lane * (HD / 32) + i;
                // (f16 halves: y of 2^14 and more for the row's largest, so that the low halves of elements down to
                // 2^-18 of it have all of their bits)
                const float y = v[i] * inv;
                if (KV == SLATE_KV_F32) {
                    // k steps 2j, 2j + 1 hold dims 16j + 4 t4 + {0, 1} and {2, 3}
                    const int ks = 2 * (d / 16) + ((d & 3) >> 1), t = (d & 15) >> 2, reg = 2 * (d & 1) + up;
                    uint32_t hi, lo;
                    split_tf32(y, hi, lo);
                    uint32_t* f = (uint32_t*)(sq + ((size_t)(mt * KS + ks) * S::HL) * 32 + rg * 4 + t);
                    f[reg] = hi;
                    f[MODE == 0 ? reg + 1 : 32 * 4 + reg] = lo;
                } else {
                    // f16: k = dim; 8 bits: dims 4 t4 + {0, 1} are k 2 t4 + {0, 1}, {2, 3} k + 8
                    const int ks = d / 16, w = d & 15;
                    const int t = KV == SLATE_KV_Q8 ? w >> 2 : (w & 7) >> 1;
                    const int reg = 2 * (KV == SLATE_KV_Q8 ? (w & 3) >> 1 : w >> 3) + up;
                    const __half hi = __float2half_rn(y), lo = __float2half_rn(y - __half2float(hi));
                    __half* f = (__half*)(sq + ((size_t)(mt * KS + ks) * S::HL) * 32 + rg * 4 + t);
                    f[2 * reg + (d & 1)] = hi;
                    f[(MODE == 0 ? 2 * (reg + 1) : 32 * 8 + 2 * reg) + (d & 1)] = lo;
                }
            }
            }
        }
        __syncthreads();

        float o[MT][NTD][4], m[RI], l[RI], rs[RI];
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int j = 0; j < NTD; ++j) o[a][j][0] = o[a][j][1] = o[a][j][2] = o[a][j][3] = 0.f;
#pragma unroll
        for (int i = 0; i < RI; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
            rs[i] = rowscale[8 * i + g];
        }
        float vtop[RI];                                // 8 bits: row's o is in units of 2^(vtop - 15)
#pragma unroll
        for (int i = 0; i < RI; ++i) vtop[i] = -1e30f;

        // ---- the warp's tiles: KT tokens each, tiles warp, warp + MW, ...
        const int tiles = (tok1 - tok0 + KT - 1) / KT;
        const int mine = warp < tiles ? (tiles - 1 - warp) / MW + 1 : 0;
        constexpr int PPT = KT > 16 ? KT / 16 : 1;     // pages a tile
        // lane i: pages of the warp's tile (base + i), of these 32 tiles and the next
        int win[PPT], nwin[PPT];
        uint32_t absent = 0;                           // bit (stage, page): the table has no such page
        auto load_window = [&](int base, int (&w)[PPT]) {
#pragma unroll
            for (int p = 0; p < PPT; ++p) {
                const int t = tok0 + (warp + (base + lane) * MW) * KT + 16 * p;
                w[p] = base + lane < mine && t < tok1 ? sb_kv_page(c, sq_.slot, t) : -1;
            }
        };
        load_window(0, win);
        load_window(32, nwin);
        const size_t kv_step = (size_t)nkv * page_blk, page_step = 2 * kv_step;
        const unsigned char* pool = sb_kv_block(c, layer, 0, 0, kvh);
        auto issue = [&](int i) {                      // the warp's i-th tile into stage i % NS
            if (i < mine) {
                if (i > 0 && (i & 31) == 0) {
#pragma unroll
                    for (int p = 0; p < PPT; ++p) win[p] = nwin[p];
                    load_window(i + 32, nwin);
                }
                const int t0 = tok0 + (warp + i * MW) * KT;
                const uint32_t st = myring_s + (i % NS) * TB;
#pragma unroll
                for (int p = 0; p < PPT; ++p) {
                    const int page = __shfl_sync(FULL, win[p], i & 31);
                    const uint32_t bit = 1u << ((i % NS) * PPT + p);
                    absent = page < 0 ? absent | bit : absent & ~bit;
                    const unsigned char* kb = pool + max(page, 0) * page_step;
                    const unsigned char* vb = kb + kv_step;
                    constexpr int ROWS = KT < 16 ? KT : 16, HEAD = KV == SLATE_KV_Q8 ? SB_Q8_SCALES : 0;
                    const int rsrc = KT < 16 ? t0 & 15 : 0;
#pragma unroll
                    for (int e = lane; e < ROWS * S::CPR; e += 32) {
                        const int r = e / S::CPR, ch = e % S::CPR;
                        const bool ok = page >= 0 && t0 + 16 * p + r < end;
                        const size_t so = HEAD + (size_t)(rsrc + r) * RB + ch * 16;
                        const uint32_t d = swz<KV, RB>(16 * p + r, ch);
                        cp16(st + d, kb + so, ok);
                        cp16(st + KT * RB + d, vb + so, ok);
                    }
                    if (KV == SLATE_KV_Q8 && lane < 8)
                        cp16(st + 2 * KT * RB + (lane >= 4 ? 4 * KT : 0) + 64 * p + 16 * (lane & 3),
                             (lane >= 4 ? vb : kb) + 16 * (lane & 3), page >= 0);
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) issue(i);
        for (int i = 0; i < mine; ++i) {
            cp_wait<NS - 2>();
            __syncwarp();
            const int t0 = tok0 + (warp + i * MW) * KT;
            const unsigned char* st = myring + (size_t)(i % NS) * TB;
            const uint32_t ks_ = myring_s + (i % NS) * TB, vs_ = ks_ + KT * RB;
            const float* ksc = (const float*)(st + 2 * KT * RB);
            const float* vsc = ksc + KT;
            float sc[MT][NTK][4];
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int j = 0; j < NTK; ++j) sc[a][j][0] = sc[a][j][1] = sc[a][j][2] = sc[a][j][3] = 0.f;
            // ---- scores
            if constexpr (KV == SLATE_KV_F32) {
                // the products with a low half in sums of their own: a tensor-core sum is cut off at every
                // step, and the large one takes a third of the steps this way
                float sx[MT][NTK][4];
#pragma unroll
                for (int a = 0; a < MT; ++a)
#pragma unroll
                    for (int j = 0; j < NTK; ++j) sx[a][j][0] = sx[a][j][1] = sx[a][j][2] = sx[a][j][3] = 0.f;
#pragma unroll
                for (int cc = 0; cc < HD / 16; ++cc) {
                    uint4 A[MT][2][S::HL];
#pragma unroll
                    for (int a = 0; a < MT; ++a)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int h = 0; h < S::HL; ++h)
                                A[a][k][h] = sq[((size_t)(a * KS + 2 * cc + k) * S::HL + h) * 32 + lane];
                    uint32_t bh[NTK][4], bl[NTK][4];
#pragma unroll
                    for (int j = 0; j < NTK; ++j) {
                        const float4 x = *(const float4*)(st + swz<KV, RB>(8 * j + g, 4 * cc + t4));
                        split_tf32(x.x, bh[j][0], bl[j][0]);
                        split_tf32(x.y, bh[j][1], bl[j][1]);
                        split_tf32(x.z, bh[j][2], bl[j][2]);
                        split_tf32(x.w, bh[j][3], bl[j][3]);
                    }
                    // (a sum's next product stands behind those of the other sums)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int z = 0; z < 3; ++z)        // hi lo, hi hi, lo hi
#pragma unroll
                            for (int j = 0; j < NTK; ++j)
#pragma unroll
                                for (int a = 0; a < MT; ++a) {
                                    const uint4 q4 = A[a][k][z < 2 ? 0 : S::HL - 1];
                                    const uint32_t aq[4] = {q4.x, q4.y, q4.z, q4.w};
                                    if (z == 0) mma_tf32(sx[a][j], aq, bl[j][2 * k], bl[j][2 * k + 1]);
                                    if (z == 1) mma_tf32(sc[a][j], aq, bh[j][2 * k], bh[j][2 * k + 1]);
                                    if (z == 2 && MODE) mma_tf32(sx[a][j], aq, bh[j][2 * k], bh[j][2 * k + 1]);
                                }
                }
#pragma unroll
                for (int a = 0; a < MT; ++a)
#pragma unroll
                    for (int j = 0; j < NTK; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[a][j][e] += sx[a][j][e];
            } else if constexpr (S::I8) {
                // exact: |sum| <= 128 * 127 * 128 < 2^21.  The sums start at the bits of 1.5 * 2^23, so that
                // the result read as a float is 1.5 * 2^23 + sum
                constexpr float BIAS = 12582912.f;
                int acc[S::HL][NTK][4];
#pragma unroll
                for (int h = 0; h < S::HL; ++h)
#pragma unroll
                    for (int j = 0; j < NTK; ++j)
                        acc[h][j][0] = acc[h][j][1] = acc[h][j][2] = acc[h][j][3] = 0x4b400000;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t A[S::HL][4];
#pragma unroll
                    for (int h = 0; h < S::HL; ++h) {
                        const uint4 x = sq[(k * S::HL + h) * 32 + lane];
                        A[h][0] = x.x, A[h][1] = x.y, A[h][2] = x.z, A[h][3] = x.w;
                    }
#pragma unroll
                    for (int jp = 0; jp < NTK / 2; ++jp) {
                        uint32_t r[4];
                        ldsm4(ks_ + swz<KV, RB>(16 * jp + (lane >> 4) * 8 + (lane & 7), 2 * k + ((lane >> 3) & 1)), r);
#pragma unroll
                        for (int h = 0; h < S::HL; ++h) {
                            mma_i8(acc[h][2 * jp], A[h], r[0], r[1]);
                            mma_i8(acc[h][2 * jp + 1], A[h], r[2], r[3]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < NTK; ++j)
#pragma unroll
                    for (int e = 0; e < (MODE == 0 ? 2 : 4); ++e) {
                        float x = 0.f;
#pragma unroll
                        for (int h = 0; h < 4; ++h)
                            x = fmaf(x, 256.f, __int_as_float(acc[MODE == 0 ? h / 2 : h][j][MODE == 0 ? 2 * (h % 2) + e : e]) - BIAS);
                        sc[0][j][e] = x;
                    }
            } else {
                // an ldmatrix.x4 brings two 8-token tiles: f16 of one k step, 8 bits of two
                constexpr int KPL = KV == SLATE_KV_Q8 ? 2 : 1;
#pragma unroll
                for (int cc = 0; cc < KS / KPL; ++cc) {
                    uint4 A[MT][KPL][S::HL];
#pragma unroll
                    for (int a = 0; a < MT; ++a)
#pragma unroll
                        for (int k = 0; k < KPL; ++k)
#pragma unroll
                            for (int h = 0; h < S::HL; ++h)
                                A[a][k][h] = sq[((size_t)(a * KS + KPL * cc + k) * S::HL + h) * 32 + lane];
#pragma unroll
                    for (int jp = 0; jp < NTK / 2; ++jp) {
                        uint32_t r[4];
                        ldsm4(ks_ + swz<KV, RB>(16 * jp + (lane >> 4) * 8 + (lane & 7), 2 * cc + ((lane >> 3) & 1)), r);
#pragma unroll
                        for (int k = 0; k < KPL; ++k) {
                            uint32_t b[2][2];
#pragma unroll
                            for (int jj = 0; jj < 2; ++jj) {
                                b[jj][0] = KV == SLATE_KV_Q8 ? i8_f16<0x4140>(r[2 * jj + k]) : r[2 * jj];
                                b[jj][1] = KV == SLATE_KV_Q8 ? i8_f16<0x4342>(r[2 * jj + k]) : r[2 * jj + 1];
                            }
#pragma unroll
                            for (int h = S::HL - 1; h >= 0; --h)
#pragma unroll
                                for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                                    for (int a = 0; a < MT; ++a) {
                                        const uint4 x = A[a][k][h];
                                        const uint32_t af[4] = {x.x, x.y, x.z, x.w};
                                        mma_f16(sc[a][2 * jp + jj], af, b[jj][0], b[jj][1]);
                                    }
                        }
                    }
                }
            }
            // ---- softmax over the tile: lane holds tokens 8 j + 2 t4 + e of rows 8 ri + g
            const uint32_t gone = absent >> ((i % NS) * PPT) & ((1u << PPT) - 1);
            const bool tail = t0 + KT > sq_.ctx || gone;
            float p[RI][NTK][2], kf[NTK][2];
#pragma unroll
            for (int j = 0; j < NTK; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) kf[j][e] = 1.f;
            if (KV == SLATE_KV_Q8)
#pragma unroll
                for (int j = 0; j < NTK; ++j) {
                    const float2 x = *(const float2*)(ksc + 8 * j + 2 * t4);
                    kf[j][0] = no_inf(x.x), kf[j][1] = no_inf(x.y);
                }
            float corr[RI];
#pragma unroll
            for (int ri = 0; ri < RI; ++ri) {
                float mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < NTK; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float d = S::I8 && MODE == 0 ? sc[0][j][e]
                                        : MODE == 0    ? sc[0][j][e] + sc[0][j][2 + e]
                                                       : sc[ri >> 1][j][2 * (ri & 1) + e];
                        p[ri][j][e] = d * (KV == SLATE_KV_Q8 ? rs[ri] * kf[j][e] : rs[ri]);
                    }
                if (tail) {
                    const uint64_t mk = rowmask[8 * ri + g];
#pragma unroll
                    for (int j = 0; j < NTK; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int x = t0 + 8 * j + 2 * t4 + e - sq_.ctx;
                            if ((x >= 0 && (x >= sq_.n || !(mk >> x & 1))) || (gone >> (8 * j / 16) & 1))
                                p[ri][j][e] = -INFINITY;
                        }
                }
#pragma unroll
                for (int j = 0; j < NTK; ++j) mx = fmaxf(mx, fmaxf(p[ri][j][0], p[ri][j][1]));
                mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 2));
                const float mn = fmaxf(m[ri], mx), base = mn == -INFINITY ? 0.f : mn;
                corr[ri] = ex2(m[ri] - base);
                m[ri] = mn;
                l[ri] *= corr[ri];
#pragma unroll
                for (int j = 0; j < NTK; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        p[ri][j][e] = ex2(p[ri][j][e] - base);
                        l[ri] += p[ri][j][e];
                    }
            }
            // ---- weights of v: 8 bits: p vscale against the row's largest so far: that of the tokens which it
            // sees, with their p, so that no scale that weighs nothing in a row takes the others' bits in f16.
            // vtop = m + its log2 only grows.  0 stays 0 whatever the scale
            if (KV == SLATE_KV_Q8) {
                float vf[NTK][2];
#pragma unroll
                for (int j = 0; j < NTK; ++j) {
                    const float2 x = *(const float2*)(vsc + 8 * j + 2 * t4);
                    vf[j][0] = x.x, vf[j][1] = x.y;
                }
#pragma unroll
                for (int ri = 0; ri < RI; ++ri) {
                    float top = 0.f;
#pragma unroll
                    for (int j = 0; j < NTK; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            p[ri][j][e] = tail && p[ri][j][e] == 0.f ? 0.f : p[ri][j][e] * vf[j][e];
                            top = fmaxf(top, fabsf(p[ri][j][e]));
                        }
                    top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
                    const float grown = fmaxf(vtop[ri], m[ri] + fmaxf(lg2(top), -100.f));
                    corr[ri] = ex2(vtop[ri] - grown);
                    vtop[ri] = grown;
                    const float f = ex2(m[ri] - grown + 15.f);
#pragma unroll
                    for (int j = 0; j < NTK; ++j) p[ri][j][0] *= f, p[ri][j][1] *= f;
                }
            }
            // An infinity or NaN in a v that only some rows see would reach the others as
            // 0 * inf: such values are taken out of the tile (8 bits: their p is 0 already), and the rows that see
            // them made NaN, to be computed by the formula.
            if (tail) {
                uint32_t odd = 0;
                if (KV == SLATE_KV_Q8)
                    odd = __ballot_sync(FULL, t0 + lane >= sq_.ctx && t0 + lane < end && !(fabsf(vsc[lane]) < INFINITY));
                else {
                    for (int e = lane; e < KT * S::CPR; e += 32) {
                        const int r = e / S::CPR;
                        uint32_t* w = (uint32_t*)(st + KT * RB + swz<KV, RB>(r, e % S::CPR));
                        if (t0 + r < sq_.ctx) continue;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t x = w[k];
                            uint32_t keep = 0xffffffffu;
                            if (KV == SLATE_KV_F32) {
                                if ((x & 0x7f800000u) == 0x7f800000u) keep = 0;
                            } else {
                                if ((x & 0x7c00u) == 0x7c00u) keep &= 0xffff0000u;
                                if ((x & 0x7c000000u) == 0x7c000000u) keep &= 0x0000ffffu;
                            }
                            if (keep != 0xffffffffu) {
                                w[k] = x & keep;
                                odd |= 1u << r;
                            }
                        }
                    }
                    odd = __reduce_or_sync(FULL, odd);
                    __syncwarp();                      // other lanes read the words that this one changed
                }
                if (odd) {
                    const int x = t0 - sq_.ctx;        // above -32
#pragma unroll
                    for (int ri = 0; ri < RI; ++ri) {
                        const uint64_t mk = rowmask[8 * ri + g];
                        if (odd & (uint32_t)(x >= 0 ? mk >> x : mk << -x)) l[ri] = NAN;
                    }
                }
            }
            // ---- o = o corr + p v
            if constexpr (KV == SLATE_KV_F32) {
                // up to 8 rows: rows 0-7 of ph hold the high halves, rows 8-15 the low ones
                uint32_t ph[MT][NTK][4], pl[MT][NTK][4];
#pragma unroll
                for (int a = 0; a < MT; ++a)
#pragma unroll
                    for (int j = 0; j < NTK; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (MODE == 0) {
                                split_tf32(p[0][j][e], ph[a][j][2 * e], ph[a][j][2 * e + 1]);
                            } else {
                                split_tf32(p[(2 * a) % RI][j][e], ph[a][j][2 * e], pl[a][j][2 * e]);
                                split_tf32(p[(2 * a + 1) % RI][j][e], ph[a][j][2 * e + 1], pl[a][j][2 * e + 1]);
                            }
#pragma unroll
                for (int jd = 0; jd < NTD; jd += 2) {
                    float d[2][MT][4];
                    uint32_t bh[2][NTK][2], bl[2][NTK][2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
#pragma unroll
                        for (int a = 0; a < MT; ++a) d[x][a][0] = d[x][a][1] = d[x][a][2] = d[x][a][3] = 0.f;
#pragma unroll
                        for (int j = 0; j < NTK; ++j) {
                            // k = t4 is token 2 t4, k = t4 + 4 token 2 t4 + 1 of the 8
                            const int r = 8 * j + 2 * t4, ch = 2 * (jd + x) + (g >> 2);
                            split_tf32(*(const float*)(st + KT * RB + swz<KV, RB>(r, ch) + 4 * (g & 3)), bh[x][j][0], bl[x][j][0]);
                            split_tf32(*(const float*)(st + KT * RB + swz<KV, RB>(r + 1, ch) + 4 * (g & 3)), bh[x][j][1], bl[x][j][1]);
                        }
                    }
                    // the products with a low half first, while the sum is small
#pragma unroll
                    for (int z = 0; z < 3; ++z)            // lo hi, hi lo, hi hi
#pragma unroll
                        for (int j = 0; j < NTK; ++j)
#pragma unroll
                            for (int x = 0; x < 2; ++x)
#pragma unroll
                                for (int a = 0; a < MT; ++a) {
                                    if (z == 0 && MODE) mma_tf32(d[x][a], pl[a][j], bh[x][j][0], bh[x][j][1]);
                                    if (z == 1) mma_tf32(d[x][a], ph[a][j], bl[x][j][0], bl[x][j][1]);
                                    if (z == 2) mma_tf32(d[x][a], ph[a][j], bh[x][j][0], bh[x][j][1]);
                                }
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int a = 0; a < MT; ++a)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                o[a][jd + x][e] =
                                    fmaf(o[a][jd + x][e], corr[MODE == 0 ? 0 : (2 * a + (e >> 1)) % RI], d[x][a][e]);
                }
            } else {
                constexpr int PH = MODE == 0 ? 1 : 2;
                uint32_t P[MT][NTK / 2][PH][4];
#pragma unroll
                for (int a = 0; a < MT; ++a)
#pragma unroll
                    for (int k = 0; k < NTK / 2; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {          // tokens 16 k + 8 h + 2 t4 + {0, 1}
                            const float f = KV == SLATE_KV_Q8 ? 1.f : 32768.f;
                            const int j = 2 * k + h;
                            if (MODE == 0) {
                                split_f16(p[0][j][0] * f, p[0][j][1] * f, P[a][k][0][2 * h], P[a][k][0][2 * h + 1]);
                            } else {
                                split_f16(p[(2 * a) % RI][j][0] * f, p[(2 * a) % RI][j][1] * f, P[a][k][0][2 * h],
                                          P[a][k][PH - 1][2 * h]);
                                split_f16(p[(2 * a + 1) % RI][j][0] * f, p[(2 * a + 1) % RI][j][1] * f,
                                          P[a][k][0][2 * h + 1], P[a][k][PH - 1][2 * h + 1]);
                            }
                        }
                // 8 bits: one ldmatrix.x4.trans brings 16 dims of 32 tokens or 32 dims of 16; each
                // word holds dims (2g, 2g + 1) of two tokens: even dims are one output tile, odd the next
#pragma unroll
                for (int jd = 0; jd < NTD; jd += 2) {
                    float d[MT][2][4];
#pragma unroll
                    for (int a = 0; a < MT; ++a)
#pragma unroll
                        for (int x = 0; x < 2; ++x) d[a][x][0] = d[a][x][1] = d[a][x][2] = d[a][x][3] = 0.f;
                    if constexpr (KV == SLATE_KV_Q8) {
#pragma unroll
                        for (int k2 = 0; k2 < NTK / 4; ++k2) {
                            uint32_t r[4];
                            ldsm4t(vs_ + swz<KV, RB>(32 * k2 + lane, jd / 2), r);
#pragma unroll
                            for (int k = 0; k < 2; ++k)
#pragma unroll
                                for (int h = PH - 1; h >= 0; --h)
#pragma unroll
                                    for (int x = 0; x < 2; ++x) {
                                        const uint32_t b0 = x ? i8_f16<0x4341>(r[2 * k]) : i8_f16<0x4240>(r[2 * k]);
                                        const uint32_t b1 = x ? i8_f16<0x4341>(r[2 * k + 1]) : i8_f16<0x4240>(r[2 * k + 1]);
#pragma unroll
                                        for (int a = 0; a < MT; ++a) mma_f16(d[a][x], P[a][2 * k2 + k][h], b0, b1);
                                    }
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < NTK / 2; ++k) {
                            uint32_t r[4];
                            ldsm4t(vs_ + swz<KV, RB>(16 * k + ((lane >> 3) & 1) * 8 + (lane & 7), jd + (lane >> 4)), r);
#pragma unroll
                            for (int h = PH - 1; h >= 0; --h)
#pragma unroll
                                for (int x = 0; x < 2; ++x)
#pragma unroll
                                    for (int a = 0; a < MT; ++a) mma_f16(d[a][x], P[a][k][h], r[2 * x], r[2 * x + 1]);
                        }
                    }
#pragma unroll
                    for (int a = 0; a < MT; ++a)
#pragma unroll
                        for (int x = 0; x < 2; ++x)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                o[a][jd + x][e] = fmaf(o[a][jd + x][e], corr[MODE == 0 ? 0 : (2 * a + (e >> 1)) % RI], d[a][x][e]);
                }
            }
            __syncwarp();                              // the stage is read: it may be filled again
            issue(i + NS - 1);
        }
        cp_wait<0>();
        __syncthreads();                               // every warp's ring is drained: reuse it

        // ---- join the four warps: [MW][MR][HD + 2]
        float* mg = (float*)ring;
#pragma unroll
        for (int ri = 0; ri < RI; ++ri) {
            float* rec = mg + ((size_t)warp * MR + 8 * ri + g) * (HD + 2);
            const float of = KV == SLATE_KV_Q8    ? ex2(fminf(vtop[ri] - m[ri] - 15.f, 120.f))
                             : KV == SLATE_KV_F16 ? 0x1p-15f
                                                  : 1.f;
            float ls = l[ri];
            ls += __shfl_xor_sync(FULL, ls, 1);
            ls += __shfl_xor_sync(FULL, ls, 2);
            if (t4 == 0) {
                rec[0] = m[ri];
                rec[1] = ls;
            }
#pragma unroll
            for (int jd = 0; jd < NTD; ++jd)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = MODE == 0 ? o[0][jd][e] + o[0][jd][2 + e] : o[ri >> 1][jd][2 * (ri & 1) + e];
                    const int dd = KV == SLATE_KV_Q8 ? 16 * (jd / 2) + 2 * (2 * t4 + e) + (jd & 1) : 8 * jd + 2 * t4 + e;
                    rec[2 + dd] = x * of;
                }
        }
        __syncthreads();
        const bool whole = u0 == 0 && u1 == sq_.units;
        float* part = ws + (size_t)(2 * blockIdx.x + (seg ? 1 : 0)) * MR * (HD + 2);
        for (int e = tid; e < n_rows * HD; e += 32 * MW) {
            const int r = e / HD, d = e % HD;
            float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
            for (int w = 0; w < MW; ++w) M = fmaxf(M, mg[((size_t)w * MR + r) * (HD + 2)]);
#pragma unroll
            for (int w = 0; w < MW; ++w) {
                const float* rec = mg + ((size_t)w * MR + r) * (HD + 2);
                // a part without a maximum holds zeros, or NaN if it saw one
                const float f = rec[0] == -INFINITY ? 1.f : ex2(rec[0] - M);
                L = fmaf(rec[1], f, L);
                O = fmaf(rec[2 + d], f, O);
            }
            if (whole) {
                const int row = r_base + r;
                O = L == 0.f ? 0.f : O / L;
                out[(size_t)(sq_.r0 + row / G) * ld_out + (size_t)(kvh * G + row % G) * HD + d] = O;
                if (O != O) nan_words(ws, HD)[blockIdx.x] = 1;
            } else {
                float* rec = part + (size_t)r * (HD + 2);
                if (d == 0) {
                    rec[0] = M;
                    rec[1] = L;
                }
                rec[2 + d] = O;
            }
        }
    }
}

// Rows row0 + i of sequence s and a kv head, for each bit i of `which`, by a warp (of their dims, `blocks`).
template <int E>
__device__ __forceinline__ void rows_by_formula(const slate_kv_cache_t& c, int layer, const slate_tree_t& tr, int s, int kvh, int G, int row0,
                                                uint32_t which, uint32_t blocks, float* out, int ld_out, const float* q, int ld_q,
                                                float scale) {
    const Seq a = seq_of(c, tr, s, G, 1, 1);             // (read anew: the sums have no registers for it)
    for (; which; which &= which - 1) {
        const int row = row0 + __ffs(which) - 1, rr = a.r0 + row / G, hd = c.head_dim;
        const size_t head = (size_t)(kvh * G + row % G) * hd;
        row_by_formula<E>(row_job(c, layer, kvh, a.slot, a.ctx, a.n, __ldg(tr.mask + rr)), q + (size_t)rr * ld_q + head, scale,
                          out + (size_t)rr * ld_out + head, blocks);
    }
}

// Joins the partials of the cut items: a CTA a (sequence, kv head, `rpc` rows), W warps a row,
// each with every W-th record: lane i forms the weight of the warp's record i, then the lanes
// sum their dims over the records, F records in flight.  The loads' latency is what bounds it.
// A row that comes out as NaN, here or in the CTA that wrote it whole, is computed by the formula.
template <int HD, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W) attn_tree_join(
    const slate_kv_cache_t c, int layer, const slate_tree_t tr, int nq, int MR, int unit, int slack, int ctas, int rpc,
    float* __restrict__ out, int ld_out, const float* __restrict__ qs, int ld_q, float scale, const float* __restrict__ ws) {
    constexpr int E = HD / 32;                           // dims a lane: 2 or 4
    // records in flight: at head_dim 128 eight take more than the 72 registers (of a warp a row) that seven CTAs an SM
    // leave, and an eighth of the threads an SM with eight warps a row
    constexpr int F = HD == 128 ? 6 : 8;
    __shared__ PlanBuf buf;
    __shared__ float sm[W], sl[W], so[W][HD];
    const int nkv = c.n_kv_heads, G = nq / nkv, tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int chunks = (tr.max_nodes * G + rpc - 1) / rpc, s = blockIdx.x / chunks, kvh = blockIdx.y;
    // no early release: the next call's CTAs have to find the SMs empty, all of them at once
    Seq q;
    int64_t before;
    const int64_t total = plan_of(c, tr, G, MR, unit, slack, ctas, s, buf, q, before);
    const Cut cut(total, ctas);
    sb_grid_wait();        // the partials; before any return, so that the chain stays ordered
    const int row0 = blockIdx.x % chunks * rpc, w = W == 1 ? 0 : warp;
    uint32_t again = 0;                                  // the warp's rows that came out as NaN
    for (int row = row0 + (W == 1 ? warp : 0); row < min(row0 + rpc, q.n * G); row += W == 1 ? 4 : 1) {
        const int64_t first = before + (int64_t)(kvh * q.tiles + row / MR) * q.units;
        const int c0 = cut.owner(first), n = cut.owner(first + q.units - 1) - c0 + 1;
        const auto place = [&]() { return out + (size_t)(q.r0 + row / G) * ld_out + (size_t)(kvh * G + row % G) * HD; };
        bool nan = false;
        if (n == 1) {                                    // written by its CTA
            if (nan_words(ws, HD)[c0] && w < E) {
                const float* o = place();
                if (W == 1)
                    for (int k = 0; k < E; ++k) nan |= o[32 * k + lane] != o[32 * k + lane];
                else
                    nan = o[32 * w + lane] != o[32 * w + lane];
                if (__any_sync(FULL, nan)) again |= 1u << (row - row0);
            }
            continue;
        }
        // an item that begins inside its first CTA's range is that CTA's later segment
        const size_t rec = (size_t)MR * (HD + 2);
        const float* base = ws + (size_t)2 * c0 * rec + (size_t)(row % MR) * (HD + 2);
        const size_t late = cut.first(c0) < first ? rec : 0;
        float M = -INFINITY, L = 0.f, O[E];
        for (int i = w + W * lane; i < n; i += 32 * W) M = fmaxf(M, base[2 * i * rec + (i ? 0 : late)]);
        for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor_sync(FULL, M, x));
#pragma unroll
        for (int k = 0; k < E; ++k) O[k] = 0.f;
        for (int i0 = w; i0 < n; i0 += 32 * W) {
            float f = 0.f;
            if (i0 + W * lane < n) {
                const int i = i0 + W * lane;
                const float2 ml = *(const float2*)(base + 2 * i * rec + (i ? 0 : late));
                f = ml.x == -INFINITY ? 1.f : ex2(ml.x - M);
                L = fmaf(ml.y, f, L);
            }
            for (int j0 = 0; j0 < 32 && i0 + W * j0 < n; j0 += F) {
                float2 y[F][E / 2];
#pragma unroll
                for (int u = 0; u < F; ++u) {
                    const int i = i0 + W * (j0 + u);
                    if (i >= n) break;
#pragma unroll
                    for (int k = 0; k < E / 2; ++k)
                        y[u][k] = *(const float2*)(base + 2 * i * rec + (i ? 0 : late) + 2 + E * lane + 2 * k);
                }
#pragma unroll
                for (int u = 0; u < F; ++u) {
                    if (i0 + W * (j0 + u) >= n) break;
                    const float v = __shfl_sync(FULL, f, j0 + u);
#pragma unroll
                    for (int k = 0; k < E / 2; ++k) {
                        O[2 * k] = fmaf(y[u][k].x, v, O[2 * k]);
                        O[2 * k + 1] = fmaf(y[u][k].y, v, O[2 * k + 1]);
                    }
                }
            }
        }
        for (int x = 16; x; x >>= 1) L += __shfl_xor_sync(FULL, L, x);
        float* o = place();
        if (W == 1) {
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const float x = L == 0.f ? 0.f : O[k] / L;
                o[E * lane + k] = x;
                nan |= x != x;
            }
            if (__any_sync(FULL, nan)) again |= 1u << (row - row0);
            continue;
        }
        // (one row a CTA: nothing of a row before it is still read)
        if (lane == 0) {
            sm[w] = M;
            sl[w] = L;
        }
#pragma unroll
        for (int k = 0; k < E; ++k) so[w][E * lane + k] = O[k];
        __syncthreads();
        if (tid >= HD) return;
        M = -INFINITY, L = 0.f;
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) M = fmaxf(M, sm[i]);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float f = sm[i] == -INFINITY ? 1.f : ex2(sm[i] - M);
            L = fmaf(sl[i], f, L);
            x = fmaf(so[i][tid], f, x);
        }
        x = L == 0.f ? 0.f : x / L;
        o[tid] = x;
        if (__any_sync(FULL, x != x)) again = 1;         // (a warp: the dims that it wrote)
    }
    __syncwarp();                                        // the row's lanes change below
    if (again) rows_by_formula<E>(c, layer, tr, s, kvh, G, row0, again, W == 1 ? ~0u : 1u << warp, out, ld_out, qs, ld_q, scale);
}

template <int HD>
int join(const slate_kv_cache_t& c, int layer, const slate_tree_t& tr, int nq, int MR, int unit, int slack, int ctas, float* out,
         int ld_out, const float* q, int ld_q, float scale, float* ws, cudaStream_t st) {
    const int R = tr.max_nodes * (nq / c.n_kv_heads);
    // eight warps a row where an item, if long, is cut into eight records or more: one token over 3000
    // tokens of 8 heads 10.2 us against 12.9 with a warp a row, over 700 9.1 against 9.6 (whole calls; 16 nodes over
    // 100 tokens, which are not cut, 16.0 against 14.0); more items than that fill
    // the GPU with a warp a row
    if ((int64_t)tr.n_seq * c.n_kv_heads * ((R + MR - 1) / MR) * 8 <= ctas)
        return sb_cuda_check(sb_launch_pdl(attn_tree_join<HD, 8>, dim3((unsigned)(tr.n_seq * R), (unsigned)c.n_kv_heads), dim3(256), 0,
                                           st, c, layer, tr, nq, MR, unit, slack, ctas, 1, out, ld_out, q, ld_q, scale, ws),
                             "attention_tree join");
    const int rpc = R >= 128 ? 16 : 4;
    const dim3 grid((unsigned)(tr.n_seq * ((R + rpc - 1) / rpc)), (unsigned)c.n_kv_heads);
    return sb_cuda_check(sb_launch_pdl(attn_tree_join<HD, 1>, grid, dim3(128), 0, st, c, layer, tr, nq, MR, unit, slack, ctas, rpc, out,
                                       ld_out, q, ld_q, scale, ws),
                         "attention_tree join");
}
template <int KV, int HD, int MODE>
int launch_mma(const slate_kv_cache_t& c, int layer, const slate_tree_t& tr, int nq, float* out,
               int ld_out, const float* q, int ld_q, float scale, float* ws, cudaStream_t st) {
    using S = Shape<KV, HD, MODE>;
    const auto k = attn_tree_mma<KV, HD, MODE>;
    static unsigned long long ready = 0;
    const cudaError_t may = sb_allow_smem((const void*)k, S::SMEM, &ready);
    if (may != cudaSuccess) return sb_cuda_check(may, "attention_tree shared memory");
    const int rc = sb_cuda_check(sb_launch_pdl(k, dim3(S::CPS * SMS), dim3(32 * MW), S::SMEM, st, c, layer, tr, nq, out,
                                               ld_out, q, ld_q, scale, ws),
                                 "attention_tree");
    return rc ? rc : join<HD>(c, layer, tr, nq, S::MR, UNIT, S::SLACK, S::CPS * SMS, out, ld_out, q, ld_q, scale, ws, st);
}
template <int KV, int HD>
int launch_mode(const slate_kv_cache_t& c, int layer, const slate_tree_t& tr, int nq, float* out,
                int ld_out, const float* q, int ld_q, float scale, float* ws, cudaStream_t st) {
    const int M = tr.max_nodes * (nq / c.n_kv_heads);
    // attn_tree_mma with 32 rows against attn_tree_tc, 16 sequences of 8 nodes x 4 heads: head_dim 128 over
    // 1000 tokens of 8 bits 37.5 and 32.3 us, over 8000 110 and 103, of f16 103 and 86; head_dim 64 over 8000 of
    // f16 59.6 and 69.7, of 8 bits 62 and 89
    constexpr int few = KV != SLATE_KV_F32 && HD == 128 ? 16 : 32;
    if (M <= 8) return launch_mma<KV, HD, 0>(c, layer, tr, nq, out, ld_out, q, ld_q, scale, ws, st);
    if (M <= 16) return launch_mma<KV, HD, 1>(c, layer, tr, nq, out, ld_out, q, ld_q, scale, ws, st);
    if constexpr (few > 16)
        if (KV == SLATE_KV_F32 || M <= few)
            return launch_mma<KV, HD, 2>(c, layer, tr, nq, out, ld_out, q, ld_q, scale, ws, st);
    const int rc = attend_tc(c, layer, tr, nq, out, ld_out, q, ld_q, scale, ws, st);
    return rc ? rc : join<HD>(c, layer, tr, nq, TC_ROWS, TC_UNIT, TC_SLACK, SMS, out, ld_out, q, ld_q, scale, ws, st);
}
bool takes_mma(const slate_kv_cache_t* c) { return c->head_dim == 64 || c->head_dim == 128; }

}  // namespace

extern "C" size_t slate_cuda_attention_tree_workspace(const slate_kv_cache_t* cache, int n_heads,
                                                      int n_seq, int rows, int max_nodes) {
    if (!cache || n_heads < 1 || n_seq < 1 || rows < 0 || max_nodes < 1) return 0;
    // two partials for each CTA: 148 of 128 rows, or 3 * 148 of 8, 2 * 148 of 32 at most; a word for each
    return takes_mma(cache) ? 4 * (partial_floats(cache->head_dim) + MAX_CTAS) : 16;
}

extern "C" int slate_cuda_attention_tree(const slate_kv_cache_t* cache, int layer,
                                         const slate_tree_t* tree, int n_heads, float* out,
                                         int ld_out, const float* q, int ld_q, float scale, void* ws,
                                         size_t ws_bytes, void* stream) {
    if (sb_kv_check(cache, "attention_tree") || sb_tree_check(tree, "attention_tree")) return -1;
    const int hd = cache->head_dim;
    if (layer < 0 || layer >= cache->n_layers || n_heads < 1 || n_heads % cache->n_kv_heads ||
        n_heads > 65535 || (int64_t)tree->n_seq * tree->max_nodes * n_heads > 0x7fffffff || !out || !q ||
        ld_out < n_heads * hd || ld_q < n_heads * hd ||
        !(fabsf(scale) < INFINITY)) {
        sb_set_error("attention_tree: bad arguments");
        return -1;
    }
    if (!ws || ((uintptr_t)ws & 15) ||
        ws_bytes < slate_cuda_attention_tree_workspace(cache, n_heads, tree->n_seq, tree->rows,
                                                       tree->max_nodes)) {
        sb_set_error("attention_tree: workspace of %zu bytes is too small or not aligned", ws_bytes);
        return -1;
    }
    if (tree->rows == 0) return 0;
    if (takes_mma(cache)) {
        const auto f = hd == 64 ? cache->kv_dtype == SLATE_KV_F32   ? launch_mode<SLATE_KV_F32, 64>
                                  : cache->kv_dtype == SLATE_KV_F16 ? launch_mode<SLATE_KV_F16, 64>
                                                                    : launch_mode<SLATE_KV_Q8, 64>
                       : cache->kv_dtype == SLATE_KV_F32   ? launch_mode<SLATE_KV_F32, 128>
                       : cache->kv_dtype == SLATE_KV_F16 ? launch_mode<SLATE_KV_F16, 128>
                                                         : launch_mode<SLATE_KV_Q8, 128>;
        return f(*cache, layer, *tree, n_heads, out, ld_out, q, ld_q, scale, (float*)ws,
                 (cudaStream_t)stream);
    }
    return sb_cuda_check(sb_launch_pdl(attn_tree_rows, dim3((unsigned)tree->rows, (unsigned)n_heads), dim3(32 * NW), 0, (cudaStream_t)stream,
                                       *cache, layer, *tree, n_heads, out, ld_out, q, ld_q, scale),
                         "attention_tree");
}
