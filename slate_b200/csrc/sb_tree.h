/*
 * sb_tree.h -- what the tree-attention kernels share (attn_tree.cu,
 * attn_tree_tc.cu; internal, CUDA C++ only): the cut of the work over the CTAs,
 * the splitting of operands and the rows that halves cannot form.
 */
#ifndef SB_TREE_H
#define SB_TREE_H

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "sb_kernels.h"
#include "sb_kv.h"

namespace sb_tree {

constexpr unsigned FULL = 0xffffffffu;
constexpr int SMS = 148;

// ---------------------------------------------------------------- shared plan
// The cache's tokens are dealt out evenly: an item is one (sequence, kv head, tile
// of MR rows), its work ceil(tokens / unit) units; the items' units in order are
// cut into as many equal ranges as there are CTAs.  A CTA that holds the whole of
// an item writes its output; of a cut item each CTA leaves a partial (max, sum, o)
// for attn_tree_join.  Contexts of any lengths thereby load every SM alike.  With few items the
// unit grows (below), so that a CTA has one range of one item and starts once.
struct Seq {
    int s, r0, n, slot, ctx;      // rows r0 .. r0 + n - 1
    int tiles, units;             // row tiles a head; units an item
};
__device__ __forceinline__ Seq seq_of(const slate_kv_cache_t& c, const slate_tree_t& tr, int s,
                                      int G, int MR, int unit) {
    Seq q;
    q.s = s;
    q.r0 = max(__ldg(tr.row_off + s), 0);
    q.n = min(max(min(__ldg(tr.row_off + s + 1), tr.rows) - q.r0, 0), tr.max_nodes);
    q.slot = __ldg(tr.slot + s);
    q.ctx = min(max(__ldg(tr.ctx + s), 0), c.max_pages * SB_PAGE_TOKENS);
    q.tiles = (q.n * G + MR - 1) / MR;
    q.units = (q.ctx + q.n + unit - 1) / unit;
    return q;
}
__device__ __forceinline__ int64_t seq_units(const Seq& q, int nkv) {
    return (int64_t)q.tiles * nkv * q.units;
}

// Block-wide: the units of all sequences, those before this thread's sequences
// (`per` consecutive ones a thread, the first 128 threads).
struct PlanBuf {
    int64_t sum[4];
    int64_t before;
    int s;
};
__device__ __forceinline__ int64_t plan_total(const slate_kv_cache_t& c, const slate_tree_t& tr, int G, int MR, int unit,
                                              PlanBuf& buf, int64_t& before) {
    const int per = (tr.n_seq + 127) / 128, tid = threadIdx.x;
    int64_t mine = 0;
    for (int s = tid * per; s < min(tr.n_seq, (tid + 1) * per); ++s)
        mine += seq_units(seq_of(c, tr, s, G, MR, unit), c.n_kv_heads);
    int64_t incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(FULL, incl, o);
        if ((tid & 31) >= o) incl += x;
    }
    if ((tid & 31) == 31 && tid < 128) buf.sum[tid / 32] = incl;
    __syncthreads();
    int64_t base = 0, total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < tid / 32) base += buf.sum[w];
        total += buf.sum[w];
    }
    before = base + incl - mine;
    return total;
}
// The sequence that holds unit `at` and the units before it.
__device__ __forceinline__ int plan_find(const slate_kv_cache_t& c, const slate_tree_t& tr, int G, int MR, int unit,
                                         PlanBuf& buf, int64_t before, int64_t at, int64_t& seq_before) {
    const int per = (tr.n_seq + 127) / 128, tid = threadIdx.x;
    int64_t b = before;
    for (int s = tid * per; s < min(tr.n_seq, (tid + 1) * per) && b <= at; ++s) {
        const int64_t u = seq_units(seq_of(c, tr, s, G, MR, unit), c.n_kv_heads);
        if (at < b + u) {
            buf.s = s;
            buf.before = b;
        }
        b += u;
    }
    __syncthreads();
    seq_before = buf.before;
    return buf.s;
}
// The cut of `total` units over the C CTAs that have work: the first `more` hold
// `each` + 1 units, the others `each`.
struct Cut {
    int C, more;
    int64_t each;
    __device__ Cut(int64_t total, int ctas) {
        C = (int)min((int64_t)ctas, total);
        // 32-bit division where it does (the usual case): a 64-bit one takes a microsecond
        each = total < 0x7fffffff ? (int64_t)((uint32_t)total / (uint32_t)max(C, 1)) : total / max(C, 1);
        more = (int)(total - each * C);
    }
    __device__ int64_t first(int i) const { return each * i + min(i, more); }
    __device__ int owner(int64_t x) const {
        const int64_t big = (each + 1) * more;
        if (x < big) return (int)(x < 0x7fffffff ? (uint32_t)x / (uint32_t)(each + 1) : x / (each + 1));
        x -= big;
        return more + (int)(x < 0x7fffffff ? (uint32_t)x / (uint32_t)each : x / each);
    }
};
// The item that holds unit `rel` of a sequence, and the unit's place in it.
__device__ __forceinline__ int item_of(int64_t rel, int units, int& u0) {
    const int item = (int)(rel < 0x7fffffff ? (uint32_t)rel / (uint32_t)units : rel / units);
    u0 = (int)(rel - (int64_t)item * units);
    return item;
}

// Where a CTA begins: its units [at, stop), the sequence that holds `at`, the units before
// that sequence.  False for a CTA without work.  Up to 32 sequences (the calls where the
// microsecond counts) every warp finds it alone, a lane a sequence, without a barrier.
struct Start {
    int64_t at, stop, seq_before;
    Seq sq;
};
__device__ __forceinline__ Seq seq_from(const Seq& q, int lane) {
    Seq r;
    r.s = lane;
    r.r0 = __shfl_sync(FULL, q.r0, lane);
    r.n = __shfl_sync(FULL, q.n, lane);
    r.slot = __shfl_sync(FULL, q.slot, lane);
    r.ctx = __shfl_sync(FULL, q.ctx, lane);
    r.tiles = __shfl_sync(FULL, q.tiles, lane);
    r.units = __shfl_sync(FULL, q.units, lane);
    return r;
}
// A second range costs a CTA about `slack` units (q, the first tile's latency, O): a unit of T
// units, T up to `slack` more than the even share, is taken if that leaves a CTA one range.
// 8 x 16 nodes over 8000 tokens of f16: 51 us against 58 with slack 0, of 8 bits 60 against 68 (slack 4; 16 makes 20000
// tokens slower, 136 against 127).
__device__ __forceinline__ int64_t plan_warp(const slate_kv_cache_t& c, const slate_tree_t& tr, int G, int MR,
                                             int& unit, int slack, int ctas, Seq& q, int64_t& before) {
    const int lane = threadIdx.x & 31;
    q = seq_of(c, tr, min(lane, tr.n_seq - 1), G, MR, unit);
    int64_t mine = lane < tr.n_seq ? seq_units(q, c.n_kv_heads) : 0;
    const uint32_t sum = __reduce_add_sync(FULL, (uint32_t)min(mine, (int64_t)1 << 26));
    if (sum > (uint32_t)ctas) {
        const uint32_t items = mine ? min((uint32_t)(q.tiles * c.n_kv_heads), 1000u) : 0;
        const uint32_t even = (sum + ctas - 1) / ctas;
        for (uint32_t T = even; T <= even + slack; ++T) {
            const uint32_t n = (q.units + T - 1) / T;
            if (__reduce_add_sync(FULL, items * min(n, 1000u)) > (uint32_t)ctas) continue;
            unit *= T;
            q.units = (int)n;
            mine = (int64_t)items * n;
            break;
        }
    }
    int64_t incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(FULL, incl, o);
        if (lane >= o) incl += x;
    }
    before = incl - mine;
    return __shfl_sync(FULL, incl, 31);
}
__device__ __forceinline__ bool plan_start(const slate_kv_cache_t& c, const slate_tree_t& tr, int G, int MR, int& unit,
                                           int slack, int ctas, PlanBuf& buf, Start& st) {
    int64_t before;
    if (tr.n_seq <= 32) {
        Seq q;
        const int64_t total = plan_warp(c, tr, G, MR, unit, slack, ctas, q, before);
        const Cut cut(total, ctas);
        if ((int)blockIdx.x >= cut.C) return false;
        st.at = cut.first(blockIdx.x);
        st.stop = cut.first(blockIdx.x + 1);
        // the last sequence that begins at or before `at` and has units
        const unsigned hit = __ballot_sync(FULL, (int)(threadIdx.x & 31) < tr.n_seq && before <= st.at && seq_units(q, c.n_kv_heads) > 0);
        const int s = 31 - __clz(hit);
        st.seq_before = __shfl_sync(FULL, before, s);
        st.sq = seq_from(q, s);
        return true;
    }
    const int64_t total = plan_total(c, tr, G, MR, unit, buf, before);
    const Cut cut(total, ctas);
    if ((int)blockIdx.x >= cut.C) return false;
    st.at = cut.first(blockIdx.x);
    st.stop = cut.first(blockIdx.x + 1);
    const int s = plan_find(c, tr, G, MR, unit, buf, before, st.at, st.seq_before);
    st.sq = seq_of(c, tr, s, G, MR, unit);
    return true;
}
// Sequence s, the units before it, and the total.
__device__ __forceinline__ int64_t plan_of(const slate_kv_cache_t& c, const slate_tree_t& tr, int G, int MR, int unit,
                                           int slack, int ctas, int s, PlanBuf& buf, Seq& sq, int64_t& before) {
    if (tr.n_seq <= 32) {
        Seq q;
        int64_t b;
        const int64_t total = plan_warp(c, tr, G, MR, unit, slack, ctas, q, b);
        sq = seq_from(q, s);
        before = __shfl_sync(FULL, b, s);
        return total;
    }
    const int64_t total = plan_total(c, tr, G, MR, unit, buf, before);
    const int per = (tr.n_seq + 127) / 128, tid = threadIdx.x;
    if (tid == s / per) {          // from the thread that counted them
        for (int x = tid * per; x < s; ++x) before += seq_units(seq_of(c, tr, x, G, MR, unit), c.n_kv_heads);
        buf.before = before;
    }
    __syncthreads();
    before = buf.before;
    sq = seq_of(c, tr, s, G, MR, unit);
    return total;
}

__device__ __forceinline__ uint32_t su32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
// 16 bytes global -> shared; 0 bytes read and zeros written where !ok.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two values as f16 pairs: x = hi + lo
__device__ __forceinline__ void split_f16(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 b = __half22float2(h);
    const float2 r = __fadd2_rn(make_float2(x0, x1), make_float2(-b.x, -b.y));
    const __half2 l = __floats2half2_rn(r.x, r.y);
    hi = *(const uint32_t*)&h;
    lo = *(const uint32_t*)&l;
}
// Two of the four int8 of w as exact f16: the byte with its sign bit turned is
// u = x + 128; 0x6400 | u is the f16 1024 + u; minus 1152 leaves x.
template <int SEL>
__device__ __forceinline__ uint32_t i8_f16(uint32_t w) {
    const uint32_t p = __byte_perm(w ^ 0x80808080u, 0x64646464u, SEL);
    const __half2 h = __hsub2(*(const __half2*)&p, __floats2half2_rn(1152.f, 1152.f));
    return *(const uint32_t*)&h;
}

// An 8-bit key's infinite scale as NaN: its row holds infinities and, from zeros, NaN.
__device__ __forceinline__ float no_inf(float x) { return fmaf(0.f, x, x); }

// ---------------------------------------------------------------- rows by the formula itself
// Products of halves know no infinities (hi * inf + lo * inf, lo of either sign or 0, is NaN where q * inf is not),
// and a sum of halves neither.  So whatever gave NaN is computed again here, a warp a row, in f32 with sums in
// f64: a key of score -inf is as if not seen; one of +inf or NaN makes the row NaN; an infinity or NaN in v of a
// key that is seen makes that dim it, whatever the key's weight.  Rows without such values never come here.
struct RowJob {
    const unsigned char* pool;       // block of (layer, page 0, K, kv head)
    size_t page_step, kv_step;
    const int32_t* pages;            // of the slot, `last` of them
    int last, n_pages, hd, kv_dtype, ctx, n;
    uint64_t mask;
};
__device__ __forceinline__ RowJob row_job(const slate_kv_cache_t& c, int layer, int kvh, int slot, int ctx, int n, uint64_t mask) {
    RowJob j;
    j.pool = sb_kv_block(c, layer, 0, 0, kvh);
    j.kv_step = (size_t)c.n_kv_heads * sb_kv_block_bytes(c.kv_dtype, c.head_dim);
    j.page_step = 2 * j.kv_step;
    const bool in = slot >= 0 && slot < c.n_slots;
    j.pages = c.page_table + (in ? (size_t)slot * c.max_pages : 0);
    j.last = in ? min(c.max_pages, (ctx + n + SB_PAGE_TOKENS - 1) / SB_PAGE_TOKENS) : 0;
    j.n_pages = (int)c.n_pages;
    j.hd = c.head_dim;
    j.kv_dtype = c.kv_dtype;
    j.ctx = ctx;
    j.n = n;
    j.mask = mask;
    return j;
}
__device__ __forceinline__ float kv_element(const unsigned char* blk, int kv_dtype, int at) {
    return kv_dtype == SLATE_KV_F32   ? ((const float*)blk)[at]
           : kv_dtype == SLATE_KV_F16 ? __half2float(((const __half*)blk)[at])
                                      : (float)((const int8_t*)blk)[SB_Q8_SCALES + at];
}
// E: dims a lane, head_dim up to 32 E; writes the blocks of 32 dims that `blocks` has bits for
template <int E>
__device__ __forceinline__ void row_by_formula(const RowJob& j, const float* q, float scale, float* out, uint32_t blocks = ~0u) {
    const int lane = threadIdx.x & 31;
    const bool q8 = j.kv_dtype == SLATE_KV_Q8;
    float qv[E], top = -INFINITY;
    double o[E], l = 0.;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        qv[i] = lane + 32 * i < j.hd ? q[lane + 32 * i] * scale : 0.f;
        o[i] = 0.;
        nan |= qv[i] != qv[i];
    }
    nan = __any_sync(FULL, nan);
#pragma unroll 1
    for (uint32_t x = 0, len = 16u * j.last; x < 2 * len && !nan; ++x) {       // the maximum, then the sums
        const bool sums = x >= len;
        const int at = sums ? x - len : x, page = __ldg(j.pages + at / 16), node = at - j.ctx;
        if (page < 0 || page >= j.n_pages || node >= j.n || (node >= 0 && !(j.mask >> node & 1))) continue;
        const unsigned char *kb = j.pool + page * j.page_step, *vb = kb + j.kv_step;
        const int t = at % 16;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (lane + 32 * i < j.hd) s = fmaf(qv[i], kv_element(kb, j.kv_dtype, t * j.hd + lane + 32 * i), s);
        for (int y = 16; y; y >>= 1) s += __shfl_xor_sync(FULL, s, y);
        if (q8) s *= no_inf(((const float*)kb)[t]);
        if (s == -INFINITY) continue;
        nan = !(s < INFINITY);
        if (!sums) {
            top = fmaxf(top, s);
            continue;
        }
        const float p = expf(s - top), vs = q8 ? ((const float*)vb)[t] : 1.f;
        l += p;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (lane + 32 * i < j.hd) {
                const float v = kv_element(vb, j.kv_dtype, t * j.hd + lane + 32 * i) * vs;
                o[i] += (double)(fabsf(v) < INFINITY ? p : 1.f) * v;   // (an infinity is one whatever its weight)
            }
    }
    const float inv = l == 0. ? 0.f : 1.f / (float)l;
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (lane + 32 * i < j.hd && blocks >> i & 1) out[lane + 32 * i] = nan ? NAN : (float)(o[i] * inv);
}

// attn_tree_tc.cu: rows in tiles of TC_ROWS, units of TC_UNIT tokens, SMS CTAs; two
// partials of TC_ROWS x (head_dim + 2) floats for each in ws.  Behind the partials, a word a CTA: some row that it
// wrote whole holds NaN (attn_tree_join looks for it).
constexpr int TC_ROWS = 128, TC_UNIT = 128, TC_SLACK = 4, MAX_CTAS = 3 * SMS;
__host__ __device__ constexpr size_t partial_floats(int hd) { return (size_t)2 * SMS * TC_ROWS * (hd + 2); }
__device__ __forceinline__ int* nan_words(float* ws, int hd) { return (int*)(ws + partial_floats(hd)); }
__device__ __forceinline__ const int* nan_words(const float* ws, int hd) { return (const int*)(ws + partial_floats(hd)); }
int attend_tc(const slate_kv_cache_t& c, int layer, const slate_tree_t& tr, int nq, float* out, int ld_out,
              const float* q, int ld_q, float scale, float* ws, cudaStream_t st);

}  // namespace sb_tree

#endif
