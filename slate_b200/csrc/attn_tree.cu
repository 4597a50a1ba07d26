// attn_tree.cu -- attention of token-tree nodes over the paged cache
// (slate_cuda_attention_tree): for row i of a sequence, kv head h and each query
// head of its group
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - max_j),
// over j < ctx (the context) and the nodes j that bit j - ctx of the row's mask
// names.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "sb_internal.h"
#include "sb_kernels.h"
#include "sb_kv.h"

namespace {

constexpr unsigned FULL = 0xffffffffu;

__device__ __forceinline__ float element(const unsigned char* blk, int kv_dtype, int at) {
    return kv_dtype == SLATE_KV_F32   ? ((const float*)blk)[at]
           : kv_dtype == SLATE_KV_F16 ? __half2float(((const __half*)blk)[at])
                                      : (float)((const int8_t*)blk)[SB_Q8_SCALES + at];
}

// Any head_dim: one CTA per (row, query head), its four warps take pages in
// turn.  A page's scores are formed first, then its maximum joins the running
// one and its sum of p v is formed by itself before it joins the running sum,
// which keeps the f32 sums of long contexts two levels deep.  Keys that the row
// does not see are skipped, so nothing they hold can reach it.
constexpr int NW = 4;
__global__ void __launch_bounds__(32 * NW) attn_tree_rows(
    const slate_kv_cache_t c, int layer, const slate_tree_t tr, int nq, float* __restrict__ out,
    int ld_out, const float* __restrict__ q, int ld_q, float scale) {
    __shared__ float sm[NW], sl[NW], so[NW][256];
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
    const int n = min(max(min(tr.row_off[lo + 1], tr.rows) - r0, 0), SLATE_TREE_MAX_NODES);
    const bool in = row >= r0 && row < r0 + n;
    const uint64_t mask = in ? tr.mask[row] : 0;
    const int end = in ? ctx + n : 0;
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
                if (lane + 32 * i < hd) s = fmaf(qv[i], element(kb, c.kv_dtype, t * hd + lane + 32 * i), s);
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(FULL, s, x);
            if (c.kv_dtype == SLATE_KV_Q8) s *= ((const float*)kb)[t];
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
                    po[i] = fmaf(pt, element(vb, c.kv_dtype, t * hd + lane + 32 * i), po[i]);
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
    for (int d = tid; d < hd; d += 32 * NW) {
        float O = 0.f;
        for (int w = 0; w < NW; ++w) O += so[w][d] * (sm[w] == -INFINITY ? 1.f : expf(sm[w] - M));
        out[(size_t)row * ld_out + (size_t)h * hd + d] = L == 0.f ? 0.f : O / L;
    }
}

}  // namespace

extern "C" size_t slate_cuda_attention_tree_workspace(const slate_kv_cache_t* cache, int n_heads,
                                                      int n_seq, int rows, int max_nodes) {
    if (!cache || n_heads < 1 || n_seq < 1 || rows < 0 || max_nodes < 1) return 0;
    return 16;
}

extern "C" int slate_cuda_attention_tree(const slate_kv_cache_t* cache, int layer,
                                         const slate_tree_t* tree, int n_heads, float* out,
                                         int ld_out, const float* q, int ld_q, float scale, void* ws,
                                         size_t ws_bytes, void* stream) {
    if (sb_kv_check(cache, "attention_tree") || sb_tree_check(tree, "attention_tree")) return -1;
    const int hd = cache->head_dim;
    if (layer < 0 || layer >= cache->n_layers || n_heads < 1 || n_heads % cache->n_kv_heads ||
        n_heads > 65535 || !out || !q || ld_out < n_heads * hd || ld_q < n_heads * hd ||
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
    attn_tree_rows<<<dim3((unsigned)tree->rows, (unsigned)n_heads), 32 * NW, 0,
                     (cudaStream_t)stream>>>(*cache, layer, *tree, n_heads, out, ld_out, q, ld_q, scale);
    return sb_cuda_check(cudaGetLastError(), "attention_tree");
}
