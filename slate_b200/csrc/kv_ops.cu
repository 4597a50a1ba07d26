// kv_ops.cu -- the cache operators that move rows: rotary append, read-back,
// acceptance of a drafted tree with the compaction of its path.  Interfaces and
// the 8-bit rule: include/slate_cuda.h.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "sb_internal.h"
#include "sb_kernels.h"
#include "sb_kv.h"

namespace {

constexpr unsigned FULL = 0xffffffffu;

// One warp per (row, head): heads [0, nq) are query heads, then key heads, then
// value heads.  Each product and sum is rounded by itself (no fused multiply-
// add), so that an element next to a rounding boundary of the 8-bit grid falls
// on the side that the plain f32 formula gives.
__global__ void __launch_bounds__(256) rope_append_kernel(
    const slate_kv_cache_t c, int layer, const slate_rope_t rope, int rows, int nq,
    float* __restrict__ q_out, int ld_qo, const float* q, int ld_q, const float* __restrict__ k,
    int ld_k, const float* __restrict__ v, int ld_v, const int32_t* __restrict__ row_slot,
    const int32_t* __restrict__ row_index, const int32_t* __restrict__ row_pos) {
    const int lane = threadIdx.x & 31, hd = c.head_dim, nkv = c.n_kv_heads;
    const int heads = nq + 2 * nkv, half = rope.rot_dim / 2;
    const int64_t w = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (w >= (int64_t)rows * heads) return;
    const int r = (int)(w / heads), h = (int)(w % heads);
    const int index = row_index[r], pos = row_pos[r];
    if (index < 0 || pos < 0 || pos >= rope.n_pos) return;
    const float* x = h < nq ? q + (size_t)r * ld_q + (size_t)h * hd
                   : h < nq + nkv ? k + (size_t)r * ld_k + (size_t)(h - nq) * hd
                                  : v + (size_t)r * ld_v + (size_t)(h - nq - nkv) * hd;
    float y[8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        y[i] = 0.f;
        if (d < hd) {
            y[i] = x[d];
            if (d < rope.rot_dim && h < nq + nkv) {
                const bool inter = rope.layout == SLATE_ROPE_INTERLEAVED;
                const int j = inter ? d / 2 : d % half;
                const bool second = inter ? d & 1 : d >= half;
                const float o = x[inter ? d ^ 1 : second ? d - half : d + half];
                const float cs = rope.cos[(size_t)pos * half + j], sn = rope.sin[(size_t)pos * half + j];
                y[i] = second ? __fadd_rn(__fmul_rn(o, sn), __fmul_rn(y[i], cs))
                              : __fsub_rn(__fmul_rn(y[i], cs), __fmul_rn(o, sn));
            }
            top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);   // NaN above infinity above numbers
        }
    }
    __syncwarp();                       // q_out may be q: the pairs are read before any is written
    if (h < nq) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd) q_out[(size_t)r * ld_qo + (size_t)h * hd + lane + 32 * i] = y[i];
        return;
    }
    const int page = sb_kv_page(c, row_slot[r], index);
    if (page < 0) return;
    const int t = index % SB_PAGE_TOKENS, hk = (h - nq) % nkv;
    unsigned char* blk = sb_kv_block(c, layer, page, (h - nq) / nkv, hk);
    if (c.kv_dtype != SLATE_KV_Q8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = lane + 32 * i;
            if (d >= hd) break;
            if (c.kv_dtype == SLATE_KV_F32) ((float*)blk)[t * hd + d] = y[i];
            else ((__half*)blk)[t * hd + d] = __float2half_rn(y[i]);
        }
        return;
    }
    const float scale = __fmul_rn(__uint_as_float(__reduce_max_sync(FULL, top)), (float)(1.0 / 127.0));
    const bool plain = scale > 0.f && scale < INFINITY;
    if (lane == 0) ((float*)blk)[t] = scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < hd)
            ((int8_t*)blk)[SB_Q8_SCALES + t * hd + d] =
                plain ? (int8_t)fminf(fmaxf(rintf(__fdiv_rn(y[i], scale)), -127.f), 127.f) : 0;
    }
}

// One warp per (layer, row, K|V, head).
template <typename OT>
__global__ void __launch_bounds__(256) kv_read_kernel(
    const slate_kv_cache_t c, int layer0, int n_layers, int rows,
    const int32_t* __restrict__ row_slot, const int32_t* __restrict__ row_index,
    OT* __restrict__ K, OT* __restrict__ V) {
    const int lane = threadIdx.x & 31, hd = c.head_dim, nkv = c.n_kv_heads;
    int64_t w = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (w >= (int64_t)n_layers * rows * 2 * nkv) return;
    const int h = (int)(w % nkv);
    w /= nkv;
    const int which = (int)(w & 1);
    w >>= 1;                                             // layer * rows + row
    const int r = (int)(w % rows), layer = layer0 + (int)(w / rows);
    const int index = row_index[r], page = sb_kv_page(c, row_slot[r], index);
    const int t = index % SB_PAGE_TOKENS;
    const unsigned char* blk = page < 0 ? nullptr : sb_kv_block(c, layer, page, which, h);
    OT* o = (which ? V : K) + ((size_t)w * nkv + h) * hd;
    const float scale = blk && c.kv_dtype == SLATE_KV_Q8 ? ((const float*)blk)[t] : 0.f;
    for (int d = lane; d < hd; d += 32) {
        float x = 0.f;
        if (blk)
            x = c.kv_dtype == SLATE_KV_F32   ? ((const float*)blk)[t * hd + d]
                : c.kv_dtype == SLATE_KV_F16 ? __half2float(((const __half*)blk)[t * hd + d])
                                             : (float)((const int8_t*)blk)[SB_Q8_SCALES + t * hd + d] * scale;
        o[d] = (OT)x;
    }
}

// One CTA per (sequence, layer): the path is found by every CTA of a sequence
// (64 nodes, two warp votes), then each thread moves 16-byte (or 4-byte) columns
// of the path's rows in order.  The path's indexes rise, so the k-th row's place
// (k) never lies at or behind a later row's source (path[k'] >= k' > k): moving
// in order never overwrites what is still to be read.
constexpr int AT = 256;
template <typename U>
__device__ void move_rows(const slate_kv_cache_t& c, int layer, int n, const int* src_page,
                          const int* src_t, const int* dst_page, const int* dst_t) {
    const int rb = sb_kv_row_bytes(c.kv_dtype, c.head_dim), cols = rb / (int)sizeof(U);
    const int head_off = c.kv_dtype == SLATE_KV_Q8 ? SB_Q8_SCALES : 0;
    for (int e = threadIdx.x; e < 2 * c.n_kv_heads * cols; e += AT) {
        const int col = e % cols, hw = e / cols, which = hw / c.n_kv_heads, h = hw % c.n_kv_heads;
        for (int k = 0; k < n; ++k) {
            if (src_page[k] < 0 || dst_page[k] < 0) continue;
            const U x = *(const U*)(sb_kv_block(c, layer, src_page[k], which, h) + head_off +
                                    src_t[k] * rb + col * sizeof(U));
            *(U*)(sb_kv_block(c, layer, dst_page[k], which, h) + head_off + dst_t[k] * rb +
                  col * sizeof(U)) = x;
        }
    }
}

__global__ void __launch_bounds__(AT) tree_accept_kernel(
    const slate_kv_cache_t c, const slate_tree_t tr, const int32_t* __restrict__ parent,
    const int32_t* __restrict__ token, const int32_t* __restrict__ target, int32_t* out_count,
    int32_t* out_node, int32_t* out_token) {
    __shared__ uint32_t ok_s[2];
    __shared__ int best_s[2];
    __shared__ int src_page[64], src_t[64], dst_page[64], dst_t[64];
    const int s = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x;
    const int r0 = max(tr.row_off[s], 0), r1 = min(tr.row_off[s + 1], tr.rows);
    const int n = min(max(r1 - r0, 0), SLATE_TREE_MAX_NODES);
    const uint64_t live = n == 64 ? ~0ull : (1ull << n) - 1;
    const int slot = tr.slot[s], ctx = min(max(tr.ctx[s], 0), c.max_pages * SB_PAGE_TOKENS);
    uint64_t m = 0;
    if (tid < 64) {
        bool ok = false;
        if (tid < n) {
            const int p = parent[r0 + tid];
            m = tr.mask[r0 + tid] & live;
            ok = p < 0 || (p < n && token[r0 + tid] == target[r0 + p]);
        }
        const uint32_t b = __ballot_sync(FULL, ok);
        if ((tid & 31) == 0) ok_s[tid >> 5] = b;
    }
    __syncthreads();
    if (tid < 64) {
        const uint64_t ok = ok_s[0] | (uint64_t)ok_s[1] << 32;
        // deepest first, then the lowest index
        const int score = tid < n && !(m & ~ok) ? __popcll(m) * 64 + 63 - tid : 0;
        const int b = (int)__reduce_max_sync(FULL, (unsigned)score);
        if ((tid & 31) == 0) best_s[tid >> 5] = b;
    }
    __syncthreads();
    const int best = max(best_s[0], best_s[1]);
    const uint64_t path = best ? tr.mask[r0 + 63 - best % 64] & live : 0;
    const int cnt = __popcll(path);
    if (tid < 64) {
        const bool on = path >> tid & 1;
        const int k = __popcll(path & ((1ull << tid) - 1));
        if (on) {
            const int i = ctx + tid, j = ctx + k;
            src_page[k] = i == j ? -1 : sb_kv_page(c, slot, i);
            src_t[k] = i % SB_PAGE_TOKENS;
            dst_page[k] = sb_kv_page(c, slot, j);
            dst_t[k] = j % SB_PAGE_TOKENS;
        }
        if (layer == 0) {
            if (tid == 0) out_count[s] = cnt;
            if (on) {
                out_node[s * 64 + k] = tid;
                out_token[s * 64 + k] = target[r0 + tid];
            }
            if (tid >= cnt) out_node[s * 64 + tid] = out_token[s * 64 + tid] = -1;
        }
    }
    __syncthreads();
    if (sb_kv_row_bytes(c.kv_dtype, c.head_dim) % 16 == 0)
        move_rows<uint4>(c, layer, cnt, src_page, src_t, dst_page, dst_t);
    else
        move_rows<uint32_t>(c, layer, cnt, src_page, src_t, dst_page, dst_t);
    if (c.kv_dtype == SLATE_KV_Q8)
        for (int hw = tid; hw < 2 * c.n_kv_heads; hw += AT)
            for (int k = 0; k < cnt; ++k) {
                if (src_page[k] < 0 || dst_page[k] < 0) continue;
                const int which = hw / c.n_kv_heads, h = hw % c.n_kv_heads;
                ((float*)sb_kv_block(c, layer, dst_page[k], which, h))[dst_t[k]] =
                    ((const float*)sb_kv_block(c, layer, src_page[k], which, h))[src_t[k]];
            }
}

}  // namespace

extern "C" int slate_cuda_rope_append(const slate_kv_cache_t* cache, int layer,
                                      const slate_rope_t* rope, int rows, int n_heads,
                                      float* q_out, int ld_q_out, const float* q, int ld_q,
                                      const float* k, int ld_k, const float* v, int ld_v,
                                      const int32_t* row_slot, const int32_t* row_index,
                                      const int32_t* row_pos, void* stream) {
    if (sb_kv_check(cache, "rope_append")) return -1;
    const int hd = cache->head_dim, nkv = cache->n_kv_heads;
    if (!rope || !rope->cos || !rope->sin || rope->n_pos < 1 || rope->rot_dim < 2 ||
        rope->rot_dim % 2 || rope->rot_dim > hd ||
        (rope->layout != SLATE_ROPE_HALF && rope->layout != SLATE_ROPE_INTERLEAVED)) {
        sb_set_error("rope_append: bad rope descriptor (rot_dim even, 2 to head_dim)");
        return -1;
    }
    if (layer < 0 || layer >= cache->n_layers || rows < 0 || n_heads < 1 || !q_out || !q || !k || !v ||
        !row_slot || !row_index || !row_pos || ld_q < n_heads * hd || ld_q_out < n_heads * hd ||
        ld_k < nkv * hd || ld_v < nkv * hd) {
        sb_set_error("rope_append: bad arguments");
        return -1;
    }
    if (rows == 0) return 0;
    const int64_t warps = (int64_t)rows * (n_heads + 2 * nkv);
    if ((warps + 7) / 8 > 0x7fffffff) {
        sb_set_error("rope_append: %d rows are too many", rows);
        return -1;
    }
    rope_append_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, (cudaStream_t)stream>>>(
        *cache, layer, *rope, rows, n_heads, q_out, ld_q_out, q, ld_q, k, ld_k, v, ld_v, row_slot,
        row_index, row_pos);
    return sb_cuda_check(cudaGetLastError(), "rope_append");
}

extern "C" int slate_cuda_kv_read(const slate_kv_cache_t* cache, int layer0, int n_layers, int rows,
                                  const int32_t* row_slot, const int32_t* row_index, void* K, void* V,
                                  int out_dtype, void* stream) {
    if (sb_kv_check(cache, "kv_read")) return -1;
    if (layer0 < 0 || n_layers < 1 || layer0 > cache->n_layers - n_layers || rows < 0 || !row_slot ||
        !row_index || !K || !V || (out_dtype != SLATE_KV_F32 && out_dtype != SLATE_KV_F16)) {
        sb_set_error("kv_read: bad arguments");
        return -1;
    }
    if (rows == 0) return 0;
    const int64_t warps = (int64_t)n_layers * rows * 2 * cache->n_kv_heads;
    if ((warps + 7) / 8 > 0x7fffffff) {
        sb_set_error("kv_read: %d rows of %d layers are too many", rows, n_layers);
        return -1;
    }
    const unsigned grid = (unsigned)((warps + 7) / 8);
    if (out_dtype == SLATE_KV_F16)
        kv_read_kernel<__half><<<grid, 256, 0, (cudaStream_t)stream>>>(
            *cache, layer0, n_layers, rows, row_slot, row_index, (__half*)K, (__half*)V);
    else
        kv_read_kernel<float><<<grid, 256, 0, (cudaStream_t)stream>>>(
            *cache, layer0, n_layers, rows, row_slot, row_index, (float*)K, (float*)V);
    return sb_cuda_check(cudaGetLastError(), "kv_read");
}

extern "C" int slate_cuda_tree_accept(const slate_kv_cache_t* cache, const slate_tree_t* tree,
                                      const int32_t* parent, const int32_t* token,
                                      const int32_t* target, int32_t* out_count, int32_t* out_node,
                                      int32_t* out_token, void* stream) {
    if (sb_kv_check(cache, "tree_accept") || sb_tree_check(tree, "tree_accept")) return -1;
    if (!parent || !token || !target || !out_count || !out_node || !out_token ||
        cache->n_layers > 65535) {
        sb_set_error("tree_accept: bad arguments");
        return -1;
    }
    tree_accept_kernel<<<dim3((unsigned)tree->n_seq, (unsigned)cache->n_layers), AT, 0,
                         (cudaStream_t)stream>>>(*cache, *tree, parent, token, target, out_count,
                                                 out_node, out_token);
    return sb_cuda_check(cudaGetLastError(), "tree_accept");
}
