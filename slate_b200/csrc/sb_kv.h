/*
 * sb_kv.h -- addressing of the paged KV cache for the cache operators
 * (kv_ops.cu, attn_tree.cu; internal, CUDA C++ only).  Layout and the 8-bit
 * rule are documented at slate_kv_cache_t in include/slate_cuda.h.
 */
#ifndef SB_KV_H
#define SB_KV_H

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "sb_kernels.h"

#define SB_KV_MAX_PAGES (1 << 26)           /* a slot: 2^30 tokens, so that ends and looks ahead stay within an int */
#define SB_Q8_SCALES (4 * SB_PAGE_TOKENS)   /* bytes of scales in front of a block's int8 rows */

/* Bytes of one (page, K|V, head) block and of one row of it. */
static __host__ __device__ __forceinline__ int sb_kv_row_bytes(int kv_dtype, int hd) {
    return kv_dtype == SLATE_KV_F32 ? 4 * hd : kv_dtype == SLATE_KV_F16 ? 2 * hd : hd;
}
static __host__ __device__ __forceinline__ int sb_kv_block_bytes(int kv_dtype, int hd) {
    return SB_PAGE_TOKENS * sb_kv_row_bytes(kv_dtype, hd) +
           (kv_dtype == SLATE_KV_Q8 ? SB_Q8_SCALES : 0);
}

#ifdef __CUDACC__
/* Page of place `index` of `slot`, -1 when there is none (or the table holds
 * one outside the pool). */
static __device__ __forceinline__ int sb_kv_page(const slate_kv_cache_t& c, int slot, int index) {
    if (slot < 0 || slot >= c.n_slots || index < 0 || index / SB_PAGE_TOKENS >= c.max_pages)
        return -1;
    const int page = __ldg(c.page_table + (size_t)slot * c.max_pages + index / SB_PAGE_TOKENS);
    return page < 0 || page >= c.n_pages ? -1 : page;
}
/* Block of (layer, page, K = 0 | V = 1, head): 64-bit throughout, a pool may
 * exceed 4 GB many times over. */
static __device__ __forceinline__ unsigned char* sb_kv_block(const slate_kv_cache_t& c, int layer,
                                                             int page, int which, int head) {
    const size_t n = (((size_t)layer * c.n_pages + page) * 2 + which) * c.n_kv_heads + head;
    return (unsigned char*)c.pool + n * sb_kv_block_bytes(c.kv_dtype, c.head_dim);
}
#endif

#ifdef __cplusplus
extern "C" {
#endif
/* Checks a cache descriptor; records the message and returns -1 when it is
 * unusable (rope.c). */
int sb_kv_check(const slate_kv_cache_t* c, const char* who);
int sb_tree_check(const slate_tree_t* t, const char* who);
#ifdef __cplusplus
}
#endif
#endif
