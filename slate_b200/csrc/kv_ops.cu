// kv_ops.cu -- the cache operators that move rows: rotary append, read-back,
// acceptance of a drafted tree with the compaction of its path.  Interfaces and
// the 8-bit rule: include/slate_cuda.h.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "sb_internal.h"
#include "sb_kernels.h"
#include "sb_kv.h"
#include "sb_pdl.h"

namespace {

// Every kernel here begins with it: it may have been launched before the one ahead of it in the
// stream ended, and lets the next one do so if its own blocks are all running by then (blocks
// that wait would take the place of those still to come).
__device__ __forceinline__ void chain() {
    sb_grid_wait();
    if (gridDim.x * gridDim.y <= 2 * 148) sb_grid_release();
}

constexpr unsigned FULL = 0xffffffffu;

// One warp per (row, head): heads [0, nq) are query heads, then key heads, then
// value heads.  Each product and sum is rounded by itself (no fused multiply-
// add), so that an element next to a rounding boundary of the 8-bit grid falls
// on the side that the plain f32 formula gives.
__global__ void __launch_bounds__(256) rope_append_kernel(
    const slate_kv_cache_t c, int layer, const slate_rope_t rope, int rows, int nq,
    float* q_out, int ld_qo, const float* q, int ld_q, const float* __restrict__ k,
    int ld_k, const float* __restrict__ v, int ld_v, const int32_t* __restrict__ row_slot,
    const int32_t* __restrict__ row_index, const int32_t* __restrict__ row_pos) {
    chain();
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

// The same in 16-byte vectors, for head_dim up to 128 and rot_dim % 8 == 0 (every
// common head): LPH lanes hold a head, four dims each, so a pair's other half is in the
// same lane (interleaved) or rot_dim / 8 lanes away (one shuffle an element), and a
// warp keeps RU * 32 / LPH heads in flight; query heads and key/value heads go to warps
// of their own, so neither carries the other's branches.  Bound by HBM: q is read and
// written, k and v read, the cache written once; nothing else moves.  8191 rows of 32 + 8
// + 8 heads of 128 on the 8-bit cache, with their read-back: 82 us, 5.4 TB/s (exact
// division for every element: 101 us; q and k heads in one warp: 95 us).  Blocks an SM: six
// on 8 bits, where instructions count (82 us; 86 with the four that registers would leave),
// five else (8191 rows of f16 62 us; six spill, 66).
template <int LPH, int KV, int RU>
__global__ void __launch_bounds__(256, KV == SLATE_KV_Q8 ? 6 : 5) rope_append_vec(
    const slate_kv_cache_t c, int layer, const slate_rope_t rope, int rows, int nq,
    float* q_out, int ld_qo, const float* q, int ld_q, const float* __restrict__ k, int ld_k,
    const float* __restrict__ v, int ld_v, const int32_t* __restrict__ row_slot,
    const int32_t* __restrict__ row_index, const int32_t* __restrict__ row_pos, int parts_q, int parts) {
    chain();
    constexpr int HPW = 32 / LPH;                          // heads a warp holds at once
    const int lane = threadIdx.x & 31, sub = lane % LPH, hd = c.head_dim, nkv = c.n_kv_heads;
    const int half = rope.rot_dim / 2, d = 4 * sub;
    const unsigned w = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, r = w / parts;
    if (r >= (unsigned)rows) return;
    // parts [0, parts_q) of a row are its query heads, the others its key and then value heads
    const int part = (int)(w - r * parts);
    const bool keys = part >= parts_q;
    const int n = keys ? 2 * nkv : nq, h0 = (keys ? part - parts_q : part) * (RU * HPW) + lane / LPH;
    const int index = row_index[r], pos = row_pos[r], slot = row_slot[r];
    const bool in = d < hd;
    float4 x[RU];                                          // asked for before the row is looked at
    {
        const float* first = (keys ? k + (size_t)r * ld_k : q + (size_t)r * ld_q) + d;
        const float* vals = v + (size_t)r * ld_v - nkv * hd + d;
#pragma unroll
        for (int u = 0; u < RU; ++u) {
            const int h = h0 + u * HPW;
            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (in && h < n) x[u] = *(const float4*)((keys && h >= nkv ? vals : first) + h * hd);
        }
    }
    if (index < 0 || pos < 0 || pos >= rope.n_pos) return;
    const bool inter = rope.layout == SLATE_ROPE_INTERLEAVED, second = d >= half;
    // An element is its own value times cos plus its partner's times sin, -sin for the first of a
    // pair; dims beyond rot_dim keep their value (and are spared the product: 0 * NaN).
    const bool turn = d < rope.rot_dim;
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    if (turn) {
        const size_t j = (size_t)pos * half + (inter ? d / 2 : second ? d - half : d);
        if (inter) {
            const float2 a = *(const float2*)(rope.cos + j), b = *(const float2*)(rope.sin + j);
            cs = make_float4(a.x, a.x, a.y, a.y);
            sn = make_float4(-b.x, b.x, -b.y, b.y);
        } else {
            cs = *(const float4*)(rope.cos + j);
            sn = *(const float4*)(rope.sin + j);
            if (!second) sn = make_float4(-sn.x, -sn.y, -sn.z, -sn.w);
        }
    }
    const int from = inter ? lane : second ? lane - half / 4 : lane + half / 4;
    const auto turned = [&](const float4& a) {
        float4 o = make_float4(a.y, a.x, a.w, a.z);        // the partners
        if (!inter) {
            o.x = __shfl_sync(FULL, a.x, from & 31);
            o.y = __shfl_sync(FULL, a.y, from & 31);
            o.z = __shfl_sync(FULL, a.z, from & 31);
            o.w = __shfl_sync(FULL, a.w, from & 31);
        }
        if (!turn) return a;
        return make_float4(__fadd_rn(__fmul_rn(a.x, cs.x), __fmul_rn(o.x, sn.x)),
                           __fadd_rn(__fmul_rn(a.y, cs.y), __fmul_rn(o.y, sn.y)),
                           __fadd_rn(__fmul_rn(a.z, cs.z), __fmul_rn(o.z, sn.z)),
                           __fadd_rn(__fmul_rn(a.w, cs.w), __fmul_rn(o.w, sn.w)));
    };
    if (!keys) {
        float* o = q_out + (size_t)r * ld_qo + d;
#pragma unroll
        for (int u = 0; u < RU; ++u) {
            const int h = h0 + u * HPW;
            const float4 y = turned(x[u]);
            if (in && h < n) *(float4*)(o + h * hd) = y;
        }
        return;
    }
    const int page = sb_kv_page(c, slot, index), t = index % SB_PAGE_TOKENS;
    if (page < 0) return;
    unsigned char* blocks = sb_kv_block(c, layer, page, 0, 0);     // K heads, then V heads
    const int bb = sb_kv_block_bytes(KV, hd);
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const int h = h0 + u * HPW;
        float4 y = turned(x[u]);
        if (h >= nkv) y = x[u];                            // (the shuffles above take every lane)
        uint32_t top = 0;
        if (KV == SLATE_KV_Q8) {
            const uint32_t m = 0x7fffffffu;
            top = max(max(__float_as_uint(y.x) & m, __float_as_uint(y.y) & m),
                      max(__float_as_uint(y.z) & m, __float_as_uint(y.w) & m));
            if (LPH == 32) top = __reduce_max_sync(FULL, top);
            else
#pragma unroll
                for (int z = LPH / 2; z; z >>= 1) top = max(top, __shfl_xor_sync(FULL, top, z));
        }
        if (!in || h >= n) continue;
        unsigned char* blk = blocks + (size_t)h * bb;
        if (KV == SLATE_KV_F32) {
            *(float4*)((float*)blk + t * hd + d) = y;
        } else if (KV == SLATE_KV_F16) {
            const __half2 a = __floats2half2_rn(y.x, y.y), b = __floats2half2_rn(y.z, y.w);
            *(uint2*)((__half*)blk + t * hd + d) = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
        } else {
            const float scale = __fmul_rn(__uint_as_float(top), (float)(1.0 / 127.0));
            // rint(x / scale): from x * (1 / scale), off by at most 1.5e-5, and the division itself where
            // that lies as near as 1e-4 to a boundary between two integers (or 1 / scale is no number).
            // Adding 1.5 * 2^23 rounds to the integer and leaves it in the low byte.
            const float inv = __frcp_rn(scale);
            const bool plain = scale > 0.f && scale < INFINITY, fast = plain && inv < INFINITY;
            const auto near = [&](float a) {
                const float z = a * inv;
                return fabsf(fabsf(z - ((z + 12582912.f) - 12582912.f)) - 0.5f) < 1e-4f;
            };
            const auto divided = [&](float a) {
                return plain ? (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(a, scale)), -127.f), 127.f) : 0u;
            };
            uint32_t q4[4];
            if (!fast || near(y.x) || near(y.y) || near(y.z) || near(y.w)) {
                q4[0] = divided(y.x), q4[1] = divided(y.y), q4[2] = divided(y.z), q4[3] = divided(y.w);
            } else {
                q4[0] = __float_as_uint(y.x * inv + 12582912.f), q4[1] = __float_as_uint(y.y * inv + 12582912.f);
                q4[2] = __float_as_uint(y.z * inv + 12582912.f), q4[3] = __float_as_uint(y.w * inv + 12582912.f);
            }
            if (sub == 0) ((float*)blk)[t] = scale;
            *(uint32_t*)(blk + SB_Q8_SCALES + t * hd + d) =
                __byte_perm(__byte_perm(q4[0], q4[1], 0x0040), __byte_perm(q4[2], q4[3], 0x0040), 0x5410);
        }
    }
}

// A warp per (layer, row), K and V: its n_kv_heads * head_dim / 4 vectors of four in
// steps of 32, RV vectors of each in flight.  Consecutive lanes write consecutive 16
// (f16: 8) bytes, and read 4, 8 or 16.  Bound by HBM, mostly by what it writes: 32760 rows of
// 4 layers from 8 bits to f32 in 210 us, 6.4 TB/s; 517 rows of 2 layers 2.8 us, launch and latency.
constexpr int RV = 4;
template <int KV>
struct Vec4 {
    using T = uint32_t;
};
template <>
struct Vec4<SLATE_KV_F16> {
    using T = uint2;
};
template <>
struct Vec4<SLATE_KV_F32> {
    using T = float4;
};
__device__ __forceinline__ float4 widen(float4 x, float) { return x; }
__device__ __forceinline__ float4 widen(uint2 x, float) {
    const float2 a = __half22float2(*(const __half2*)&x.x), b = __half22float2(*(const __half2*)&x.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 widen(uint32_t x, float s) {
    return make_float4((float)(int8_t)x * s, (float)(int8_t)(x >> 8) * s, (float)(int8_t)(x >> 16) * s,
                       (float)(int8_t)(x >> 24) * s);
}
__device__ __forceinline__ void put4(float* p, float4 x) { *(float4*)p = x; }
__device__ __forceinline__ void put4(__half* p, float4 x) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    *(uint2*)p = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
}
template <typename OT, int KV>
__global__ void __launch_bounds__(256) kv_read_kernel(
    const slate_kv_cache_t c, int layer0, int n_layers, int rows,
    const int32_t* __restrict__ row_slot, const int32_t* __restrict__ row_index,
    OT* __restrict__ K, OT* __restrict__ V) {
    chain();
    using T = typename Vec4<KV>::T;
    const int lane = threadIdx.x & 31, hd4 = c.head_dim / 4, nv = c.n_kv_heads * hd4;
    const int64_t w = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (w >= (int64_t)n_layers * rows) return;
    const int r = (int)(w % rows), layer = layer0 + (int)(w / rows);
    const int index = row_index[r], page = sb_kv_page(c, row_slot[r], index), t = index % SB_PAGE_TOKENS;
    const size_t bb = sb_kv_block_bytes(KV, c.head_dim);
    const unsigned char* kb = page < 0 ? nullptr : sb_kv_block(c, layer, page, 0, 0);
    const size_t head = KV == SLATE_KV_Q8 ? SB_Q8_SCALES : 0, vo = (size_t)c.n_kv_heads * bb;
    for (int e0 = lane; e0 < nv; e0 += 32 * RV) {
        T k[RV] = {}, v[RV] = {};
        float ks[RV] = {}, vs[RV] = {};
        if (kb) {
#pragma unroll
            for (int i = 0; i < RV; ++i) {
                const int e = e0 + 32 * i;
                if (e >= nv) break;
                const int h = e / hd4;
                const unsigned char* b = kb + h * bb;
                const size_t at = head + ((size_t)t * hd4 + (e - h * hd4)) * sizeof(T);
                k[i] = *(const T*)(b + at);
                v[i] = *(const T*)(b + vo + at);
                if (KV == SLATE_KV_Q8) {
                    ks[i] = ((const float*)b)[t];
                    vs[i] = ((const float*)(b + vo))[t];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < RV; ++i) {
            const int e = e0 + 32 * i;
            if (e >= nv) break;
            put4(K + ((size_t)w * nv + e) * 4, widen(k[i], ks[i]));
            put4(V + ((size_t)w * nv + e) * 4, widen(v[i], vs[i]));
        }
    }
}

// One warp per (layer, row, K|V, head): outputs that are not aligned to a vector.
template <typename OT>
__global__ void __launch_bounds__(256) kv_read_scalar(
    const slate_kv_cache_t c, int layer0, int n_layers, int rows,
    const int32_t* __restrict__ row_slot, const int32_t* __restrict__ row_index,
    OT* __restrict__ K, OT* __restrict__ V) {
    chain();
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
// in order never overwrites what is still to be read, nor does reading MU rows ahead.  Bound by
// latency for few sequences (13 nodes, 16 layers: 3.6 us) and by scattered rows of HBM for many (48
// x 40 nodes, 32 layers of f16: 21 us, 4.9 TB/s).
constexpr int AT = 256, MU = 8;
template <typename U>
__device__ void move_rows(const slate_kv_cache_t& c, int layer, int n, const int* src_page,
                          const int* src_t, const int* dst_page, const int* dst_t) {
    const int rb = sb_kv_row_bytes(c.kv_dtype, c.head_dim), cols = rb / (int)sizeof(U);
    const int head_off = c.kv_dtype == SLATE_KV_Q8 ? SB_Q8_SCALES : 0;
    const int bb = sb_kv_block_bytes(c.kv_dtype, c.head_dim);
    const size_t page_bytes = (size_t)2 * c.n_kv_heads * bb;
    for (int e = threadIdx.x; e < 2 * c.n_kv_heads * cols; e += AT) {
        const int col = e % cols, hw = e / cols;
        unsigned char* base = sb_kv_block(c, layer, 0, 0, 0) + hw * (size_t)bb + head_off + col * sizeof(U);
        for (int k0 = 0; k0 < n; k0 += MU) {
            U x[MU];
#pragma unroll
            for (int u = 0; u < MU; ++u)
                if (k0 + u < n && src_page[k0 + u] >= 0 && dst_page[k0 + u] >= 0)
                    x[u] = *(const U*)(base + src_page[k0 + u] * page_bytes + src_t[k0 + u] * rb);
#pragma unroll
            for (int u = 0; u < MU; ++u)
                if (k0 + u < n && src_page[k0 + u] >= 0 && dst_page[k0 + u] >= 0)
                    *(U*)(base + dst_page[k0 + u] * page_bytes + dst_t[k0 + u] * rb) = x[u];
        }
    }
}

__global__ void __launch_bounds__(AT) tree_accept_kernel(
    const slate_kv_cache_t c, const slate_tree_t tr, const int32_t* __restrict__ parent,
    const int32_t* __restrict__ token, const int32_t* __restrict__ target, int32_t* out_count,
    int32_t* out_node, int32_t* out_token) {
    chain();
    __shared__ uint32_t ok_s[2];
    __shared__ int best_s[2];
    __shared__ int src_page[64], src_t[64], dst_page[64], dst_t[64];
    const int s = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x;
    const int r0 = max(tr.row_off[s], 0), r1 = min(tr.row_off[s + 1], tr.rows);
    const int n = min(max(r1 - r0, 0), tr.max_nodes);    // as the attention
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
        // the node itself and all of its mask; deepest first, then the lowest index
        const int score = tid < n && !((m | 1ull << tid) & ~ok) ? __popcll(m) * 64 + 63 - tid : 0;
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
            const size_t o = (size_t)s * SLATE_TREE_MAX_NODES;       // passes 32 bits from 2^25 sequences
            if (on) {
                out_node[o + k] = tid;
                out_token[o + k] = target[r0 + tid];
            }
            if (tid >= cnt) out_node[o + tid] = out_token[o + tid] = -1;
        }
    }
    __syncthreads();
    if (sb_kv_row_bytes(c.kv_dtype, c.head_dim) % 16 == 0)
        move_rows<uint4>(c, layer, cnt, src_page, src_t, dst_page, dst_t);
    else
        move_rows<uint32_t>(c, layer, cnt, src_page, src_t, dst_page, dst_t);
    if (c.kv_dtype == SLATE_KV_Q8)
        for (int hw = AT - 1 - tid; hw < 2 * c.n_kv_heads; hw += AT) { // the scales, alike, by threads that had fewer columns
            const int which = hw / c.n_kv_heads, h = hw % c.n_kv_heads;
            for (int k0 = 0; k0 < cnt; k0 += MU) {
                float x[MU];
#pragma unroll
                for (int u = 0; u < MU; ++u)
                    if (k0 + u < cnt && src_page[k0 + u] >= 0 && dst_page[k0 + u] >= 0)
                        x[u] = ((const float*)sb_kv_block(c, layer, src_page[k0 + u], which, h))[src_t[k0 + u]];
#pragma unroll
                for (int u = 0; u < MU; ++u)
                    if (k0 + u < cnt && src_page[k0 + u] >= 0 && dst_page[k0 + u] >= 0)
                        ((float*)sb_kv_block(c, layer, dst_page[k0 + u], which, h))[dst_t[k0 + u]] = x[u];
            }
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
        !row_slot || !row_index || !row_pos || ld_q < (int64_t)n_heads * hd || ld_q_out < (int64_t)n_heads * hd ||
        ld_k < (int64_t)nkv * hd || ld_v < (int64_t)nkv * hd) {
        sb_set_error("rope_append: bad arguments");
        return -1;
    }
    if (rows == 0) return 0;
    const int64_t warps = (int64_t)rows * (n_heads + 2 * nkv);      // of the scalar kernel, the most
    if ((warps + 7) / 8 > 0x7fffffff) {
        sb_set_error("rope_append: %d rows are too many", rows);
        return -1;
    }
    const auto al = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
    // vectors need rows and tables on 16 bytes; other strides take the scalar kernel
    if (hd <= 128 && rope->rot_dim % 8 == 0 && al(q) && al(q_out) && al(k) && al(v) && al(rope->cos) &&
        al(rope->sin) && ld_q % 4 == 0 && ld_q_out % 4 == 0 && ld_k % 4 == 0 && ld_v % 4 == 0) {
        const int lph = hd > 64 ? 32 : hd > 32 ? 16 : 8, hpw = 32 / lph, heads = n_heads + 2 * nkv;
        // RU head groups a warp in flight: four where two would still make a full wave of warps (64 an
        // SM; 8191 rows of 48 heads: 82 us against 95 with two), else two (16 such rows: 6.9 against 7.5)
        const int ru = (int64_t)rows * heads / (2 * hpw) > 148 * 64 ? 4 : 2;
        const int parts_q = (n_heads + ru * hpw - 1) / (ru * hpw);
        const int parts = parts_q + (2 * nkv + ru * hpw - 1) / (ru * hpw);
        const int64_t n = (int64_t)rows * parts;
        const auto go = [&](auto kernel) {
            return sb_launch_pdl(kernel, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, (cudaStream_t)stream, *cache,
                                 layer, *rope, rows, n_heads, q_out, ld_q_out, q, ld_q, k, ld_k, v, ld_v, row_slot,
                                 row_index, row_pos, parts_q, parts);
        };
        const auto by_type = [&](auto l, auto u) {
            constexpr int L = decltype(l)::value, U = decltype(u)::value;
            return cache->kv_dtype == SLATE_KV_F32   ? go(rope_append_vec<L, SLATE_KV_F32, U>)
                   : cache->kv_dtype == SLATE_KV_F16 ? go(rope_append_vec<L, SLATE_KV_F16, U>)
                                                     : go(rope_append_vec<L, SLATE_KV_Q8, U>);
        };
        const auto by_ru = [&](auto l) {
            return ru == 2 ? by_type(l, std::integral_constant<int, 2>{}) : by_type(l, std::integral_constant<int, 4>{});
        };
        return sb_cuda_check(lph == 32   ? by_ru(std::integral_constant<int, 32>{})
                             : lph == 16 ? by_ru(std::integral_constant<int, 16>{})
                                         : by_ru(std::integral_constant<int, 8>{}),
                             "rope_append");
    }
    return sb_cuda_check(sb_launch_pdl(rope_append_kernel, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0,
                                       (cudaStream_t)stream, *cache, layer, *rope, rows, n_heads, q_out, ld_q_out, q,
                                       ld_q, k, ld_k, v, ld_v, row_slot, row_index, row_pos),
                         "rope_append");
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
    const int64_t each = (int64_t)n_layers * 2 * cache->n_kv_heads;          // warps a row of the scalar kernel
    if (rows > 0x3fffffff8 / each) {                                         // 2^31 - 1 blocks of 8 warps
        sb_set_error("kv_read: %d rows of %d layers are too many", rows, n_layers);
        return -1;
    }
    const int64_t warps = rows * each;
    const cudaStream_t st = (cudaStream_t)stream;
    const uintptr_t mis = ((uintptr_t)K | (uintptr_t)V) & (out_dtype == SLATE_KV_F16 ? 7 : 15);
    const auto go = [&](auto vec, auto scalar, auto* k, auto* v) {
        const int64_t n = mis ? warps : (int64_t)n_layers * rows;
        return sb_launch_pdl(mis ? scalar : vec, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, st, *cache, layer0, n_layers,
                             rows, row_slot, row_index, k, v);
    };
    const int kt = cache->kv_dtype;
    const cudaError_t err =
        out_dtype == SLATE_KV_F16 ? go(kt == SLATE_KV_F32   ? kv_read_kernel<__half, SLATE_KV_F32>
                                       : kt == SLATE_KV_F16 ? kv_read_kernel<__half, SLATE_KV_F16>
                                                            : kv_read_kernel<__half, SLATE_KV_Q8>,
                                       kv_read_scalar<__half>, (__half*)K, (__half*)V)
                                  : go(kt == SLATE_KV_F32   ? kv_read_kernel<float, SLATE_KV_F32>
                                       : kt == SLATE_KV_F16 ? kv_read_kernel<float, SLATE_KV_F16>
                                                            : kv_read_kernel<float, SLATE_KV_Q8>,
                                       kv_read_scalar<float>, (float*)K, (float*)V);
    return sb_cuda_check(err, "kv_read");
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
    return sb_cuda_check(sb_launch_pdl(tree_accept_kernel, dim3((unsigned)tree->n_seq, (unsigned)cache->n_layers), dim3(AT),
                                       0, (cudaStream_t)stream, *cache, *tree, parent, token, target, out_count, out_node,
                                       out_token),
                         "tree_accept");
}
