/*
 * rope.c -- host side of the cache operators: rotary tables, tree masks, the
 * checks of their descriptors.
 */
#define _GNU_SOURCE
#include "sb_internal.h"
#include "sb_kernels.h"
#include "sb_kv.h"

#include <math.h>

size_t slate_kv_pool_bytes(int kv_dtype, int64_t n_pages, int n_layers, int n_kv_heads,
                           int head_dim) {
    if (kv_dtype < SLATE_KV_F32 || kv_dtype > SLATE_KV_Q8 || n_pages < 1 || n_layers < 1 ||
        n_kv_heads < 1 || head_dim < 1)
        return 0;
    const size_t row = kv_dtype == SLATE_KV_F32 ? 4u * (size_t)head_dim
                       : kv_dtype == SLATE_KV_F16 ? 2u * (size_t)head_dim
                                                  : (size_t)head_dim + 4;
    return (size_t)n_pages * (size_t)n_layers * 2 * (size_t)n_kv_heads * SB_PAGE_TOKENS * row;
}

/* The frequency of pair j is theta^(-2j / rot_dim).  Everything is formed in
 * f64: at position 10^5 a product in f32 would already be off by 4e-3. */
int slate_rope_tables(float* cos_t, float* sin_t, int n_pos, int rot_dim, float theta,
                      const slate_rope_scaling_t* sc) {
    if (!cos_t || !sin_t || n_pos < 1 || rot_dim < 2 || rot_dim % 2 || !(theta > 0.f)) {
        sb_set_error("rope_tables: bad arguments");
        return -1;
    }
    const int kind = sc ? sc->kind : SLATE_ROPE_SCALE_NONE;
    const double f = sc && kind != SLATE_ROPE_SCALE_NONE ? (double)sc->factor : 1.0;
    if (kind < SLATE_ROPE_SCALE_NONE || kind > SLATE_ROPE_SCALE_BANDS || !(f >= 1.0) || isinf(f) ||
        (kind == SLATE_ROPE_SCALE_NTK && rot_dim < 4) ||
        (kind == SLATE_ROPE_SCALE_BANDS &&
         (!(sc->low > 0.f) || !(sc->high > sc->low) || sc->trained < 1)) ||
        (sc && !(sc->magnitude >= 0.f && !isinf(sc->magnitude)))) {
        sb_set_error("rope_tables: bad scaling");
        return -1;
    }
    const double mag = sc && sc->magnitude > 0.f ? (double)sc->magnitude : 1.0;
    const double base = kind == SLATE_ROPE_SCALE_NTK
                            ? (double)theta * pow(f, (double)rot_dim / (rot_dim - 2))
                            : (double)theta;
    const int half = rot_dim / 2;
    for (int j = 0; j < half; ++j) {
        double w = pow(base, -2.0 * j / rot_dim);
        if (kind == SLATE_ROPE_SCALE_LINEAR) w /= f;
        if (kind == SLATE_ROPE_SCALE_BANDS) {
            /* full turns of this pair over the trained length: few turns (long
             * wavelengths) are compressed, many are kept */
            const double turns = sc->trained * w / (2.0 * M_PI);
            double keep = (turns - sc->low) / ((double)sc->high - sc->low);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            w = w * keep + w / f * (1 - keep);
        }
        for (int p = 0; p < n_pos; ++p) {
            cos_t[(size_t)p * half + j] = (float)(mag * cos(p * w));
            sin_t[(size_t)p * half + j] = (float)(mag * sin(p * w));
        }
    }
    return 0;
}

int slate_tree_masks(uint64_t* mask, const int32_t* parent, int n) {
    if (!mask || !parent || n < 0 || n > SLATE_TREE_MAX_NODES) {
        sb_set_error("tree_masks: bad arguments");
        return -1;
    }
    for (int i = 0; i < n; ++i) {
        if (parent[i] < -1 || parent[i] >= i) {
            sb_set_error("tree_masks: node %d has parent %d (a parent comes before its node)", i,
                         (int)parent[i]);
            return -1;
        }
        mask[i] = (parent[i] >= 0 ? mask[parent[i]] : 0) | (uint64_t)1 << i;
    }
    return 0;
}

int sb_kv_check(const slate_kv_cache_t* c, const char* who) {
    if (!c || !c->pool || !c->page_table || ((uintptr_t)c->pool & 15) || c->n_pages < 1 ||
        c->n_pages > 0x7fffffff || c->n_slots < 1 || c->max_pages < 1 ||
        c->max_pages > SB_KV_MAX_PAGES || c->n_layers < 1 || c->n_kv_heads < 1) {
        sb_set_error("%s: bad cache descriptor", who);
        return -1;
    }
    if (c->head_dim < 4 || c->head_dim > 256 || c->head_dim % 4) {
        sb_set_error("%s: head_dim %d (a multiple of 4 from 4 to 256)", who, c->head_dim);
        return -1;
    }
    if (c->kv_dtype < SLATE_KV_F32 || c->kv_dtype > SLATE_KV_Q8) {
        sb_set_error("%s: kv_dtype %d", who, c->kv_dtype);
        return -1;
    }
    return 0;
}

int sb_tree_check(const slate_tree_t* t, const char* who) {
    if (!t || t->n_seq < 1 || t->rows < 0 || t->max_nodes < 1 || !t->row_off || !t->slot ||
        !t->ctx || !t->mask) {
        sb_set_error("%s: bad tree descriptor", who);
        return -1;
    }
    if (t->max_nodes > SLATE_TREE_MAX_NODES ||
        (int64_t)t->rows > (int64_t)t->n_seq * t->max_nodes) {
        sb_set_error("%s: %d rows in %d sequences of up to %d nodes (at most %d)", who, t->rows,
                     t->n_seq, t->max_nodes, SLATE_TREE_MAX_NODES);
        return -1;
    }
    return 0;
}
