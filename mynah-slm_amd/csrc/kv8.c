/* kv8.c — host side of the 8-bit cache (include/mynah_cache.h; kernels in
 * kv8.hip): argument checks and launch geometry.
 *
 * SPDX-License-Identifier: MIT */
#include "mynah_cache.h"

#include "args.h"

#include <float.h>
#include <math.h>
#include <string.h>

static int cache_check(const mynah_kv8_cache *c, uint32_t n_seqs, uint64_t max_kv,
                       const char *what) {
    if (c->k == NULL || c->v == NULL || c->k_scale == NULL || c->v_scale == NULL)
        return refuse("null argument");
    if (c->format != MYNAH_KV_I8 && c->format != MYNAH_KV_E4M3) {
        mynah_set_error("%s: unknown format %d", what, c->format);
        return -1;
    }
    const size_t hd = c->head_dim;
    if ((hd != 64 && hd != 128 && hd != 256) || c->n_kv_heads == 0 || c->n_kv_heads > 65536) {
        mynah_set_error("%s: %u heads of %u values: head_dim 64, 128 or 256 is taken", what,
                        c->n_kv_heads, c->head_dim);
        return -1;
    }
    if (!is_power(c->block) || c->block < 16 || c->block > 256) {
        mynah_set_error("%s: a block of %u positions: powers of two from 16 to 256 are taken",
                        what, c->block);
        return -1;
    }
    if (c->n_slots == 0 || c->n_slots > (size_t)1 << 40 || c->n_slots % c->block != 0) {
        mynah_set_error("%s: %zu cache rows: whole blocks are needed", what, c->n_slots);
        return -1;
    }
    if (c->pages != NULL) {
        if (!is_power(c->page_size) || c->page_size < c->block) {
            mynah_set_error("%s: page_size must be a power of two, a block at least", what);
            return -1;
        }
        if ((uint64_t)c->max_pages * c->page_size < max_kv) {
            mynah_set_error("%s: max_kv positions do not fit the page table", what);
            return -1;
        }
    } else if (n_seqs > 1 &&
               (c->seq_slots > ((size_t)1 << 40) / n_seqs || c->seq_slots % c->block != 0)) {
        mynah_set_error("%s: bad seq_slots", what);
        return -1;
    }
    if (c->slot_stride < c->n_kv_heads * hd || c->slot_stride >= (size_t)1 << 24) {
        mynah_set_error("%s: bad slot_stride", what);
        return -1;
    }
    if ((((uintptr_t)c->k | (uintptr_t)c->v | c->slot_stride) & 15u) != 0 ||
        (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale | (uintptr_t)c->pages) & 3u) != 0) {
        mynah_set_error("%s: the cache and its rows must be 16-byte aligned", what);
        return -1;
    }
    return 0;
}

/* ── rows into the cache ─────────────────────────────────────────────────── */

int mynah_hip_kv8_store_dev(const mynah_kv8_store *p, void *stream) {
    if (p == NULL || p->k == NULL || p->v == NULL || p->seq_start == NULL || p->n_past == NULL)
        return refuse("null argument");
    const size_t size = elem_size(p->type);
    if (size == 0) {
        mynah_set_error("kv8_store: type %d is not f32, f16 or bf16", p->type);
        return -1;
    }
    if (p->n_seqs == 0 || p->n_seqs > 65536 || p->n_rows == 0 || p->n_rows > 0x7fffffffu ||
        p->max_nodes == 0 || p->max_nodes > 1u << 24 || p->max_kv == 0 || p->max_kv > 1u << 26)
        return refuse("kv8_store: bad counts (sequences, rows, tokens or positions)");
    const mynah_kv8_cache *c = &p->cache;
    if (cache_check(c, p->n_seqs, p->max_kv, "kv8_store") != 0) return -1;
    /* Two sequences' rows may not meet: a block has one owner. */
    if (c->pages == NULL && p->n_seqs > 1 && p->max_kv > c->seq_slots)
        return refuse("kv8_store: max_kv positions do not fit seq_slots");
    const size_t row = (size_t)c->n_kv_heads * c->head_dim;
    if (p->k_stride < row || p->v_stride < row || !fits(p->n_rows, p->k_stride, row, size) ||
        !fits(p->n_rows, p->v_stride, row, size))
        return refuse("kv8_store: bad stride");
    if ((((uintptr_t)p->k | (uintptr_t)p->v | p->k_stride * size | p->v_stride * size) & 15u) != 0 ||
        (((uintptr_t)p->seq_start | (uintptr_t)p->n_past) & 3u) != 0)
        return refuse("kv8_store: k, v and strides must be 16-byte aligned");
    mynah_kv8_store_args a;
    memset(&a, 0, sizeof a);
    a.x[0] = p->k;
    a.x[1] = p->v;
    a.x_stride[0] = p->k_stride;
    a.x_stride[1] = p->v_stride;
    a.c[0] = c->k;
    a.c[1] = c->v;
    a.s[0] = c->k_scale;
    a.s[1] = c->v_scale;
    a.seq_start = p->seq_start;
    a.n_past = p->n_past;
    a.pages = c->pages;
    a.slot_stride = c->slot_stride;
    a.seq_slots = c->seq_slots;
    a.n_slots = c->n_slots;
    a.n_seqs = p->n_seqs;
    a.n_kv = c->n_kv_heads;
    a.n_rows = p->n_rows;
    if (c->pages != NULL) a.page_log2 = log2_of(c->page_size);
    a.max_pages = c->max_pages;
    a.block_log2 = log2_of(c->block);
    a.max_nodes = p->max_nodes;
    a.max_kv = p->max_kv;
    a.format = (uint32_t)c->format;
    /* The most blocks that max_nodes positions in a row touch. */
    a.blocks = (p->max_nodes + c->block - 2) / c->block + 1;
    const unsigned long long all = (unsigned long long)p->n_seqs * a.blocks;
    /* A search of the sequence costs a microsecond or two, empty workgroups more where
     * they are many. */
    const unsigned long long few = p->n_rows / c->block + 2ull * p->n_seqs;
    a.ragged = all > 4 * few + 4096;
    const unsigned long long units = (a.ragged ? few : all) * 2 * a.n_kv;
    /* A wave a block where a call's few rows fill no workgroup. */
    const uint32_t most = p->max_nodes < c->block ? p->max_nodes : c->block;
    const uint32_t wide = most * c->head_dim > 512u ? 1u : 0u;
    if (units > MYNAH_MOST_WGS(wide ? 256 : 64))
        return refuse("kv8_store: too many blocks for one launch");
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    const int h = c->head_dim == 64 ? 0 : c->head_dim == 128 ? 1 : 2;
    void *args[] = {&a};
    return mynah_launch(d, MYNAH_K_KV8_STORE + 6 * type_index(p->type) + 2 * h + (int)wide,
                        (unsigned)units, 1, wide ? 256 : 64, 0,
                        mynah_stream_or_default(d, stream), args);
}

/* ── attention ───────────────────────────────────────────────────────────── */

/* What a call launches: kernels of few rows (16 `tiles` a workgroup) or, wide,
 * of many; a workgroup of `waves` waves for each key head, group of `rows` query rows
 * and slot: a sequence's, or with more slots than sequences a piece of one. */
typedef struct {
    uint32_t wide, tiles, waves, rows, groups, slots;
} kv8_plan;
#define KV8_WAVES 4u                /* of the kernels of few rows (= Kv8Shape::W) */
#define KV8_WIDE_WAVES 8u           /* of those of many (= Kv8Wide::W) */

static void make_plan(const mynah_kv8_attention *p, uint32_t cus, kv8_plan *t) {
    const uint32_t group = p->n_heads / p->cache.n_kv_heads, hd = p->cache.head_dim;
    const uint64_t rows = (uint64_t)p->max_nodes * group;
    /* Several workgroups of few rows read the same keys, each for itself; from some
     * number of rows on the shared chunk wins. Few against wide in us, 32 heads, 8 of
     * keys, i8, 4 sequences over 4000 positions, 64 rows a key head and 96: bf16 of 128
     * values 28.2 and 30.2, 39.7 and 31.8; f16 28.0 and 35.5, 39.1 and 37.5; f32 of 64
     * 23.1 and 25.0, 31.0 and 30.1. 32 sequences over 2000, 48 rows: 50 and 61 (bf16), 49
     * and 80 (f16). Queries of more bytes lose earlier, 36 rows: bf16 of 256 45.7 and 36.2,
     * f32 of 128 31.9 and 29.8. */
    t->wide = rows > (hd * elem_size(p->type) <= 256 ? 64u : 32u);
    t->tiles = rows > 16 && hd != 256 ? 2u : 1u;
    t->waves = t->wide ? KV8_WIDE_WAVES : KV8_WAVES;
    t->rows = !t->wide ? 16u * t->tiles : p->type == MYNAH_F32 || hd == 256 ? 128u : 256u;
    t->groups = (uint32_t)((rows + t->rows - 1) / t->rows);
    const uint64_t base = (uint64_t)p->cache.n_kv_heads * t->groups;
    const uint32_t chunk = t->wide ? (hd == 256 ? 32u : 64u) : hd * t->tiles >= 256 ? 32u : 64u;
    const uint32_t turn = t->wide ? chunk : KV8_WAVES * chunk;
    /* Pieces enough for every CU, of a turn each at least; and, of 16 turns at least,
     * four workgroups a CU, so that long sequences beside short ones do not set the
     * time alone: 32 of up to 16,384 e4m3 positions 134 us, 144 with two, 186 with one. A
     * sequence cut in two costs 4 to 5 us of a join and as much again in the workgroups: 32
     * of 4000 positions 46 us uncut, 58 cut, 64 of up to 2048 36 and 46. */
    const uint64_t turns = (p->max_kv + turn - 1) / turn;
    uint64_t s = cus / base, more = 4 * cus / base;
    if (s > p->n_seqs * turns) s = p->n_seqs * turns;
    if (more > p->n_seqs * ((turns + 15) / 16)) more = p->n_seqs * ((turns + 15) / 16);
    if (!t->wide && s < more) s = more;
    if (s > 256) s = 256;                       /* four sequences a lane share them */
    t->slots = s > p->n_seqs ? (uint32_t)s : p->n_seqs;
}

static int attn_check(const mynah_kv8_attention *p) {
    if (p == NULL || p->q == NULL || p->out == NULL || p->seq_start == NULL || p->n_past == NULL)
        return refuse("null argument");
    const size_t size = elem_size(p->type);
    if (size == 0) {
        mynah_set_error("kv8_attention: type %d is not f32, f16 or bf16", p->type);
        return -1;
    }
    if (p->n_seqs == 0 || p->n_seqs > 65536 || p->n_rows == 0 || p->n_rows > 0x7fffffffu ||
        p->max_nodes == 0 || p->max_nodes > 65535 || p->max_kv == 0 || p->max_kv > 1u << 26)
        return refuse("kv8_attention: bad counts (sequences, rows, nodes or positions)");
    const mynah_kv8_cache *c = &p->cache;
    if (cache_check(c, p->n_seqs, p->max_kv, "kv8_attention") != 0) return -1;
    if (p->n_heads == 0 || p->n_heads % c->n_kv_heads != 0 || p->n_heads / c->n_kv_heads > 64 ||
        p->n_heads > 65536) {
        mynah_set_error("kv8_attention: %u heads over %u: 1 to 64 heads to a key head are taken",
                        p->n_heads, c->n_kv_heads);
        return -1;
    }
    if (p->mask != NULL && (p->mask_words == 0 || p->max_nodes > 32ull * p->mask_words))
        return refuse("kv8_attention: mask_words too few for max_nodes");
    if (p->mask != NULL && (uint64_t)p->n_rows * p->mask_words > UINT32_MAX)
        return refuse("kv8_attention: a mask of more than 2^32 words");
    const size_t row = (size_t)p->n_heads * c->head_dim;
    if (p->q_stride < row || p->out_stride < row || !fits(p->n_rows, p->q_stride, row, size) ||
        !fits(p->n_rows, p->out_stride, row, size))
        return refuse("kv8_attention: bad stride");
    if ((((uintptr_t)p->q | (uintptr_t)p->out | p->q_stride * size | p->out_stride * size) & 15u) !=
            0 ||
        (((uintptr_t)p->seq_start | (uintptr_t)p->n_past | (uintptr_t)p->mask) & 3u) != 0)
        return refuse("kv8_attention: q, out and strides must be 16-byte aligned");
    if (!isfinite(p->scale)) return refuse("kv8_attention: the scale must be finite");
    kv8_plan t;                                 /* of whole sequences, the most there are */
    make_plan(p, 1, &t);
    if ((uint64_t)p->n_seqs * c->n_kv_heads * t.groups > MYNAH_MOST_WGS(64 * t.waves))
        return refuse("kv8_attention: too many workgroups for one launch");
    return 0;
}

static size_t attn_ws(const mynah_kv8_attention *p, const kv8_plan *t) {
    if (t->slots == p->n_seqs) return 256;
    const size_t rows = (size_t)t->slots * p->cache.n_kv_heads * t->groups * t->rows;
    return rows * (p->cache.head_dim + 2) * sizeof(float) +
           2 * (size_t)p->n_seqs * sizeof(int32_t) + 256;
}

size_t mynah_hip_kv8_attention_workspace(const mynah_kv8_attention *p) {
    if (attn_check(p) != 0) return 0;
    mynah_device *d = mynah_dev();
    if (d == NULL) return 0;
    kv8_plan t;
    make_plan(p, (uint32_t)d->cus, &t);
    return attn_ws(p, &t);
}

int mynah_hip_kv8_attention_dev(const mynah_kv8_attention *p, void *workspace,
                                size_t workspace_bytes, void *stream) {
    if (attn_check(p) != 0) return -1;
    if (workspace == NULL || ((uintptr_t)workspace & 255u) != 0)
        return refuse("kv8_attention: a workspace aligned to 256 bytes is needed");
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    const mynah_kv8_cache *c = &p->cache;
    kv8_plan t;
    make_plan(p, (uint32_t)d->cus, &t);
    if (workspace_bytes < attn_ws(p, &t)) {
        mynah_set_error("kv8_attention: a workspace of %zu bytes, %zu are needed",
                        workspace_bytes, attn_ws(p, &t));
        return -1;
    }
    mynah_kv8_args a;
    memset(&a, 0, sizeof a);
    a.t.q = p->q;
    a.t.k = c->k;
    a.t.v = c->v;
    a.t.out = p->out;
    a.t.q_stride = p->q_stride;
    a.t.out_stride = p->out_stride;
    a.t.slot_stride = c->slot_stride;
    a.t.seq_slots = c->seq_slots;
    a.t.pages = c->pages;
    a.t.seq_start = p->seq_start;
    a.t.n_past = p->n_past;
    a.t.mask = p->mask;
    a.t.wg_rows = t.rows;
    const uint64_t wgs = (uint64_t)t.slots * c->n_kv_heads * t.groups;
    const size_t parts = (size_t)wgs * a.t.wg_rows;
    a.t.po = (float *)workspace;
    a.t.pm = a.t.po + parts * c->head_dim;
    a.t.pl = a.t.pm + parts;
    a.t.plan = (int32_t *)(a.t.pl + parts);
    a.t.n_slots = c->n_slots;
    a.t.n_seqs = p->n_seqs;
    a.t.n_heads = p->n_heads;
    a.t.n_kv = c->n_kv_heads;
    a.t.group = p->n_heads / c->n_kv_heads;
    a.t.n_rows = p->n_rows;
    if (c->pages != NULL) a.t.page_log2 = log2_of(c->page_size);
    a.t.max_pages = c->max_pages;
    a.t.mask_words = p->mask_words;
    a.t.max_nodes = p->max_nodes;
    a.t.max_kv = p->max_kv;
    a.t.slots = t.slots;
    a.t.groups = t.groups;
    a.t.scale2 = 1.0f;                          /* the pieces' references are in log2 units */
    a.ks = c->k_scale;
    a.vs = c->v_scale;
    a.block_log2 = log2_of(c->block);
    /* Queries change sign where the scale is negative. */
    a.scale2 = fminf(fabsf(p->scale) * 1.44269504088896341f, FLT_MAX);
    if (p->scale < 0.0f) a.t.flip = p->type == MYNAH_F32 ? 0x80000000u : 0x80008000u;
    hipStream_t st = mynah_stream_or_default(d, stream);
    void *args[] = {&a}, *join[] = {&a.t};
    const int h = c->head_dim == 64 ? 0 : c->head_dim == 128 ? 1 : 2, ti = type_index(p->type);
    if (mynah_launch(d, t.wide ? MYNAH_K_KV8_WIDE + 6 * ti + 2 * h + c->format
                               : MYNAH_K_KV8_ATTN + 10 * ti + 5 * c->format + 2 * h + (int)t.tiles - 1, (unsigned)wgs, 1,
                     64 * t.waves, 0, st, args) != 0)
        return -1;
    if (t.slots == p->n_seqs) return 0;
    return mynah_launch3(d, MYNAH_K_TREE_JOIN + 3 * ti + h, p->n_seqs, p->max_nodes,
                         (p->n_heads + 3) / 4, 256, 0, st, join);
}
