/* attention.c — host side of the attention's operators on their own
 * (include/mynah_attention.h; kernels in rope.hip and tree_attn.hip): argument
 * checks, launch geometry, the rotary frequency table.
 *
 * SPDX-License-Identifier: MIT */
#include "mynah_attention.h"
#include "kernels_hip.h"
#include "runtime_internal.h"

#include <float.h>
#include <math.h>
#include <stdlib.h>
#include <string.h>

#define PI 3.14159265358979323846

static int refuse(const char *what) {
    mynah_set_error("%s", what);
    return -1;
}

static size_t elem_size(int type) {
    return type == MYNAH_F32 ? 4u : type == MYNAH_F16 || type == MYNAH_BF16 ? 2u : 0u;
}

static int type_index(int type) { return type == MYNAH_F32 ? 0 : type == MYNAH_F16 ? 1 : 2; }

/* ── rotary positions ────────────────────────────────────────────────────── */

int mynah_hip_rope_freqs(const mynah_rope_params *p, double *freqs, float *mscale) {
    if (p == NULL || freqs == NULL || mscale == NULL) return refuse("null argument");
    /* Comparisons written so that NaN is refused too. */
    if (p->rot_dim == 0 || p->rot_dim % 2 != 0 || !(p->theta > 1.0) || !isfinite(p->theta) ||
        !(p->mscale >= 0.0) || !isfinite(p->mscale))
        return refuse("rope: rot_dim even, theta above 1 and mscale not negative are needed");
    if (p->scaling < MYNAH_ROPE_NONE || p->scaling > MYNAH_ROPE_BANDS) {
        mynah_set_error("rope: unknown scaling %d", p->scaling);
        return -1;
    }
    const int scaled = p->scaling != MYNAH_ROPE_NONE, ramp = p->scaling >= MYNAH_ROPE_YARN;
    if (scaled && (!(p->factor > 0.0) || !isfinite(p->factor)))
        return refuse("rope: the factor must be above 0");
    if (ramp && (!(p->trained > 0.0) || !isfinite(p->trained) || !(p->low > 0.0) ||
                 !(p->high > p->low) || !isfinite(p->high)))
        return refuse("rope: trained above 0 and high above low above 0 are needed");
    const double r = (double)p->rot_dim;
    double a = 0.0, b = 0.0;
    if (p->scaling == MYNAH_ROPE_YARN) {
        const double d = r / (2.0 * log(p->theta));
        a = fmax(floor(d * log(p->trained / (p->high * 2.0 * PI))), 0.0);
        b = fmin(ceil(d * log(p->trained / (p->low * 2.0 * PI))), r - 1.0);
    }
    for (uint32_t i = 0; i < p->rot_dim / 2; i++) {
        const double f = pow(p->theta, -2.0 * (double)i / r);
        double keep = 1.0;                              /* share of f left as it is */
        if (p->scaling == MYNAH_ROPE_LINEAR) keep = 0.0;
        else if (p->scaling == MYNAH_ROPE_YARN)
            keep = 1.0 - fmin(fmax(((double)i - a) / fmax(b - a, 0.001), 0.0), 1.0);
        else if (p->scaling == MYNAH_ROPE_BANDS)
            keep = fmin(fmax((p->trained * f / (2.0 * PI) - p->low) / (p->high - p->low), 0.0),
                        1.0);
        freqs[i] = scaled ? f / p->factor * (1.0 - keep) + f * keep : f;
    }
    double m = 1.0;
    if (p->mscale > 0.0) m = p->mscale;
    else if (p->scaling == MYNAH_ROPE_YARN && p->factor > 1.0) m = 0.1 * log(p->factor) + 1.0;
    *mscale = (float)m;
    return 0;
}

/* Slots of lanes (one head each) to spread a launch over before one slot takes
 * several heads of its token, whose cos and sin it then computes once. */
#define ROPE_SLOTS 65536u

/* Whether every run of four elements lies on its own size. */
static int seg_vec(const mynah_rope_seg *s, size_t in_size, size_t out_size) {
    return s->heads == 0 ||
           (((s->in_token | s->in_head | s->out_token | s->out_head) & 3u) == 0 &&
            (uintptr_t)s->in % (4u * in_size) == 0 && (uintptr_t)s->out % (4u * out_size) == 0);
}

static int rope_launch(int type, int out_type, int layout, mynah_rope_args *a, size_t tokens,
                       void *stream) {
    a->lanes_log2 = 0;
    while ((8u << a->lanes_log2) < a->hd) a->lanes_log2++;
    a->heads = a->seg[0].heads + a->seg[1].heads + a->seg[2].heads;
    uint32_t each = 1;
    while (each < 8 && tokens * ((a->heads + 2 * each - 1) / (2 * each)) >= ROPE_SLOTS) each *= 2;
    a->groups = (a->heads + each - 1) / each;
    a->units = (unsigned long long)tokens * a->groups;
    const uint32_t per_wg = 256u >> a->lanes_log2;
    const unsigned long long wgs = (a->units + per_wg - 1) / per_wg;
    if (wgs > MYNAH_MOST_WGS(256)) return refuse("rope: too many rows for one launch");
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    int vec = 1;
    for (int i = 0; i < 3; i++)
        vec &= seg_vec(&a->seg[i], elem_size(type), elem_size(out_type));
    uint32_t mode = (layout == MYNAH_ROPE_HALF ? 2u : 0u) | (uint32_t)vec;
    void *args[] = {a, &mode};
    return mynah_launch(d, MYNAH_K_ROPE + 3 * type_index(type) + type_index(out_type),
                        (unsigned)wgs, 1, 256, 0, mynah_stream_or_default(d, stream), args);
}

static int rope_shape(int layout, uint32_t head_dim, uint32_t rot_dim, size_t tokens,
                      size_t heads) {
    if (layout != MYNAH_ROPE_HALF && layout != MYNAH_ROPE_INTERLEAVED) {
        mynah_set_error("rope: unknown layout %d", layout);
        return -1;
    }
    if (head_dim == 0 || head_dim % 8 != 0 || head_dim > 512 || rot_dim == 0 ||
        rot_dim % 8 != 0 || rot_dim > head_dim) {
        mynah_set_error("rope: head_dim %u, rot_dim %u: multiples of 8, rot_dim <= head_dim <= "
                        "512 are taken", head_dim, rot_dim);
        return -1;
    }
    if (tokens == 0 || heads == 0 || heads > 65536 || tokens > 0x7fffffffu)
        return refuse("rope: bad token or head count");
    return 0;
}

/* Whether `n` rows `stride` apart, of `len` elements each, fit the address
 * space in bytes. */
static int fits(size_t n, size_t stride, size_t len, size_t size) {
    return stride <= (SIZE_MAX / 4 / size) / n && len <= SIZE_MAX / 4 / size;
}

/* Whether two of the rows at t * token + h * head, t < tokens, h < heads, of
 * `len` elements each, share an element. Every size is one that
 * fits() takes. */
static int rows_meet(size_t tokens, size_t token, size_t heads, size_t head, size_t len) {
    if ((tokens > 1 && token < len) || (heads > 1 && head < len)) return 1;
    if (tokens == 1 || heads == 1 || token >= (heads - 1) * head + len ||
        head >= (tokens - 1) * token + len)
        return 0;
    for (size_t h = 1; h < heads; h++)                  /* the tokens next to it */
        for (size_t t = h * head / token, i = 0; i < 2 && t + i < tokens; i++) {
            const size_t at = (t + i) * token, to = h * head;
            if ((at > to ? at - to : to - at) < len) return 1;
        }
    return 0;
}

int mynah_hip_rope_dev(int type, int layout, const void *x, size_t x_token, size_t x_head,
                       void *y, size_t y_token, size_t y_head, size_t tokens, size_t heads,
                       uint32_t head_dim, uint32_t rot_dim, const double *freqs, float mscale,
                       const int32_t *pos, void *stream) {
    const size_t size = elem_size(type);
    if (x == NULL || y == NULL || freqs == NULL) return refuse("null argument");
    if (size == 0) {
        mynah_set_error("rope: type %d is not f32, f16 or bf16", type);
        return -1;
    }
    if (rope_shape(layout, head_dim, rot_dim, tokens, heads) != 0) return -1;
    if (!fits(tokens, x_token, head_dim, size) || !fits(heads, x_head, head_dim, size) ||
        !fits(tokens, y_token, head_dim, size) || !fits(heads, y_head, head_dim, size))
        return refuse("size overflow");
    if (rows_meet(tokens, y_token, heads, y_head, head_dim))
        return refuse("rope: rows of y overlap");
    if ((uintptr_t)x % size != 0 || (uintptr_t)y % size != 0 || (uintptr_t)freqs % 8 != 0 ||
        (uintptr_t)pos % 4 != 0)
        return refuse("rope: misaligned operand");
    mynah_rope_args a;
    memset(&a, 0, sizeof a);
    a.seg[0].in = x;
    a.seg[0].out = y;
    a.seg[0].in_token = x_token;
    a.seg[0].in_head = x_head;
    a.seg[0].out_token = y_token;
    a.seg[0].out_head = y_head;
    a.seg[0].heads = (uint32_t)heads;
    a.seg[0].rotate = 1;
    a.freqs = freqs;
    a.pos = pos;
    a.hd = head_dim;
    a.rot = rot_dim;
    a.mscale = mscale;
    return rope_launch(type, type, layout, &a, tokens, stream);
}

int mynah_hip_qk_norm_rope_dev(const mynah_qk_norm_rope *p, void *stream) {
    if (p == NULL) return refuse("null argument");
    const size_t size = elem_size(p->type), out = elem_size(p->out_type);
    if (size == 0 || out == 0) {
        mynah_set_error("qk_norm_rope: types %d, %d: f32, f16 and bf16 are taken", p->type,
                        p->out_type);
        return -1;
    }
    const size_t nq = p->n_heads, nk = p->n_kv_heads, hd = p->head_dim;
    if (rope_shape(p->layout, p->head_dim, p->rot_dim, p->tokens, nq > nk ? nq : nk) != 0)
        return -1;
    if (p->freqs == NULL || (nq && (p->q == NULL || p->q_out == NULL)) ||
        (nk && (p->k == NULL || p->k_cache == NULL)) ||
        (nk && p->v != NULL && p->v_cache == NULL))
        return refuse("null argument");
    if (nk && (p->n_slots == 0 || p->n_slots > 0x7fffffffu))
        return refuse("qk_norm_rope: bad slot count");
    if (!(p->eps >= 0.0f)) return refuse("qk_norm_rope: eps must not be negative");
    if ((nq && (!fits(p->tokens, p->q_stride, nq * hd, size) ||
                !fits(p->tokens, p->q_out_stride, nq * hd, out))) ||
        (nk && (!fits(p->tokens, p->k_stride, nk * hd, size) ||
                !fits(p->tokens, p->v_stride, nk * hd, size) ||
                !fits(p->n_slots, p->slot_stride, nk * hd, out))))
        return refuse("size overflow");
    if ((nq && rows_meet(p->tokens, p->q_out_stride, nq, hd, hd)) ||
        (nk && rows_meet(p->n_slots, p->slot_stride, nk, hd, hd)))
        return refuse("qk_norm_rope: rows of q_out or the caches overlap");
    if ((nq && ((uintptr_t)p->q % size != 0 || (uintptr_t)p->q_out % out != 0)) ||
        (nk && ((uintptr_t)p->k % size != 0 || (uintptr_t)p->v % size != 0 ||
                (uintptr_t)p->k_cache % out != 0 || (uintptr_t)p->v_cache % out != 0)) ||
        (uintptr_t)p->q_norm % 4 != 0 || (uintptr_t)p->k_norm % 4 != 0 ||
        (uintptr_t)p->freqs % 8 != 0 || (uintptr_t)p->pos % 4 != 0 ||
        (uintptr_t)p->slots % 4 != 0)
        return refuse("qk_norm_rope: misaligned operand");
    mynah_rope_args a;
    memset(&a, 0, sizeof a);
    for (int i = 0; i < 3; i++) {
        mynah_rope_seg *s = &a.seg[i];
        if (i == 0 ? nq == 0 : nk == 0 || (i == 2 && p->v == NULL)) continue;
        s->in = i == 0 ? p->q : i == 1 ? p->k : p->v;
        s->out = i == 0 ? p->q_out : i == 1 ? p->k_cache : p->v_cache;
        s->in_token = i == 0 ? p->q_stride : i == 1 ? p->k_stride : p->v_stride;
        s->out_token = i == 0 ? p->q_out_stride : p->slot_stride;
        s->in_head = s->out_head = hd;
        s->norm = i == 0 ? p->q_norm : i == 1 ? p->k_norm : NULL;
        s->heads = (uint32_t)(i == 0 ? nq : nk);
        s->rotate = i < 2;
        s->slotted = i > 0;
    }
    a.freqs = p->freqs;
    a.pos = p->pos;
    a.slots = p->slots;
    a.n_slots = (uint32_t)p->n_slots;
    a.hd = p->head_dim;
    a.rot = p->rot_dim;
    a.eps = p->eps;
    a.mscale = p->mscale;
    return rope_launch(p->type, p->out_type, p->layout, &a, p->tokens, stream);
}

/* ── attention of drafted tokens over a cache ────────────────────────────── */

/* What a call launches: kernel `variant` of its type and head size, 16 * nt query
 * rows for each of rw row waves, `waves` waves a workgroup, a workgroup for each
 * key head, group of rows and slot: a sequence's, or with more slots than sequences a
 * piece of one. */
typedef struct {
    uint32_t variant, nt, rw, waves, groups, slots;
} tree_plan;

static void tree_make_plan(const mynah_tree_attention *p, uint32_t cus, tree_plan *t);

static int tree_check(const mynah_tree_attention *p) {
    if (p == NULL || p->q == NULL || p->out == NULL || p->k_cache == NULL ||
        p->v_cache == NULL || p->seq_start == NULL || p->n_past == NULL)
        return refuse("null argument");
    const size_t size = elem_size(p->type), hd = p->head_dim;
    if (size == 0) {
        mynah_set_error("tree_attention: type %d is not f32, f16 or bf16", p->type);
        return -1;
    }
    if ((hd != 64 && hd != 128 && hd != 256) || p->n_kv_heads == 0 ||
        p->n_heads % p->n_kv_heads != 0 || p->n_heads / p->n_kv_heads < 1 ||
        p->n_heads / p->n_kv_heads > 64 || p->n_heads > 65536) {
        mynah_set_error("tree_attention: %u heads over %u of %u values: head_dim 64, 128 or 256 "
                        "and 1 to 64 heads to a key head are taken", p->n_heads, p->n_kv_heads,
                        p->head_dim);
        return -1;
    }
    if (p->n_seqs == 0 || p->n_seqs > 65536 || p->n_rows == 0 || p->n_rows > 0x7fffffffu ||
        p->max_nodes == 0 || p->max_nodes > 65535 || p->max_kv == 0 || p->max_kv > 1u << 26 ||
        p->n_slots == 0 || p->n_slots > (size_t)1 << 40)
        return refuse("tree_attention: bad counts (sequences, rows, nodes, positions or slots)");
    if (p->mask != NULL && (p->mask_words == 0 || p->max_nodes > 32ull * p->mask_words))
        return refuse("tree_attention: mask_words too few for max_nodes");
    if (p->mask != NULL && (uint64_t)p->n_rows * p->mask_words > UINT32_MAX)
        return refuse("tree_attention: a mask of more than 2^32 words");
    if (p->pages != NULL) {
        if (p->page_size < 16 || (p->page_size & (p->page_size - 1)) != 0)
            return refuse("tree_attention: page_size must be a power of two from 16 on");
        if ((uint64_t)p->max_pages * p->page_size < p->max_kv)
            return refuse("tree_attention: max_kv positions do not fit the page table");
    } else if (p->n_seqs > 1 && p->seq_slots > ((size_t)1 << 40) / p->n_seqs) {
        return refuse("tree_attention: bad seq_slots");
    }
    const size_t qh = p->n_heads * hd, kh = p->n_kv_heads * hd;
    if (p->q_stride < qh || p->out_stride < qh || p->slot_stride < kh ||
        p->slot_stride >= ((size_t)1 << 24) / size || !fits(p->n_rows, p->q_stride, qh, size) ||
        !fits(p->n_rows, p->out_stride, qh, size))
        return refuse("tree_attention: bad stride");
    if ((((uintptr_t)p->q | (uintptr_t)p->out | (uintptr_t)p->k_cache | (uintptr_t)p->v_cache) &
         15u) != 0 ||
        ((p->q_stride | p->out_stride | p->slot_stride) * size & 15u) != 0 ||
        (((uintptr_t)p->pages | (uintptr_t)p->seq_start | (uintptr_t)p->n_past |
          (uintptr_t)p->mask) & 3u) != 0)
        return refuse("tree_attention: q, out, caches and strides must be 16-byte aligned");
    if (!isfinite(p->scale)) return refuse("tree_attention: the scale must be finite");
    tree_plan t;                                /* of whole sequences, the most there are */
    tree_make_plan(p, 1, &t);
    if ((uint64_t)p->n_seqs * p->n_kv_heads * t.groups > MYNAH_MOST_WGS(64 * t.waves))
        return refuse("tree_attention: too many workgroups for one launch");
    return 0;
}

static void tree_make_plan(const mynah_tree_attention *p, uint32_t cus, tree_plan *t) {
    const uint32_t group = p->n_heads / p->n_kv_heads;
    const uint64_t tiles = ((uint64_t)p->max_nodes * group + 15) / 16;
    const int f32 = p->type == MYNAH_F32, wide = p->head_dim == 256;
    t->waves = wide ? 4u : 8u;
    t->nt = 1;
    if (f32) {
        /* More row waves leave a workgroup fewer keys at a time and more of them
         * idle at the ends: 96 rows over 2072 positions, 22 us with two, 30 with
         * four, 35 with eight. */
        t->variant = tiles > 1 ? 1u : 0u;
        t->rw = t->variant + 1u;
    } else if (wide) {
        t->variant = tiles > 2 ? 2u : (uint32_t)tiles - 1u;
        t->rw = 1u << t->variant;
    } else {
        /* Every row of the call in one workgroup as far as that goes, for its keys
         * then come from memory once: 256 rows over 130,001 positions, 202 us with
         * 2 x 8 tiles, 278 with every wave on keys of its own. */
        t->variant = tiles > 8 ? 4u : tiles > 4 ? 3u : tiles > 2 ? 2u : (uint32_t)tiles - 1u;
        if (t->variant == 4u && p->head_dim == 64) t->variant = 3u;
        t->nt = t->variant > 1u ? 2u : 1u;
        t->rw = t->variant == 0u ? 1u : 1u << (t->variant - (t->nt == 2u));
    }
    t->groups = (uint32_t)((tiles + t->nt * t->rw - 1) / (t->nt * t->rw));
    /* At most one workgroup for each CU. A 128- or 256-wide one of one or two row
     * waves fills its LDS: 264 on 256 CUs took 39 us where 240 take 22, and two or
     * three a CU, one after the other, are slower too (16 sequences of up to 8207 bf16
     * positions cut alike 99, 109 and 121 us). Two of head size 64 fit, and gain and
     * lose: bf16, one node over 65,536 positions 43 us with two, 37 with one, the 16
     * sequences 60 and 55; f32, 64 nodes over 130,000 586 and 657.
     * So where sequences times key heads times row groups reach the CUs, nothing is
     * cut, and the longest sequence has the call to itself: one of 32,768 bf16
     * positions beside 15 of 512 47 us, beside 30 196 (one piece to spare), beside 31
     * to 63 345 to 353. */
    const uint64_t base = (uint64_t)p->n_kv_heads * t->groups;
    const uint32_t turn = t->waves / t->rw * (f32 ? 16u : 32u) * (t->rw > 1 ? 2u : 1u);
    const uint64_t turns = (uint64_t)p->n_seqs * ((p->max_kv + turn - 1) / turn);
    uint64_t s = cus / base;
    if (s > turns) s = turns;
    if (s > 256) s = 256;                       /* four sequences a lane share them */
    t->slots = s > p->n_seqs ? (uint32_t)s : p->n_seqs;
}

static size_t tree_ws(const mynah_tree_attention *p, const tree_plan *t) {
    if (t->slots == p->n_seqs) return 256;
    const size_t rows = (size_t)t->slots * p->n_kv_heads * t->groups * 16 * t->nt * t->rw;
    return rows * (p->head_dim + 2) * sizeof(float) + 2 * (size_t)p->n_seqs * sizeof(int32_t) + 256;
}

size_t mynah_hip_tree_attention_workspace(const mynah_tree_attention *p) {
    if (tree_check(p) != 0) return 0;
    mynah_device *d = mynah_dev();
    if (d == NULL) return 0;
    tree_plan t;
    tree_make_plan(p, (uint32_t)d->cus, &t);
    return tree_ws(p, &t);
}

static int tree_kernel(const mynah_tree_attention *p, uint32_t variant) {
    /* The first variant of head sizes 64, 128 and 256, in the kernel ids' order. */
    static const int first[2][3] = {{0, 4, 9}, {0, 2, 4}};
    const int h = p->head_dim == 64 ? 0 : p->head_dim == 128 ? 1 : 2, f32 = p->type == MYNAH_F32;
    const int type = f32 ? MYNAH_K_TREE_F32
                         : p->type == MYNAH_F16 ? MYNAH_K_TREE_F16 : MYNAH_K_TREE_BF16;
    return type + first[f32][h] + (int)variant;
}

int mynah_hip_tree_attention_dev(const mynah_tree_attention *p, void *workspace,
                                 size_t workspace_bytes, void *stream) {
    if (tree_check(p) != 0) return -1;
    if (workspace == NULL || ((uintptr_t)workspace & 255u) != 0)
        return refuse("tree_attention: a workspace aligned to 256 bytes is needed");
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    tree_plan t;
    tree_make_plan(p, (uint32_t)d->cus, &t);
    if (workspace_bytes < tree_ws(p, &t)) {
        mynah_set_error("tree_attention: a workspace of %zu bytes, %zu are needed",
                        workspace_bytes, tree_ws(p, &t));
        return -1;
    }
    mynah_tree_args a;
    memset(&a, 0, sizeof a);
    a.q = p->q;
    a.k = p->k_cache;
    a.v = p->v_cache;
    a.out = p->out;
    a.q_stride = p->q_stride;
    a.out_stride = p->out_stride;
    a.slot_stride = p->slot_stride;
    a.seq_slots = p->seq_slots;
    a.pages = p->pages;
    a.seq_start = p->seq_start;
    a.n_past = p->n_past;
    a.mask = p->mask;
    a.wg_rows = 16 * t.nt * t.rw;
    const uint64_t wgs = (uint64_t)t.slots * p->n_kv_heads * t.groups;
    const size_t parts = (size_t)wgs * a.wg_rows;
    a.po = (float *)workspace;
    a.pm = a.po + parts * p->head_dim;
    a.pl = a.pm + parts;
    a.plan = (int32_t *)(a.pl + parts);
    a.n_slots = p->n_slots;
    a.n_seqs = p->n_seqs;
    a.n_heads = p->n_heads;
    a.n_kv = p->n_kv_heads;
    a.group = p->n_heads / p->n_kv_heads;
    a.n_rows = p->n_rows;
    if (p->pages != NULL)
        while ((1u << a.page_log2) < p->page_size) a.page_log2++;
    a.max_pages = p->max_pages;
    a.mask_words = p->mask_words;
    a.max_nodes = p->max_nodes;
    a.max_kv = p->max_kv;
    a.slots = t.slots;
    a.groups = t.groups;
    /* Queries change sign where the scale is negative; no scale counts as a
     * very small one (a score of 0 within 2^-20 for products up to 10^24), so
     * that -inf stays what it is. */
    a.scale2 = fminf(fabsf(p->scale) * 1.44269504088896341f, FLT_MAX);
    if (a.scale2 < 1e-30f) a.scale2 = 1e-30f;
    a.lag = (p->type == MYNAH_F16 ? 4.0f : 8.0f) / a.scale2;   /* 2^11 2^4 fits an f16 */
    if (p->scale < 0.0f) a.flip = p->type == MYNAH_F32 ? 0x80000000u : 0x80008000u;
    hipStream_t st = mynah_stream_or_default(d, stream);
    void *args[] = {&a};
    if (mynah_launch(d, tree_kernel(p, t.variant), (unsigned)wgs, 1, 64 * t.waves, 0, st, args) != 0)
        return -1;
    if (t.slots == p->n_seqs) return 0;
    const int h = p->head_dim == 64 ? 0 : p->head_dim == 128 ? 1 : 2;
    return mynah_launch3(d, MYNAH_K_TREE_JOIN + 3 * type_index(p->type) + h, p->n_seqs,
                         p->max_nodes, (p->n_heads + 3) / 4, 256, 0, st, args);
}
