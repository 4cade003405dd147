/* logits.c — host side of the rules on logits (include/mynah_generate.h;
 * kernels in logits.hip): argument checks and the launch.
 *
 * SPDX-License-Identifier: MIT */
#include "mynah_generate.h"

#include "args.h"

#include <string.h>

int mynah_hip_logits_dev(const mynah_logits *p, void *stream) {
    if (p == NULL || p->x == NULL || p->y == NULL) return refuse("null argument");
    const size_t in = elem_size(p->type), out = elem_size(p->out_type);
    if (in == 0 || out == 0) {
        mynah_set_error("logits: types %d, %d: f32, f16 and bf16 are taken", p->type, p->out_type);
        return -1;
    }
    if (p->n_rows == 0 || p->vocab == 0 || p->vocab > 0x7fffffffu)
        return refuse("logits: bad row count or vocabulary");
    if (p->x_stride < p->vocab || p->y_stride < p->vocab ||
        !fits(p->n_rows, p->x_stride, p->vocab, in) || !fits(p->n_rows, p->y_stride, p->vocab, out))
        return refuse("logits: bad stride");
    if (p->x == p->y && (p->type != p->out_type || p->x_stride != p->y_stride))
        return refuse("logits: in place takes one type and stride");
    if (p->penalty != MYNAH_PENALTY_ONCE && p->penalty != MYNAH_PENALTY_EACH) {
        mynah_set_error("logits: unknown penalty %d", p->penalty);
        return -1;
    }
    if ((p->hist != NULL && p->hist_start == NULL) ||
        (p->bias_id != NULL && (p->bias == NULL || p->bias_start == NULL)))
        return refuse("null argument");
    if (p->allowed != NULL && (uint64_t)p->mask_words * 32 < p->vocab)
        return refuse("logits: mask_words too few for the vocabulary");
    if ((uintptr_t)p->x % in != 0 || (uintptr_t)p->y % out != 0 ||
        (((uintptr_t)p->hist_start | (uintptr_t)p->bias_start) & 7u) != 0 ||
        (((uintptr_t)p->hist | (uintptr_t)p->repeat | (uintptr_t)p->freq |
          (uintptr_t)p->presence | (uintptr_t)p->bias_id | (uintptr_t)p->bias |
          (uintptr_t)p->allowed | (uintptr_t)p->mask_row) & 3u) != 0)
        return refuse("logits: misaligned operand");
    mynah_logits_args a;
    memset(&a, 0, sizeof a);
    a.x = p->x;
    a.y = p->y;
    a.x_stride = p->x_stride;
    a.y_stride = p->y_stride;
    a.hist = p->hist;
    a.hist_start = p->hist_start;
    a.repeat = p->repeat;
    a.freq = p->freq;
    a.presence = p->presence;
    a.bias_id = p->bias_id;
    a.bias = p->bias;
    a.bias_start = p->bias_start;
    a.allowed = p->allowed;
    a.mask_row = p->mask_row;
    a.vocab = p->vocab;
    a.chunks = (p->vocab + MYNAH_LOGITS_CH - 1) / MYNAH_LOGITS_CH;
    a.mask_words = p->mask_words;
    a.n_masks = p->n_masks;
    a.each = p->penalty == MYNAH_PENALTY_EACH;
    /* Whether every run of four elements lies on its own size. */
    a.vec = ((p->x_stride | p->y_stride) & 3u) == 0 && (uintptr_t)p->x % (4 * in) == 0 &&
            (uintptr_t)p->y % (4 * out) == 0;
    const uint64_t wgs = (uint64_t)a.chunks * p->n_rows;
    if (wgs > MYNAH_MOST_WGS(512)) return refuse("logits: too many rows for one launch");
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    void *args[] = {&a};
    return mynah_launch(d, MYNAH_K_LOGITS + 3 * type_index(p->type) + type_index(p->out_type),
                        (unsigned)wgs, 1, 512, 0, mynah_stream_or_default(d, stream), args);
}
