/* mynah_attention.h — the attention's operators on their own: rotary
 * positions, the norms of query and key heads with the rotation in the same
 * pass, and the attention of drafted tokens over a key/value cache, for a
 * caller that keeps its own projections and caches. The resident decoder
 * (mynah_decode.h) checks drafted tokens through the same kernels
 * (mynah_hip_qwen3_verify). No reference counterpart: the reference has f32
 * forms of these for one sequence and one token (src/kernels.c:141-293).
 *
 * Element types are ggml's ids: F32 = 0, F16 = 1, BF16 = 30. Strides count
 * elements. All pointers are device pointers unless said otherwise; calls are
 * asynchronous on `stream` (a hipStream_t as void *, NULL = the library's own
 * stream), allocate nothing and may be captured into a HIP graph. 0, or -1
 * with the reason in mynah_hip_last_error() and nothing launched.
 *
 * SPDX-License-Identifier: MIT */
#ifndef MYNAH_ATTENTION_H
#define MYNAH_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { MYNAH_F32 = 0, MYNAH_F16 = 1, MYNAH_BF16 = 30 };

/* ── rotary positions ──────────────────────────────────────────────────── */

/* Which values of a head make pair i < rot_dim / 2: (i, i + rot_dim / 2), as
 * the reference's decoder pairs them (src/kernels.c:141-164), or
 * (2 i, 2 i + 1). Values from rot_dim on are copied. */
enum { MYNAH_ROPE_HALF = 0, MYNAH_ROPE_INTERLEAVED = 1 };

/* How the frequencies f_i = theta^(-2 i / rot_dim) are stretched for contexts
 * `factor` times as long as the trained one (`trained` positions):
 *   NONE    f_i;
 *   LINEAR  f_i / factor;
 *   YARN    a ramp over the pairs: with pair(n) = rot_dim ln(trained / (2 pi n))
 *           / (2 ln theta), the pair that turns n times over the trained
 *           context, a = max(floor(pair(high)), 0), b = min(ceil(pair(low)),
 *           rot_dim - 1) and g_i = (i - a) / max(b - a, 0.001) clamped to
 *           [0, 1]: f_i (1 - g_i) + f_i / factor g_i;
 *   BANDS   by wavelength: with g_i = (trained f_i / (2 pi) - low) /
 *           (high - low) clamped to [0, 1]: f_i g_i + f_i / factor (1 - g_i).
 * YARN multiplies cos and sin by 0.1 ln(factor) + 1 (factor > 1); mscale > 0
 * replaces that, or the 1 of the other methods. */
enum { MYNAH_ROPE_NONE = 0, MYNAH_ROPE_LINEAR = 1, MYNAH_ROPE_YARN = 2, MYNAH_ROPE_BANDS = 3 };

typedef struct {
    uint32_t rot_dim;        /* rotated values of a head: even, not 0 */
    int scaling;             /* MYNAH_ROPE_NONE .. MYNAH_ROPE_BANDS */
    double theta;            /* > 1 */
    double factor;           /* > 0; unused by NONE */
    double trained;          /* YARN, BANDS: > 0 */
    double high, low;        /* YARN (turns), BANDS (divisors of `trained`): high > low > 0 */
    double mscale;           /* 0: the method's own */
} mynah_rope_params;

/* Host only, no device needed: the radians per position of each pair into
 * freqs[rot_dim / 2] (host) and the factor of cos and sin into *mscale. The
 * operators below take the table as a device array, so any other table (one
 * read from a checkpoint) does as well. */
int mynah_hip_rope_freqs(const mynah_rope_params *p, double *freqs, float *mscale);

/* y = x rotated: row (t, h) of x starts at x + t * x_token + h * x_head and
 * holds head_dim values; y alike. Pair i turns by pos[t] * freqs[i] (the
 * product and its reduction to one turn in 64 bits, so far positions keep
 * their angle; cos and sin in 32), scaled by mscale; the result is rounded
 * once to `type`. pos[t] may be negative (a rotation back); NULL: t itself.
 * y may be x with the same strides; otherwise they do not overlap. Rows of y
 * that overlap one another are refused; rows of x may (one for all tokens).
 * head_dim and rot_dim multiples of 8, rot_dim <= head_dim <= 512; tokens and
 * heads not 0. */
int mynah_hip_rope_dev(int type, int layout, const void *x, size_t x_token, size_t x_head,
                       void *y, size_t y_token, size_t y_head, size_t tokens, size_t heads,
                       uint32_t head_dim, uint32_t rot_dim, const double *freqs, float mscale,
                       const int32_t *pos, void *stream);

/* ── norms of query and key heads, rotation, cache slots, in one pass ──── */

/* For every token t: query head h becomes q_out[t][h] = rope(norm(q[t][h])),
 * key head h goes to k_cache[slots[t]][h] = rope(norm(k[t][h])) and value head
 * h to v_cache[slots[t]][h], norm(x) = x / sqrt(mean(x^2) + eps) * w in 32 bits
 * (w NULL: no norm). Rows of a token lie head after head; a slot's rows too.
 *   - inputs are of `type`, q_out and the caches of `out_type`;
 *   - n_heads 0: no queries (q, q_out unused); n_kv_heads 0: no keys; v NULL:
 *     no values;
 *   - slots[t] outside [0, n_slots): the token's key and value are not stored
 *     (padding rows of a batch); slots NULL: token t to slot t. The slots of a
 *     call are distinct: of two tokens with one slot, each value left there is
 *     one token's or the other's;
 *   - the outputs do not overlap the inputs; strides that let rows of q_out or
 *     slots overlap one another are refused. */
typedef struct {
    int type, out_type, layout;
    uint32_t n_heads, n_kv_heads, head_dim, rot_dim;   /* as for mynah_hip_rope_dev */
    size_t tokens;
    const void *q, *k, *v;
    size_t q_stride, k_stride, v_stride;               /* between tokens */
    const float *q_norm, *k_norm;                      /* [head_dim] */
    float eps, mscale;
    const double *freqs;
    const int32_t *pos;
    const int32_t *slots;
    size_t n_slots;
    void *q_out;
    size_t q_out_stride;
    void *k_cache, *v_cache;
    size_t slot_stride;
} mynah_qk_norm_rope;

int mynah_hip_qk_norm_rope_dev(const mynah_qk_norm_rope *a, void *stream);

/* ── attention of drafted tokens over a cache ──────────────────────────── */

/* n_seqs sequences; sequence b owns the query rows seq_start[b] ..
 * seq_start[b + 1] - 1 of q and out (its nodes 0, 1, ..., heads side by side)
 * and attends n_past[b] + nodes positions of its cache: the n_past[b]
 * committed ones, which every node sees, then its own nodes' keys, of which
 * node i sees node j where bit j % 32 of mask[row of i][j / 32] is set.
 *   out[row][h] = sum_p softmax_p(scale q[row][h] . k[p][h / group]) v[p][h / group]
 * over the seen positions p, group = n_heads / n_kv_heads; a row that sees
 * nothing, or scores of -inf only, is 0. Unseen positions have no effect,
 * whatever their keys and values hold. mask NULL: node i sees nodes 0 .. i (a chain: several tokens
 * in order, or one). Statistics and sums are held in 32 bits; of 16-bit types
 * the probabilities are rounded to the type for the product with V (f16: of n
 * positions, those below 2^-25 of the row's largest are off by n 2^-36 of it
 * together at most), the result once. The sums' order depends on the sizes,
 * max_* values and lengths alone, so equal calls give equal bits. Sequences are
 * cut by their lengths over the CUs while n_seqs times n_kv_heads is below their
 * number (times row groups, where a key head has more rows, max_nodes * group, than
 * a workgroup takes: 32 in f32, 64 to 256 in 16 bits); from there on a sequence is
 * not cut and the longest one sets the time.
 *   - position p of sequence b is cache row pages[b][p / page_size] * page_size
 *     + p % page_size, or without pages b * seq_slots + p; a row outside
 *     [0, n_slots) (a page id that is no page) is not read and counts as unseen;
 *   - n_past, seq_start, pages and mask are read on the device, so a captured
 *     call follows them; max_nodes and max_kv bound nodes and n_past + nodes
 *     of every sequence: nodes past max_nodes are left out (their rows of out
 *     as they were, their keys unseen), positions past max_kv are unseen; rows
 *     of no sequence are left as they were, rows outside [0, n_rows) are not
 *     touched, and a negative n_past counts as 0;
 *   - out overlaps none of the inputs;
 *   - head_dim 64, 128 or 256; 1 <= n_heads / n_kv_heads <= 64; page_size a
 *     power of two from 16 on; q, out, caches and strides aligned to 16 bytes;
 *     slot_stride below 2^24 bytes; n_seqs and n_heads <= 65536, max_nodes
 *     <= 65535, max_kv <= 2^26, and with a mask max_nodes <= 32 *
 *     mask_words and n_rows * mask_words < 2^32. */
typedef struct {
    int type;                                   /* of q, out and the caches */
    uint32_t n_seqs, n_heads, n_kv_heads, head_dim;
    const void *q;
    size_t q_stride;                            /* between query rows */
    void *out;
    size_t out_stride;
    uint32_t n_rows;                            /* rows of q and out */
    const void *k_cache, *v_cache;
    size_t slot_stride;                         /* between cache rows */
    size_t n_slots;                             /* cache rows */
    size_t seq_slots;                           /* without pages: rows between sequences */
    const int32_t *pages;                       /* [n_seqs][max_pages], or NULL */
    uint32_t page_size, max_pages;
    const int32_t *seq_start;                   /* [n_seqs + 1] */
    const int32_t *n_past;                      /* [n_seqs] */
    const uint32_t *mask;                       /* [n_rows][mask_words], or NULL */
    uint32_t mask_words, max_nodes, max_kv;
    float scale;
} mynah_tree_attention;

/* Bytes of device workspace (aligned to 256 bytes) the call needs: partial
 * results of positions split over workgroups. 0 with the reason in
 * mynah_hip_last_error() where the arguments are refused; at least 256
 * otherwise. Calls that may overlap need workspaces of their own: two streams,
 * or two captured graphs that replay at the same time. */
size_t mynah_hip_tree_attention_workspace(const mynah_tree_attention *a);
int mynah_hip_tree_attention_dev(const mynah_tree_attention *a, void *workspace,
                                 size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
