/* mynah_cache.h — a server's key/value cache in 8 bits: storing new rows,
 * attention over it, and the pages it lives in. No reference counterpart: the
 * reference keeps one sequence's cache in f32 (src/arch_qwen3.c:89-131).
 *
 * A cache row holds one position of one layer, its heads side by side, a byte a
 * value. Each `block` rows (a run that starts at a multiple of `block`) share one
 * f32 scale for each head, of keys and of values: value = code * scale. A server's
 * step is: rows for the new tokens (mynah_hip_pages_reserve_dev), their keys and
 * values (mynah_hip_kv8_store_dev), the attention that reads them
 * (mynah_hip_kv8_attention_dev).
 *
 * Element types are ggml's ids: F32 = 0, F16 = 1, BF16 = 30. Strides count
 * elements. All pointers are device pointers unless said otherwise; calls are
 * asynchronous on `stream` (a hipStream_t as void *, NULL = the library's own
 * stream), allocate nothing and may be captured into a HIP graph. 0, or -1
 * with the reason in mynah_hip_last_error() and nothing launched.
 *
 * SPDX-License-Identifier: MIT */
#ifndef MYNAH_CACHE_H
#define MYNAH_CACHE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* What a code stands for: a signed integer, or e4m3 (one sign, four exponent,
 * three mantissa bits, no infinities, largest value 448). */
enum { MYNAH_KV_I8 = 0, MYNAH_KV_E4M3 = 1 };

/* Position p of sequence b is cache row pages[b][p / page_size] * page_size + p %
 * page_size, or without pages b * seq_slots + p. A row outside [0, n_slots) (a
 * page id that is no page) is not touched, and counts as unseen.
 *   - head_dim 64, 128 or 256; block a power of two from 16 to 256 that divides
 *     n_slots and, without pages and with more than one sequence, seq_slots;
 *     page_size a power of two, block at least;
 *   - k, v and slot_stride (bytes, heads * head_dim at least, below 2^24) are
 *     multiples of 16; n_slots <= 2^40. */
typedef struct {
    int format;                                 /* MYNAH_KV_I8 or MYNAH_KV_E4M3 */
    uint32_t n_kv_heads, head_dim, block;
    uint8_t *k, *v;                             /* [n_slots], slot_stride apart */
    size_t slot_stride, n_slots;
    float *k_scale, *v_scale;                   /* [n_slots / block][n_kv_heads] */
    size_t seq_slots;                           /* without pages: rows between sequences */
    const int32_t *pages;                       /* [n_seqs][max_pages], or NULL */
    uint32_t page_size, max_pages;
} mynah_kv8_cache;

/* ── new rows into the cache ───────────────────────────────────────────── */

/* Sequence b's new tokens are rows seq_start[b] .. seq_start[b + 1] - 1 of k and
 * v and go to its positions n_past[b], n_past[b] + 1, ... For every block that
 * gets rows and every head, with x the call's new values there:
 *   amax   = max(2^-100, largest |x| that is finite)
 *   scale  = amax / 127 (I8); the least power of two with amax / 448 <= scale (E4M3)
 *   code   = round(x * (1 / scale)), to nearest, ties to even
 * each operation in 32 bits. Where the block has positions before n_past[b], its
 * old scale (0 unless positive and finite) is a lower bound of the new one, and if
 * the scale grows their codes become round(code * (old / scale)): of E4M3, whose
 * scales are powers of two, the same values but for those that fall below its
 * normal range. So earlier positions keep their values to half a step of the new
 * scale, and rows at and behind n_past[b] before the call count for nothing.
 * Infinities take the largest code, a NaN 0: every value of a cache that this call
 * filled is finite. All other rows stay as they were (of a block that is not full
 * the rows behind the new ones, too).
 *   - n_past, seq_start and pages are read on the device, so a captured call
 *     follows them; seq_start rises; max_nodes bounds a sequence's new tokens and max_kv its
 *     positions: tokens past either are not stored; a negative n_past counts as 0;
 *     token rows outside [0, n_rows) are not stored;
 *   - the blocks written are distinct: no two sequences of a call write to the
 *     same page (mynah_hip_pages_reserve_dev sees to that), and without pages more
 *     than one sequence with max_kv above seq_slots is refused;
 *   - k, v and their strides aligned to 16 bytes; the cache overlaps neither;
 *     n_seqs <= 65536, max_nodes <= 2^24, max_kv <= 2^26. */
typedef struct {
    mynah_kv8_cache cache;
    int type;                                   /* of k and v */
    uint32_t n_seqs;
    const void *k, *v;                          /* new rows, heads side by side */
    size_t k_stride, v_stride;
    uint32_t n_rows;                            /* rows of k and v */
    const int32_t *seq_start;                   /* [n_seqs + 1] */
    const int32_t *n_past;                      /* [n_seqs] */
    uint32_t max_nodes, max_kv;
} mynah_kv8_store;

int mynah_hip_kv8_store_dev(const mynah_kv8_store *a, void *stream);

/* ── attention over the cache ──────────────────────────────────────────── */

/* As mynah_hip_tree_attention_dev (mynah_attention.h), over 8-bit keys and
 * values: sequence b owns the query rows seq_start[b] .. seq_start[b + 1] - 1 of q
 * and out (its nodes 0, 1, ...) and attends n_past[b] + nodes positions of its
 * cache: the n_past[b] committed ones, which every node sees, then its own
 * nodes', of which node i sees node j where bit j % 32 of mask[row of i][j / 32]
 * is set; mask NULL: nodes 0 .. i, so a prompt's tokens, a draft's, or one.
 *   out[row][h] = sum_p softmax_p(scale q[row][h] . k[p][h / group]) v[p][h / group]
 * over the seen positions, group = n_heads / n_kv_heads; a row that sees nothing is
 * 0. Unseen positions have no effect, whatever their codes are. A scale that is
 * not positive and finite counts as 0. An e4m3 NaN among the keys or the committed
 * values makes the rows that see it NaN; among the nodes' values it counts as 0.
 * Probabilities below 2^-126 of a row's largest count as 0, and so does what of a
 * weight (probability times value's scale) is below 2^-126.
 *
 * Codes are widened exactly, and products of f32 and f16 queries keep all their
 * bits (of f32 queries below 2^-100 in size the upper ones); scores, statistics and
 * sums are held in 32 bits. Each probability times its value's scale is rounded for
 * the product with V: of f32 queries not at all, of f16 to 16 bits, of bf16 to 16 where
 * max_nodes times group is 64 at most (32 with head_dim 256), to 8 from there on; the
 * result once, to `type`.
 * The sums' order depends on the sizes, max_* values and lengths alone, so equal calls
 * give equal bits.
 *
 * A call is planned for max_nodes: kernels of many rows a key head (max_nodes times
 * group above 64, or 32 where a query head is more than 256 bytes) leave a long sequence
 * of one token to one workgroup a head. Where prompts and single tokens come together,
 * one call for each kind is faster (seq_start, n_past and pages from a sequence on).
 * Up to 255 sequences are cut by their lengths over the CUs while n_seqs times
 * n_kv_heads times row groups is below the CUs' number, with few rows four times that;
 * otherwise none is cut and the longest one sets the time: one of 130,000 positions beside
 * 159 of 1000 1300 us (8 key heads, few rows), beside 100 of them 200. A call of
 * its own for the long ones is faster.
 *   - n_past, seq_start, pages and mask are read on the device; max_nodes and
 *     max_kv, rows outside [0, n_rows) and of no sequence, and a negative n_past as
 *     for the tree attention;
 *   - sequences may share cache rows (pages of one prefix, or without pages seq_slots
 *     below max_kv, 0 for all the same rows);
 *   - out overlaps none of the inputs; queries are below 2^110 in size (their products
 *     with codes are summed before any scale), scores (scale q . k) below 2^29, values
 *     (code times scale) below 2^93: up to 2^26 positions' probabilities, up to 2^8
 *     before they are divided by their sum, meet in 32 bits;
 *   - 1 <= n_heads / n_kv_heads <= 64; q, out and strides aligned to 16 bytes;
 *     n_seqs and n_heads <= 65536, max_nodes <= 65535, max_kv <= 2^26, and
 *     with a mask max_nodes <= 32 * mask_words and n_rows * mask_words < 2^32. */
typedef struct {
    mynah_kv8_cache cache;
    int type;                                   /* of q and out */
    uint32_t n_seqs, n_heads;
    const void *q;
    size_t q_stride;                            /* between query rows */
    void *out;
    size_t out_stride;
    uint32_t n_rows;                            /* rows of q and out */
    const int32_t *seq_start;                   /* [n_seqs + 1] */
    const int32_t *n_past;                      /* [n_seqs] */
    const uint32_t *mask;                       /* [n_rows][mask_words], or NULL */
    uint32_t mask_words, max_nodes, max_kv;
    float scale;
} mynah_kv8_attention;

/* Bytes of device workspace (aligned to 256 bytes) the call needs: partial
 * results of positions split over workgroups. 0 with the reason in
 * mynah_hip_last_error() where the arguments are refused; at least 256
 * otherwise. Calls that may overlap need workspaces of their own: two streams,
 * or two captured graphs that replay at the same time. */
size_t mynah_hip_kv8_attention_workspace(const mynah_kv8_attention *a);
int mynah_hip_kv8_attention_dev(const mynah_kv8_attention *a, void *workspace,
                                size_t workspace_bytes, void *stream);

/* ── the pages of a cache ──────────────────────────────────────────────── */

/* A part of a page: page p's is `bytes` bytes from base + p * stride on (a layer's
 * keys, its values, their scales). Parts do not overlap. */
typedef struct {
    void *base;
    size_t stride, bytes;
} mynah_page_part;

/* A pool of pages and the sequences that hold them. Sequence b's positions p lie in
 * page pages[b][p / page_size], entries behind its pages are -1; several sequences
 * may hold a page, refs[p] counts the table's entries that name page p, and a page
 * of 0 is free. The calls keep that so. Everything is device memory and is read
 * there, so a captured call follows it; the calls of a pool go one after the other
 * (one stream, or events). Entries outside [0, n_pages) name no page.
 * n_seqs <= 65536, n_parts <= 65534, n_seqs * max_pages and n_pages < 2^28,
 * page_size a power of two. */
typedef struct {
    uint32_t n_pages, n_seqs, max_pages, page_size, n_parts;
    const mynah_page_part *parts;               /* [n_parts] */
    int32_t *refs;                              /* [n_pages] */
    int32_t *pages;                             /* [n_seqs][max_pages] */
    int32_t *n_past;                            /* [n_seqs]: positions held */
    int32_t *status;                            /* [2] */
} mynah_page_pool;

/* Bytes of device workspace (aligned to 256 bytes) that a call of this pool needs;
 * 0 with the reason in mynah_hip_last_error() where the pool is refused. */
size_t mynah_hip_pages_workspace(const mynah_page_pool *p);

/* Every sequence b becomes what sequence from[b] was before the call, or empty where
 * from[b] is outside [0, n_seqs): its pages are shared, not copied, those that b held
 * are given back. from[b] = b leaves b alone; any number may continue one (beams,
 * samples of one prompt), in any order. */
int mynah_hip_pages_fork_dev(const mynah_page_pool *p, const int32_t *from, void *workspace,
                             size_t workspace_bytes, void *stream);

/* Every sequence b gets pages of its own for positions n_past[b] .. n_past[b] +
 * n_new[b] - 1 (n_new[b] <= 0: none are asked for): an entry there that names no page
 * gets a free one, and one whose page others hold too gets a free one with, where it has
 * positions before n_past[b], a copy of the page's content. If every holder of a page asks
 * for it, the first keeps it. Free pages are given from the lowest on, in the order of
 * sequences and positions. n_past stays as it is. status[0] is the number of pages
 * that were missing, status[1] of sequences that would not fit max_pages entries: unless
 * both are 0, nothing has changed. The time grows with n_seqs times the most entries that
 * one sequence asks for: room for a token for each of 256 sequences 5 us, with 125 pages
 * for one of them 112 us, with 512 373. */
int mynah_hip_pages_reserve_dev(const mynah_page_pool *p, const int32_t *n_new, void *workspace,
                                size_t workspace_bytes, void *stream);

/* Every sequence b with keep[b] >= 0 is cut to at most keep[b] positions (0: it is
 * gone), and its pages behind those of keep[b] positions are given back, reserved ones
 * too. */
int mynah_hip_pages_release_dev(const mynah_page_pool *p, const int32_t *keep, void *stream);

/* The n pages in use move into the pages 0 .. n - 1: each page from n on, in rising
 * order, to the lowest free one, content, counts and table alike; the pages from n on
 * are free then. status[0] becomes n, status[1] the number of pages that moved. One
 * workgroup plans it over all pages: next to no content, 12 us for 640 pages, 85 for
 * 40,000. */
int mynah_hip_pages_compact_dev(const mynah_page_pool *p, void *workspace,
                                size_t workspace_bytes, void *stream);

/* The content of page from[i] to page to[i], i < n, all parts; the table and the
 * counts stay. Pairs with an index outside [0, n_pages) are left out. No page is
 * twice among `to`, nor in both. */
int mynah_hip_pages_copy_dev(const mynah_page_pool *p, const int32_t *from, const int32_t *to,
                             uint32_t n, void *stream);

#ifdef __cplusplus
}
#endif
#endif
