/* pages.c — host side of a cache's pages (include/mynah_cache.h; kernels in
 * pages.hip): argument checks, the workspace, launches.
 *
 * SPDX-License-Identifier: MIT */
#include "mynah_cache.h"

#include "args.h"

#include <string.h>

/* Entries of a thread where one workgroup forks (= PG_FORK in pages.hip). */
#define PAGES_FORK 8u

static int pool_check(const mynah_page_pool *p) {
    if (p == NULL || p->parts == NULL || p->refs == NULL || p->pages == NULL ||
        p->n_past == NULL || p->status == NULL)
        return refuse("null argument");
    if (p->n_pages == 0 || p->n_pages >= 1u << 28 || p->n_seqs == 0 || p->n_seqs > 65536 ||
        p->max_pages == 0 || (uint64_t)p->n_seqs * p->max_pages >= 1u << 28)
        return refuse("pages: bad counts (pages, sequences or entries)");
    if (p->n_parts == 0 || p->n_parts > 65534) return refuse("pages: 1 to 65534 parts are taken");
    if (!is_power(p->page_size)) return refuse("pages: page_size must be a power of two");
    if (((uintptr_t)p->parts & 7u) != 0 || (((uintptr_t)p->refs | (uintptr_t)p->pages |
         (uintptr_t)p->n_past | (uintptr_t)p->status) & 3u) != 0)
        return refuse("pages: misaligned operand");
    return 0;
}

/* The workspace in 32-bit words: rows for the table, then six arrays of a word for
 * each page, then the number of moves. */
static size_t pool_rows(const mynah_page_pool *p) {
    return (size_t)p->n_seqs * (p->max_pages + 1u);
}

size_t mynah_hip_pages_workspace(const mynah_page_pool *p) {
    if (pool_check(p) != 0) return 0;
    return (pool_rows(p) + 6 * (size_t)p->n_pages + 1) * 4;
}

static void pool_args(const mynah_page_pool *p, const int32_t *ask, void *workspace,
                      mynah_page_args *a) {
    memset(a, 0, sizeof *a);
    a->n_pages = p->n_pages;
    a->n_seqs = p->n_seqs;
    a->max_pages = p->max_pages;
    a->page_log2 = log2_of(p->page_size);
    a->n_parts = p->n_parts;
    a->parts = p->parts;
    a->refs = p->refs;
    a->pages = p->pages;
    a->n_past = p->n_past;
    a->status = p->status;
    a->ask = ask;
    if (workspace == NULL) return;
    a->rows = workspace;
    a->cnt = a->rows + pool_rows(p);
    a->first = a->cnt + p->n_pages;
    a->list = a->first + p->n_pages;
    a->from = a->list + p->n_pages;
    a->to = a->from + p->n_pages;
    a->map = (int32_t *)a->to + p->n_pages;
    a->moves = a->map + p->n_pages;
}

static int ws_check(const mynah_page_pool *p, const void *workspace, size_t bytes) {
    if (workspace == NULL || ((uintptr_t)workspace & 255u) != 0)
        return refuse("pages: a workspace aligned to 256 bytes is needed");
    const size_t need = mynah_hip_pages_workspace(p);
    if (bytes < need) {
        mynah_set_error("pages: a workspace of %zu bytes, %zu are needed", bytes, need);
        return -1;
    }
    return 0;
}

static int ask_check(const int32_t *ask) {
    if (ask == NULL) return refuse("null argument");
    if (((uintptr_t)ask & 3u) != 0) return refuse("pages: misaligned operand");
    return 0;
}

/* The content of the listed pages, workgroups enough to fill the card from the
 * larger parts alone. */
static int pool_move(mynah_device *d, mynah_page_args *a, hipStream_t st) {
    unsigned each = 8192u / a->n_parts;
    each = each < 16u ? 16u : each > 1024u ? 1024u : each;
    void *args[] = {a};
    return mynah_launch(d, MYNAH_K_PAGES_MOVE, each, a->n_parts + 1, 256, 0, st, args);
}

int mynah_hip_pages_fork_dev(const mynah_page_pool *p, const int32_t *from, void *workspace,
                             size_t workspace_bytes, void *stream) {
    if (pool_check(p) != 0 || ask_check(from) != 0 || ws_check(p, workspace, workspace_bytes) != 0)
        return -1;
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    mynah_page_args a;
    pool_args(p, from, workspace, &a);
    hipStream_t st = mynah_stream_or_default(d, stream);
    void *args[] = {&a};
    if (p->n_seqs <= 1024 && (uint64_t)p->n_seqs * p->max_pages <= 1024u * PAGES_FORK)
        return mynah_launch(d, MYNAH_K_PAGES_FORK, 1, 1, 1024, 0, st, args);
    if (mynah_launch(d, MYNAH_K_PAGES_FORK_TAKE, p->n_seqs, 1, 256, 0, st, args) != 0) return -1;
    return mynah_launch(d, MYNAH_K_PAGES_FORK_GIVE, p->n_seqs, 1, 256, 0, st, args);
}

int mynah_hip_pages_reserve_dev(const mynah_page_pool *p, const int32_t *n_new, void *workspace,
                                size_t workspace_bytes, void *stream) {
    if (pool_check(p) != 0 || ask_check(n_new) != 0 ||
        ws_check(p, workspace, workspace_bytes) != 0)
        return -1;
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    mynah_page_args a;
    pool_args(p, n_new, workspace, &a);
    hipStream_t st = mynah_stream_or_default(d, stream);
    void *args[] = {&a};
    if (mynah_launch(d, MYNAH_K_PAGES_RESERVE, 1, 1, 1024, 0, st, args) != 0) return -1;
    a.map = NULL;
    return pool_move(d, &a, st);
}

int mynah_hip_pages_release_dev(const mynah_page_pool *p, const int32_t *keep, void *stream) {
    if (pool_check(p) != 0 || ask_check(keep) != 0) return -1;
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    mynah_page_args a;
    pool_args(p, keep, NULL, &a);
    void *args[] = {&a};
    return mynah_launch(d, MYNAH_K_PAGES_RELEASE, p->n_seqs, 1, 256, 0,
                        mynah_stream_or_default(d, stream), args);
}

int mynah_hip_pages_compact_dev(const mynah_page_pool *p, void *workspace,
                                size_t workspace_bytes, void *stream) {
    if (pool_check(p) != 0 || ws_check(p, workspace, workspace_bytes) != 0) return -1;
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    mynah_page_args a;
    pool_args(p, NULL, workspace, &a);
    hipStream_t st = mynah_stream_or_default(d, stream);
    void *args[] = {&a};
    if (mynah_launch(d, MYNAH_K_PAGES_COMPACT, 1, 1, 1024, 0, st, args) != 0) return -1;
    return pool_move(d, &a, st);
}

int mynah_hip_pages_copy_dev(const mynah_page_pool *p, const int32_t *from, const int32_t *to,
                             uint32_t n, void *stream) {
    if (pool_check(p) != 0 || ask_check(from) != 0 || ask_check(to) != 0) return -1;
    if (n == 0) return refuse("pages: no pages to copy");
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    mynah_page_args a;
    pool_args(p, NULL, NULL, &a);
    a.from = from;
    a.to = to;
    a.count = n;
    return pool_move(d, &a, mynah_stream_or_default(d, stream));
}
