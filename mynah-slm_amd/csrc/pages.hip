// pages.hip — the pages of a cache (include/mynah_cache.h): which sequence holds
// which, and moving their content.
//
// The tables are small (a few thousand entries), so what needs an order over all of
// them is one workgroup's work, with prefix sums over the order of sequences and
// positions: equal calls give equal tables. Content moves in a second launch of many
// workgroups, from a list that the first one leaves in the workspace.
//
// SPDX-License-Identifier: MIT
#pragma once
#include "common.hip.h"

struct PagePart {
    uint8_t *base;
    size_t stride, bytes;
};

struct PageArgs {
    uint32_t n_pages, n_seqs, max_pages, page_log2, n_parts, count;
    const PagePart *parts;
    int32_t *refs, *pages, *n_past, *status;
    const int32_t *ask, *from, *to; // a call's [n_seqs] argument; the pairs to move
    int32_t *rows;                  // workspace: [n_seqs][max_pages + 1]
    int32_t *cnt, *first, *list;    // ... [n_pages] each
    int32_t *moves;                 // ... number of pairs
    int32_t *map;                   // ... [n_pages]
};

MYNAH_DEV bool is_page(const PageArgs &a, int32_t p) { return (uint32_t)p < a.n_pages; }

// ── continuing other sequences ──────────────────────────────────────────────
// A workgroup a sequence: what it will be goes to the workspace, the counts are
// brought up to date; then, when all have read, to the table. Grid n_seqs, block 256.
extern "C" __global__ void __launch_bounds__(256) mynah_pages_fork_take(PageArgs a) {
    const uint32_t b = blockIdx.x;
    const int32_t f = a.ask[b];
    if ((uint32_t)f == b) return;
    const bool some = (uint32_t)f < a.n_seqs;
    const int32_t *old = a.pages + (size_t)b * a.max_pages;
    const int32_t *src = a.pages + (size_t)(some ? f : 0) * a.max_pages;
    int32_t *row = a.rows + (size_t)b * (a.max_pages + 1u);
    for (uint32_t j = threadIdx.x; j < a.max_pages; j += 256u) {
        const int32_t was = old[j], p = some ? src[j] : -1;
        row[j] = p;
        if (was == p) continue;
        if (is_page(a, was)) atomicSub(a.refs + was, 1);
        if (is_page(a, p)) atomicAdd(a.refs + p, 1);
    }
    if (threadIdx.x == 0u) row[a.max_pages] = some ? a.n_past[f] : 0;
}

extern "C" __global__ void __launch_bounds__(256) mynah_pages_fork_give(PageArgs a) {
    const uint32_t b = blockIdx.x;
    if ((uint32_t)a.ask[b] == b) return;
    const int32_t *row = a.rows + (size_t)b * (a.max_pages + 1u);
    for (uint32_t j = threadIdx.x; j < a.max_pages; j += 256u)
        a.pages[(size_t)b * a.max_pages + j] = row[j];
    if (threadIdx.x == 0u) a.n_past[b] = row[a.max_pages];
}

// A small table's in one launch of one workgroup: entries stay in registers between
// the reads and the writes. Grid 1, block 1024; n_seqs <= 1024, n_seqs * max_pages <=
// 1024 PG_FORK (8 sequences of 13 entries 4 us a call where two launches took 7, 128 of
// 50 5 where they took 5.4).
#define PG_FORK 8u                  // (= PAGES_FORK in pages.c)
extern "C" __global__ void __launch_bounds__(1024) mynah_pages_fork(PageArgs a) {
    const uint32_t tid = threadIdx.x, n = a.n_seqs * a.max_pages;
    int32_t p[PG_FORK], was[PG_FORK];
    bool mine[PG_FORK];
#pragma unroll
    for (uint32_t k = 0; k < PG_FORK; k++) {
        const uint32_t i = tid + 1024u * k, b = i / a.max_pages;
        const int32_t f = i < n ? a.ask[b] : 0;
        mine[k] = i < n && (uint32_t)f != b;
        p[k] = was[k] = -1;
        if (mine[k]) {
            was[k] = a.pages[i];
            if ((uint32_t)f < a.n_seqs) p[k] = a.pages[(size_t)f * a.max_pages + (i - b * a.max_pages)];
        }
    }
    int32_t past = 0;
    const int32_t f = tid < a.n_seqs ? a.ask[tid] : (int32_t)tid;
    if ((uint32_t)f != tid && (uint32_t)f < a.n_seqs) past = a.n_past[f];
#pragma unroll
    for (uint32_t k = 0; k < PG_FORK; k++) {
        if (!mine[k] || was[k] == p[k]) continue;
        if (is_page(a, was[k])) atomicSub(a.refs + was[k], 1);
        if (is_page(a, p[k])) atomicAdd(a.refs + p[k], 1);
    }
    __syncthreads();                               // all have read
#pragma unroll
    for (uint32_t k = 0; k < PG_FORK; k++)
        if (mine[k]) a.pages[tid + 1024u * k] = p[k];
    if ((uint32_t)f != tid && tid < a.n_seqs) a.n_past[tid] = past;
}

// ── cutting sequences ───────────────────────────────────────────────────────
// Grid n_seqs, block 256.
extern "C" __global__ void __launch_bounds__(256) mynah_pages_release(PageArgs a) {
    const uint32_t b = blockIdx.x;
    const int32_t keep = a.ask[b];
    if (keep < 0) return;
    const uint32_t held = (uint32_t)(((uint64_t)keep + (1u << a.page_log2) - 1u) >> a.page_log2);
    int32_t *row = a.pages + (size_t)b * a.max_pages;
    for (uint32_t j = held + threadIdx.x; j < a.max_pages; j += 256u) {
        const int32_t p = row[j];
        if (is_page(a, p)) atomicSub(a.refs + p, 1);
        row[j] = -1;
    }
    if (threadIdx.x == 0u && a.n_past[b] > keep) a.n_past[b] = keep;
}

// ── one workgroup's sums ────────────────────────────────────────────────────
#define PG_T 1024u

// The workgroup meets, its stores and atomics done in the L2: what other waves left
// there is read past the vector cache.
MYNAH_DEV void page_sync() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}
MYNAH_DEV int32_t fresh_i32(const int32_t *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sum of n over the threads before this one; `all` the sum over all. Every thread of
// the workgroup takes part.
MYNAH_DEV uint32_t before_me(uint32_t n, uint32_t &all) {
    __shared__ uint32_t sums[PG_T / 64u];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t upto = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t x = __shfl_up(upto, d, 64);
        upto += lane >= (uint32_t)d ? x : 0u;
    }
    __syncthreads();                               // the sums of the call before
    if (lane == 63u) sums[wave] = upto;
    __syncthreads();
    uint32_t before = 0u;
    all = 0u;
#pragma unroll
    for (uint32_t w = 0; w < PG_T / 64u; w++) {
        before += w < wave ? sums[w] : 0u;
        all += sums[w];
    }
    return before + upto - n;
}

// ── pages of their own for new positions ────────────────────────────────────
struct PageSpan {
    uint32_t from, to;              // entries of the new positions
    uint64_t past;
    bool fits;
};
MYNAH_DEV PageSpan page_span(const PageArgs &a, uint32_t b) {
    PageSpan s;
    const int32_t past = a.n_past[b], n = a.ask[b];
    s.past = past > 0 ? (uint64_t)past : 0u;
    const uint64_t to = (s.past + (uint64_t)(n > 0 ? n : 0) + (1u << a.page_log2) - 1u) >> a.page_log2;
    s.from = (uint32_t)(s.past >> a.page_log2);
    s.fits = n <= 0 || to <= a.max_pages;
    s.to = n <= 0 ? s.from : to <= a.max_pages ? (uint32_t)to : a.max_pages;
    return s;
}

// The place of page p in a table of 2 PG_T places in the LDS (-1: free) that PG_T
// pages at most are put into.
MYNAH_DEV uint32_t page_place(int32_t *keys, int32_t p) {
    uint32_t h = (uint32_t)p * 2654435761u >> 21;  // 11 bits
    for (;; h = (h + 1u) & (2u * PG_T - 1u)) {
        const int32_t was = atomicCAS(keys + h, -1, p);
        if (was == -1 || was == p) return h;
    }
}

// Grid 1, block PG_T. Entries are taken sequence by sequence, K apiece, the longest
// span: i is entry i % K of sequence i / K, so that one long request among many short ones
// costs as many rounds as if all were as long. Bound by reads that need each other: up to
// PG_T entries each thread has its own, and counts and lists are in the LDS (of ten reads and
// writes one after the other, in memory, 11 us; now 6.6 of the 16 us in which 8 sequences
// are forked and get a page each, three launches).
extern "C" __global__ void __launch_bounds__(PG_T) mynah_pages_reserve(PageArgs a) {
    __shared__ uint32_t longest, too_long, copies;
    __shared__ int32_t keys[2u * PG_T], counts[2u * PG_T], firsts[2u * PG_T], given_to[PG_T];
    const uint32_t tid = threadIdx.x;
    uint32_t first_free = 0u;                      // of pages 4 tid ..
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++)
        first_free |= 4u * tid + k < a.n_pages && a.refs[4u * tid + k] <= 0 ? 1u << k : 0u;
    if (tid == 0u) longest = too_long = copies = 0u;
    for (uint32_t k = tid; k < 2u * PG_T; k += PG_T) {
        keys[k] = -1;
        counts[k] = 0;
        firsts[k] = 0x7fffffff;
    }
    __syncthreads();
    for (uint32_t b = tid; b < a.n_seqs; b += PG_T) {
        const PageSpan s = page_span(a, b);
        if (!s.fits) atomicAdd(&too_long, 1u);
        if (s.to > s.from) atomicMax(&longest, s.to - s.from);
    }
    __syncthreads();
    const uint32_t K = longest;
    const uint64_t n = (uint64_t)K * a.n_seqs;
    // The entry of i, or false.
    auto entry = [&](uint64_t i, uint32_t &b, PageSpan &s, int32_t *&at) {
        if (i >= n) return false;
        b = (uint32_t)(i / K);
        s = page_span(a, b);
        const uint32_t j = s.from + (uint32_t)(i - (uint64_t)b * K);
        at = a.pages + (size_t)b * a.max_pages + j;
        return j < s.to;
    };
    // Free pages p .. p + 3 of `free`, `at` of them before: to the list as far as wanted.
    auto list = [&](uint32_t p, uint32_t free, uint32_t at, uint32_t wanted, int32_t *to) {
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++)
            if (free >> k & 1u) {
                if (at < wanted) to[at] = (int32_t)(p + k);
                at++;
            }
    };
    auto free_of = [&](uint32_t p) {
        uint32_t free = 0u;
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++)
            free |= p + k < a.n_pages && a.refs[p + k] <= 0 ? 1u << k : 0u;
        return free;
    };
    // An entry's page is given: 2 in place of a shared one, 3 with its content.
    auto give = [&](int32_t get, int32_t *at, int32_t old, int32_t p) {
        *at = p;
        a.refs[p] = 1;
        if (get > 1) atomicSub(a.refs + old, 1);
        if (get == 3) {
            const uint32_t c = atomicAdd(&copies, 1u);
            ((int32_t *)a.from)[c] = old;
            ((int32_t *)a.to)[c] = p;
        }
    };
    auto with_content = [&](const PageSpan &s, uint32_t b, const int32_t *at) {
        return (uint64_t)(at - (a.pages + (size_t)b * a.max_pages)) << a.page_log2 < s.past ? 3 : 2;
    };
    auto tell = [&](uint32_t wanted, uint32_t found) {
        if (tid == 0u) {
            a.status[0] = found < wanted ? (int32_t)(wanted - found) : 0;
            a.status[1] = (int32_t)too_long;
        }
        return found >= wanted && too_long == 0u;
    };
    if (n <= PG_T) {
        uint32_t b = 0u;
        PageSpan s;
        int32_t *at = nullptr, p = -1, r = 0, get = 0;
        uint32_t h = 0u;
        const bool in = entry(tid, b, s, at);
        if (in) p = *at;
        const bool held = in && is_page(a, p);
        if (held) r = a.refs[p];
        if (held && r > 1) {
            h = page_place(keys, p);
            atomicAdd(counts + h, 1);
            atomicMin(firsts + h, (int32_t)b);
        }
        __syncthreads();
        if (in && !held) get = 1;
        else if (held && r > 1 && !(counts[h] == r && firsts[h] == (int32_t)b))
            get = with_content(s, b, at);
        uint32_t wanted, all;
        const uint32_t k = before_me(get ? 1u : 0u, wanted);
        uint32_t found = 0u;
        for (uint32_t p0 = 0; p0 < a.n_pages && found < wanted; p0 += 4u * PG_T) {
            const uint32_t free = p0 ? free_of(p0 + 4u * tid) : first_free;
            list(p0 + 4u * tid, free, found + before_me(__popc(free), all), wanted, given_to);
            found += all;
        }
        __syncthreads();
        if (tell(wanted, found) && get) give(get, at, p, given_to[k]);
        __syncthreads();
        if (tid == 0u) *a.moves = (int32_t)copies;
        return;
    }
    // How many ask for a page that is there, and who first.
    for (int step = 0; step < 2; step++) {
        for (uint64_t i = tid; i < n; i += PG_T) {
            uint32_t b;
            PageSpan s;
            int32_t *at;
            if (!entry(i, b, s, at) || !is_page(a, *at)) continue;
            if (step == 0) {
                __hip_atomic_store(a.cnt + *at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(a.first + *at, 0x7fffffff, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
            } else {
                atomicAdd(a.cnt + *at, 1);
                atomicMin(a.first + *at, (int32_t)b);
            }
        }
        page_sync();
    }
    // Who gets a page: 1 where there is none, 2 in place of a shared one, 3 with its content.
    uint32_t wanted = 0u;
    for (uint64_t i0 = 0; i0 < n; i0 += PG_T) {
        uint32_t b;
        PageSpan s;
        int32_t *at, get = 0;
        if (entry(i0 + tid, b, s, at)) {
            const int32_t p = *at;
            if (!is_page(a, p)) {
                get = 1;
            } else {
                const int32_t r = a.refs[p];
                if (r > 1 && !(fresh_i32(a.cnt + p) == r && fresh_i32(a.first + p) == (int32_t)b))
                    get = with_content(s, b, at);
            }
            a.rows[i0 + tid] = get;
        }
        uint32_t all;
        before_me(get ? 1u : 0u, all);
        wanted += all;
    }
    // The lowest free pages, as many as are wanted.
    uint32_t found = 0u;
    for (uint32_t p0 = 0; p0 < a.n_pages && found < wanted; p0 += 4u * PG_T) {
        const uint32_t free = p0 ? free_of(p0 + 4u * tid) : first_free;
        uint32_t all;
        const uint32_t at = found + before_me(__popc(free), all);
        list(p0 + 4u * tid, free, at, wanted, a.list);
        found += all;
    }
    page_sync();
    const bool fits = tell(wanted, found);
    uint32_t given = 0u;
    for (uint64_t i0 = 0; fits && i0 < n; i0 += PG_T) {
        uint32_t b;
        PageSpan s;
        int32_t *at;
        const int32_t get = entry(i0 + tid, b, s, at) ? fresh_i32(a.rows + i0 + tid) : 0;
        uint32_t all;
        const uint32_t k = given + before_me(get ? 1u : 0u, all);
        given += all;
        if (get) give(get, at, *at, fresh_i32(a.list + k));
    }
    __syncthreads();
    if (tid == 0u) *a.moves = (int32_t)copies;
}

// ── the pages in use to the lowest places ───────────────────────────────────
// Grid 1, block PG_T: the n-th free page below the number of pages in use gets the n-th
// page in use from there on, so that no page is read and written, and the moves need no
// order.
extern "C" __global__ void __launch_bounds__(PG_T) mynah_pages_compact(PageArgs a) {
    const uint32_t tid = threadIdx.x;
    uint32_t mine = 0u, live;
    for (uint32_t p = tid; p < a.n_pages; p += PG_T) mine += a.refs[p] > 0 ? 1u : 0u;
    before_me(mine, live);
    uint32_t n_to = 0u, n_from = 0u;
    for (uint32_t p0 = 0; p0 < a.n_pages; p0 += PG_T) {
        const uint32_t p = p0 + tid;
        const bool used = p < a.n_pages && a.refs[p] > 0;
        const bool to = p < live && !used, from = p >= live && used;
        uint32_t all, at = before_me(to ? 1u : 0u, all);
        if (to) ((int32_t *)a.to)[n_to + at] = (int32_t)p;
        n_to += all;
        at = before_me(from ? 1u : 0u, all);
        if (from) ((int32_t *)a.from)[n_from + at] = (int32_t)p;
        n_from += all;
        // An entry that names a page without a count stays.
        if (p < a.n_pages && p >= live) a.map[p] = (int32_t)p;
    }
    page_sync();
    for (uint32_t k = tid; k < n_from; k += PG_T) {
        const int32_t f = fresh_i32(a.from + k), t = fresh_i32(a.to + k);
        a.map[f] = t;
        a.refs[t] = a.refs[f];
        a.refs[f] = 0;
    }
    if (tid == 0u) {
        *a.moves = (int32_t)n_from;
        a.status[0] = (int32_t)live;
        a.status[1] = (int32_t)n_from;
    }
}

// ── content ─────────────────────────────────────────────────────────────────
// What bounds it: memory (150 pages of 6 layers, 118 MB read and as many written, 53 us,
// 4.4 TB/s where a copy of a GiB reaches 5.0; chunks of 8 KiB 54, of 32 KiB 80).
// Grid (workgroups a part, n_parts + 1), block 256: of the pairs in a.from and a.to
// (a.moves of them, or a.count without), chunks of 16 KiB of one part. The last row of
// workgroups brings the table up to date where a.map is given (compaction): entries
// from the number of pages in use (status[0]) on have moved.
template <class V>
MYNAH_DEV void copy_run(const uint8_t *from, uint8_t *to, uint32_t n) {
    const V *x = (const V *)from;
    V *y = (V *)to;
    for (uint32_t i = threadIdx.x; i < n; i += 4u * 256u) {
        V v[4];
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++)
            if (i + 256u * k < n) v[k] = x[i + 256u * k];
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++)
            if (i + 256u * k < n) y[i + 256u * k] = v[k];
    }
}

#define PG_CHUNK 16384u
extern "C" __global__ void __launch_bounds__(256) mynah_pages_move(PageArgs a) {
    if (blockIdx.y == a.n_parts) {
        if (!a.map) return;
        const size_t n = (size_t)a.n_seqs * a.max_pages;
        const uint32_t live = (uint32_t)a.status[0];
        for (size_t i = blockIdx.x * 256u + threadIdx.x; i < n; i += 256u * gridDim.x) {
            const int32_t p = a.pages[i];
            if (is_page(a, p) && (uint32_t)p >= live) a.pages[i] = a.map[p];
        }
        return;
    }
    const PagePart part = a.parts[blockIdx.y];
    const uint32_t pairs = a.moves ? (uint32_t)*a.moves : a.count;
    const uint64_t chunks = (part.bytes + PG_CHUNK - 1u) / PG_CHUNK;
    const uint64_t bits = (uint64_t)(uintptr_t)part.base | part.stride | part.bytes;
    for (uint64_t u = blockIdx.x; u < chunks * pairs; u += gridDim.x) {
        const uint64_t k = u / chunks, at = (u - k * chunks) * PG_CHUNK;
        const int32_t f = a.from[k], t = a.to[k];
        if (!is_page(a, f) || !is_page(a, t)) continue;
        const uint8_t *x = part.base + (size_t)f * part.stride + at;
        uint8_t *y = part.base + (size_t)t * part.stride + at;
        const uint32_t n = part.bytes - at < PG_CHUNK ? (uint32_t)(part.bytes - at) : PG_CHUNK;
        if ((bits & 15u) == 0u) copy_run<uint4>(x, y, n / 16u);
        else if ((bits & 3u) == 0u) copy_run<uint32_t>(x, y, n / 4u);
        else copy_run<uint8_t>(x, y, n);
    }
}
