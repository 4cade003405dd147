// tree_attn.hip — attention of drafted tokens over a key/value cache
// (include/mynah_attention.h, mynah_hip_tree_attention_dev).
//
// A key head's queries (its group of heads, of every node: row = node * group +
// head) are columns of 16 of the matrix instruction, keys its rows: S^T = K
// Q^T, so that a lane holds four keys' scores of one query, which is what the
// second product O^T = V^T P^T takes as its operand: the probabilities never
// leave their registers. Which key and which dimension an operand's place
// stands for is free as long as both operands agree, so K and V leave the LDS in
// whole runs of 8 or 16 bytes a lane; 16-bit V is turned by one v_perm per two
// values. The copies from memory go straight to the LDS (keys read from memory as
// operands, 16 rows an instruction, came at 22-31 bytes a clock and CU, the rate of
// the address unit) and stay under way while the chunk before is computed. Each
// wave keeps a running maximum and sum for its own keys; the waves meet once at the
// end, workgroups in a second launch.
//
// Bound by memory where a key head has few rows, by the matrix and exponential
// units where it has many. Measured, MI355X: 16 sequences of up to 16 nodes and
// 8207 bf16 positions in pages (32 heads, 8 of keys, 128 wide; 85,413 positions in all,
// 350 MB) 96 us, 3.6 TB/s; the same with one node each 80 us, 4.4 TB/s (75 without the
// second launch); 64 nodes over 130,065 f16 positions (533 MB, 136 GFLOP) 203-213 us; one
// sequence of 16 nodes over 65,552 69 us, 3.9 TB/s, of one node 62 us, 4.3 TB/s (56
// without); 24 f32 nodes over 2072 positions 21 us; one f32 token over 513 13 us.
//
// SPDX-License-Identifier: MIT
#pragma once
#include "common.hip.h"
#include "elem.hip.h"

struct TreeArgs {
    const void *q, *k, *v;
    void *out;
    size_t q_stride, out_stride, slot_stride, seq_slots;
    const int32_t *pages, *seq_start, *n_past;
    const uint32_t *mask;
    float *pm, *pl, *po;            // partials [workgroup][wg_rows], (x head_dim)
    int32_t *plan;                  // a sequence's first slot and their number
    unsigned long long n_slots;
    uint32_t n_seqs, n_heads, n_kv, group, n_rows, page_log2, max_pages, mask_words;
    uint32_t max_nodes, max_kv, slots, groups, wg_rows;
    float scale2;                   // |scale| log2(e), above 0 and finite
    float lag;                      // growth of a score without a new reference
    uint32_t flip;                  // sign bits of a query's dwords, where scale is below 0
};

typedef float ta_v4f __attribute__((ext_vector_type(4)));
typedef _Float16 ta_v8h __attribute__((ext_vector_type(8)));
typedef __bf16 ta_v8b __attribute__((ext_vector_type(8)));

// A word that no kernel writes while this one runs, by a scalar load (of a plain
// pointer the compiler takes a vector load, and its wait drains the prefetches).
typedef __attribute__((address_space(4))) const int32_t ta_const_i32;
MYNAH_DEV int32_t scalar_i32(const int32_t *p, size_t i) {
    return ((ta_const_i32 *)(uintptr_t)p)[i];
}

struct SeqSpan {
    long long row0;                 // first query row
    uint32_t nodes, past, kv;
};

// A sequence's rows and positions as the call bounds them.
MYNAH_DEV SeqSpan seq_span(const TreeArgs &a, uint32_t b) {
    SeqSpan s;
    s.row0 = scalar_i32(a.seq_start, b);
    const long long n = (long long)scalar_i32(a.seq_start, b + 1u) - s.row0;
    const int past = scalar_i32(a.n_past, b);
    s.nodes = n <= 0 ? 0u : n < (long long)a.max_nodes ? (uint32_t)n : a.max_nodes;
    s.past = past > 0 ? (uint32_t)past : 0u;
    const unsigned long long kv = (unsigned long long)s.past + s.nodes;
    s.kv = kv < a.max_kv ? (uint32_t)kv : a.max_kv;
    return s;
}

// A slot (a workgroup of each key head and group of rows): positions split * per ..
// of sequence b, `per` at most.
struct SlotShare {
    uint32_t b, split, per;
};

// Several sequences share the slots by their lengths: of 64 sizes of a piece, in
// turns of the key groups, the smallest that cuts all sequences into no more pieces
// than there are slots. A lane holds every 64th sequence's turns, and then tries one
// size; ceil(n * (1 / size)) in floats is the exact number or, where size divides n, at most
// one more (n < 2^22), and every workgroup finds the same. Sizes run up to
// total / (slots - n_seqs) + 1, for sum ceil(n / p) <= total / p + n_seqs. False for
// a slot that is left over. Against as many pieces for every sequence, bf16, 32 heads, 8
// of keys, 8 nodes: one sequence of 32,768 positions beside 15 of 512 51 us for 209, 4 of
// 16,000 beside 12 of 1000 76 for 138, 16 of 4000 54 for 52. Exactly equal shares,
// with slots that end one sequence and begin the next, cost more than they gave: the
// 16 sequences below 110 us for 96.
#define TA_MOST_TURNS (1u << 21)    // 2^26 positions in the smallest turn, 32
MYNAH_DEV bool share_slots(const TreeArgs &a, uint32_t slot, uint32_t turn, bool tell,
                           SlotShare &out) {
    const uint32_t lane = threadIdx.x & 63u;
    float n[4];
    uint32_t total = 0u;            // at most 255 * 2^21
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t b = 64u * c + lane;
        uint32_t turns = 0u;
        if (b < a.n_seqs) {
            const long long rows = (long long)a.seq_start[b + 1u] - a.seq_start[b];
            const uint32_t nodes = rows <= 0 ? 0u
                                 : rows < (long long)a.max_nodes ? (uint32_t)rows : a.max_nodes;
            const int past = a.n_past[b];
            const unsigned long long kv = (unsigned long long)(past > 0 ? past : 0) + nodes;
            const uint32_t k = kv < a.max_kv ? (uint32_t)kv : a.max_kv;
            turns = nodes ? (k + turn - 1u) / turn : 0u;
        }
        n[c] = (float)turns;
        total += turns;
    }
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) total += __shfl_xor(total, d, 64);
    uint32_t least = (total + a.slots - 1u) / a.slots;
    least = least ? least : 1u;
    const uint32_t most = total / (a.slots - a.n_seqs) + 1u;
    uint32_t size = least + (most - least + 61u) / 62u * lane;
    // A whole sequence a piece is few enough in any case.
    size = size < TA_MOST_TURNS && lane != 63u ? size : TA_MOST_TURNS;
    float inv = 1.0f / (float)size, pieces = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t left = a.n_seqs > 64u * c ? a.n_seqs - 64u * c : 0u;
        for (uint32_t j = 0; j < (left < 64u ? left : 64u); j++)
            pieces += ceilf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(n[c]), j)) * inv);
    }
    const uint32_t pick =
        (uint32_t)__builtin_ctzll(__ballot(pieces <= (float)a.slots || lane == 63u));
    inv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(inv), pick));
    out.per = turn * __builtin_amdgcn_readlane(size, pick);
    uint32_t before = 0u;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t count = (uint32_t)ceilf(n[c] * inv);
        uint32_t upto = count;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t x = __shfl_up(upto, d, 64);
            upto += lane >= (uint32_t)d ? x : 0u;
        }
        // Sequences that end at or before this slot.
        const uint32_t at =
            (uint32_t)__builtin_popcountll(__ballot(before + upto <= slot));
        if (at < 64u) {
            const uint32_t mine = __builtin_amdgcn_readlane(count, at);
            const uint32_t first = before + __builtin_amdgcn_readlane(upto, at) - mine;
            out.b = 64u * c + at;
            out.split = slot - first;
            if (tell && out.split == 0u && threadIdx.x == 0u) {
                a.plan[2u * out.b] = (int32_t)first;
                a.plan[2u * out.b + 1u] = (int32_t)mine;
            }
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

MYNAH_DEV float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// What an element type and head size make of the operands.
template <class T, int HD>
struct TaShape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr float UP = __is_same(T, _Float16) ? 11.0f : 0.0f; // see a.lag below
    static constexpr int TILES = F32 ? 1 : 2;         // 16-key tiles of a chunk
    static constexpr int CK = 16 * TILES;             // keys of a chunk
    static constexpr int KP = F32 ? HD / 16 : HD / 32; // 16-byte pieces of a lane's key
    static constexpr int VE = HD / 16;                // dimensions (O tiles) of a lane
    static constexpr int CW = F32 || HD == 64 ? 4 : 8; // of them side by side
    static constexpr int VP = VE / CW;                // pieces of a lane's value row
    static constexpr int VD = CW * (int)sizeof(T) / 4; // dwords of a piece
    static constexpr int KB = CK * HD * (int)sizeof(T); // bytes of a chunk's keys
    static constexpr int CPR = HD * (int)sizeof(T) / 16; // 16-byte pieces of a key
    static constexpr int RPI = 64 / CPR;              // keys that one copy takes
    // Waves of a workgroup (= tree_plan.waves in attention.c): their chunks of keys
    // and values, in flight or in use, fill the LDS.
    static constexpr int W = HD == 256 ? 4 : 8;
};

typedef __attribute__((address_space(3))) void ta_lds_void;

template <class T>
MYNAH_DEV ta_v4f ta_mfma(const uint32_t (&a)[4], const uint32_t (&b)[4], ta_v4f c) {
    if constexpr (__is_same(T, _Float16)) {
        ta_v8h x, y;
        __builtin_memcpy(&x, a, 16);
        __builtin_memcpy(&y, b, 16);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
    } else {
        ta_v8b x, y;
        __builtin_memcpy(&x, a, 16);
        __builtin_memcpy(&y, b, 16);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
    }
}

MYNAH_DEV float lane_max4(float v) {      // over the four lanes of one column
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
MYNAH_DEV float lane_sum4(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

template <int VD>
MYNAH_DEV void load_dwords(const char *p, uint32_t *d) {
    if constexpr (VD == 2) {
        const uint2 x = *(const uint2 *)p;
        d[0] = x.x; d[1] = x.y;
    } else {
        const uint4 x = *(const uint4 *)p;
        d[0] = x.x; d[1] = x.y; d[2] = x.z; d[3] = x.w;
    }
}

// A register of one f32 or two 16-bit values with zeros in the place of
// infinities and NaN.
template <class T>
MYNAH_DEV uint32_t finite_part(uint32_t d) {
    if constexpr (sizeof(T) == 4) return (d & 0x7f800000u) == 0x7f800000u ? 0u : d;
    constexpr uint32_t e = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    return ((d & e) == e ? 0u : d & 0xffffu) | (((d >> 16) & e) == e ? 0u : d & 0xffff0000u);
}

// Whether a query (node `node` of its sequence, its words of the mask from
// `words` on) sees node j, as 0 or 1.
MYNAH_DEV uint32_t sees_node(const TreeArgs &a, size_t words, uint32_t node, uint32_t j) {
    // Without a branch: a word that is there is read in any case.
    const bool chain = a.mask == nullptr;
    const uint32_t *p = chain ? (const uint32_t *)a.n_past : a.mask + words + j / 32u;
    const uint32_t bit = (*p >> (j & 31u)) & 1u;
    return chain ? (uint32_t)(j <= node) : bit;
}

// The cache row of position p of sequence b; false where it is not in the cache.
MYNAH_DEV bool cache_row(const TreeArgs &a, uint32_t b, uint32_t p, unsigned long long &row) {
    unsigned long long r = (unsigned long long)b * a.seq_slots + p;
    if (a.pages) {
        const int pg = scalar_i32(a.pages, (size_t)b * a.max_pages + (p >> a.page_log2));
        if (pg < 0) return false;
        r = ((unsigned long long)(uint32_t)pg << a.page_log2) + (p & ((1u << a.page_log2) - 1u));
    }
    row = r;
    return r < a.n_slots;
}

// A column's reference for the exponentials is left behind by scores that grow up to
// a.lag (2^8 in the probabilities, of f16 2^4): sums and 16-bit probabilities hold that
// many times their size, and most chunks then rescale nothing and compare only within
// their lanes. f16 probabilities are 2^11 times theirs, for below 2^-14 the type keeps
// fewer bits and below 2^-25 nothing: with the largest at 2^11 or above, n of them are off
// by n 2^-36 of it at most, a half step of the result at 2^25 positions. (Unscaled,
// one position 17.4 nats above 130,000 others lost 0.4 % of the result.) The sums
// carry the factor too, so it leaves with the division. 64 f16 nodes over 130,065
// positions, lag and factor 2^8 and 1: 199 us; 2^8, 2^7: 201; 2^4, 2^11: 203; 2^2, 2^13: 208.
// References are scores as the products gave them, so that the difference to one is
// exact next to it and only then scaled: a scaled reference's rounding alone is
// above a power of two from scores of 2^25 on.

// A workgroup's W waves are RW row waves, each with 16 NT query rows of its own, for
// each of W / RW key groups, which take chunks of keys in turn.
//   RW == 1: a wave's chunk is its own, one buffer of keys and one of values: the
//     next keys are copied when these are used up, values likewise; no barrier.
//   RW > 1: the row waves of a key group copy its chunk together, two buffers, one
//     barrier a chunk: what comes from the L2 is read by RW waves. (Alone, each wave
//     with its own rows and keys, 256 rows over 130,001 f16 positions read 4.3 GB
//     through the L2 at 14-16 TB/s, 278 us.)
// Grid slots * n_kv * groups (of 16 NT RW query rows), block 64 W. Workgroups go to
// the 8 XCDs in turn; each XCD takes a run of the order (slot, key head, group), so
// that groups that share keys share its L2.
template <class T, int HD, int NT, int RW>
MYNAH_DEV void tree_attn(const TreeArgs &a) {
    using S = TaShape<T, HD>;
    constexpr int KW = S::W / RW;                  // key groups
    constexpr int BUF = KW * S::KB, HALF = S::W * S::KB / 2;
    // A buffer of keys and one of values, or two of each: objects of their own, so
    // that reads of one wait for its copies alone. Half of the waves' results (of the
    // dimensions) takes the first one's place at the end.
    __shared__ __attribute__((aligned(16))) uint8_t kx[BUF > HALF ? BUF : HALF], vx[BUF];
    __shared__ __attribute__((aligned(16))) uint8_t ky[RW > 1 ? BUF : 16], vy[RW > 1 ? BUF : 16];
    __shared__ float lmax[S::W][16], lsum[S::W][16];
    __shared__ uint32_t lbad[S::W], keep[8];
    // Each wave's own: its columns' nodes, and their first words of the mask.
    __shared__ uint32_t lnode[S::W][16 * NT], lwords[S::W][16 * NT];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u, lm = lane & 15u, lk = lane >> 4;
    const uint32_t rw = wave % RW, kg = wave / RW;
    uint32_t id = blockIdx.x;
    const uint32_t even = gridDim.x & ~7u;
    if (id < even) id = (id & 7u) * (even >> 3) + (id >> 3);
    const uint32_t head_id = id / a.groups, slot = head_id / a.n_kv;
    const uint32_t kvh = head_id - slot * a.n_kv, part = id - head_id * a.groups;
    const uint32_t turn = S::CK * KW;              // keys that the groups take at a time
    SlotShare share = {slot, 0u, ~0u};
    if (a.slots > a.n_seqs) {                      // uniform
        if (a.n_seqs == 1u) share = {0u, slot, 0u};
        else if (!share_slots(a, slot, turn, kvh == 0u && part == 0u, share)) return;
    }
    // The compiler does not see that these are the wave's, and walks over lanes else (64
    // f16 nodes over 130,065 positions 231 us for 209).
    const uint32_t b = __builtin_amdgcn_readfirstlane(share.b);
    const uint32_t split = __builtin_amdgcn_readfirstlane(share.split);
    const SeqSpan sq = seq_span(a, b);
    const uint32_t rows = sq.nodes * a.group;
    const uint32_t wg0 = part * (16u * NT * RW);
    if (wg0 >= rows) return;                       // uniform
    const uint32_t rr0 = wg0 + 16u * NT * rw;      // the wave's first row
    uint32_t per = __builtin_amdgcn_readfirstlane(share.per);
    if (per == 0u) {
        per = (sq.kv + a.slots - 1u) / a.slots;
        per = (per + turn - 1u) / turn * turn;
    }
    const unsigned long long from = (unsigned long long)split * per;
    const uint32_t begin = from < sq.kv ? (uint32_t)from : sq.kv;
    const uint32_t end = sq.kv - begin < per ? sq.kv : begin + per;

    // What only the end or a mask needs waits in the LDS: in registers it would
    // spill (the 16-bit 128-wide kernels of two column tiles are at their limit, and
    // keep two registers of their own in memory).
    if (threadIdx.x == 0u) {
        keep[0] = id;
        keep[1] = kvh;
        keep[2] = wg0;
        keep[3] = rows;
        keep[4] = (uint32_t)sq.row0;
        keep[5] = b;
        keep[6] = begin;
    }

    // Queries: lane's column of each tile, as operands. Columns that are no query
    // (past the rows) hold zeros, read from row 0.
    uint4 qv[NT][S::KP];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t rr = rr0 + 16u * n + lm, nd = rr / a.group;
        const long long qrow = sq.row0 + nd;
        const bool live = rr < rows && qrow >= 0 && qrow < (long long)a.n_rows;
        lnode[wave][16 * n + lm] = nd;
        lwords[wave][16 * n + lm] = live ? (uint32_t)qrow * a.mask_words : 0u;
        const char *p = (const char *)a.q + ((live ? (size_t)qrow * a.q_stride : 0) +
                                             (size_t)(kvh * a.group + rr - nd * a.group) * HD) *
                                                sizeof(T);
#pragma unroll
        for (int c = 0; c < S::KP; c++) {
            const uint4 x = *(const uint4 *)(p + 64u * c + 16u * lk);
            qv[n][c] = uint4{live ? x.x ^ a.flip : 0u, live ? x.y ^ a.flip : 0u,
                             live ? x.z ^ a.flip : 0u, live ? x.w ^ a.flip : 0u};
        }
    }
    float m[NT], l[NT];
    ta_v4f o[NT][S::VE];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int e = 0; e < S::VE; e++) o[n][e] = ta_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // Cache rows of a tile: the first, and how many of the 16 there are.
    const uint32_t sb = (uint32_t)(a.slot_stride * sizeof(T));
    const char *kbase = (const char *)a.k + (size_t)kvh * HD * sizeof(T);
    const char *vbase = (const char *)a.v + (size_t)kvh * HD * sizeof(T);
    unsigned long long row[S::TILES];
    uint32_t nv[S::TILES];
    auto find = [&](uint32_t c) {
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            const uint32_t p = c + 16u * t;
            row[t] = 0;
            nv[t] = 0;
            unsigned long long r;
            if (p >= end || !cache_row(a, b, p, r)) continue;
            row[t] = r;
            nv[t] = end - p < 16u ? end - p : 16u;
            if (a.n_slots - r < nv[t]) nv[t] = (uint32_t)(a.n_slots - r);
        }
    };
    // Copies of whole rows, 1 KiB each, from buffers that end with the tile's last
    // row: rows past it are out of range, are not read and become zeros. 16-byte
    // piece c of key k lies at place c ^ (k % 8), so that an operand's reads (one
    // piece of 16 keys) meet no bank twice; values lie in order.
    auto load = [&](const char *base, uint8_t *to, uint32_t turned) {
#pragma unroll
        for (int j = 0; j < S::KB / 1024 / RW; j++) {
            const uint32_t i = (uint32_t)(j * RW) + rw, at16 = i * S::RPI, first = at16 & 15u;
            const bool low = S::TILES == 1 || at16 < 16u;
            const uint32_t n = low ? nv[0] : nv[S::TILES - 1];
            const unsigned long long r0 = low ? row[0] : row[S::TILES - 1];
            const uint32_t at = __umul24(lane / S::CPR, sb) +
                                16u * ((lane % S::CPR) ^ ((first + lane / S::CPR) & turned));
            const uint32_t left = __builtin_amdgcn_readfirstlane((n > first ? n - first : 0u) * sb);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                __builtin_amdgcn_make_buffer_rsrc((void *)(base + (r0 + first) * sb), 0, left,
                                                  0x00020000),
                (ta_lds_void *)(to + 1024u * i), 16, at, 0, 0, 0);
        }
    };
    // Lane's values: keys 4 lk + r of each tile, dimensions 16 CW c + CW lm + ...
    uint32_t vr[S::TILES][4][S::VP][S::VD];
    auto read_v = [&](const uint8_t *lds_v) {
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int c = 0; c < S::VP; c++)
                    load_dwords<S::VD>((const char *)lds_v +
                                           (16u * t + 4u * lk + r) * (16u * S::CPR) +
                                           (16u * c + lm) * (uint32_t)(S::CW * sizeof(T)),
                                       vr[t][r][c]);
    };
    auto pv = [&](int e, const uint32_t (&p)[4], ta_v4f acc) {
        const int c = e / S::CW;
        if constexpr (S::F32) {
#pragma unroll
            for (int r = 0; r < 4; r++)
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[0][r][c][e % 4]),
                                                           __uint_as_float(p[r]), acc, 0, 0, 0);
            return acc;
        } else {
            const int d = e % S::CW / 2;
            const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
            uint32_t va[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = i / 2, r = 2 * (i & 1);
                va[i] = __builtin_amdgcn_perm(vr[t][r + 1][c][d], vr[t][r][c][d], sel);
            }
            return ta_mfma<T>(va, p, acc);
        }
    };

    // Scores of the chunk in the registers: lane's query (column lm) against keys
    // 4 lk + r of each tile.
    float s[NT][S::TILES][4];
    auto scores = [&](const uint8_t *lds_k) {
        uint4 key[S::TILES][S::KP];
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
#pragma unroll
            for (int k = 0; k < S::KP; k++)
                key[t][k] = *(const uint4 *)(lds_k + (16u * t + lm) * (16u * S::CPR) +
                                             16u * ((4u * k + lk) ^ (lm & 7u)));
#pragma unroll
        for (int n = 0; n < NT; n++) {
            uint4 q[S::KP];
#pragma unroll
            for (int k = 0; k < S::KP; k++) q[k] = qv[n][k];
#pragma unroll
            for (int t = 0; t < S::TILES; t++) {
                ta_v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < S::KP; k++) {
                    const uint32_t qk[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
                    const uint32_t kk[4] = {key[t][k].x, key[t][k].y, key[t][k].z, key[t][k].w};
                    if constexpr (S::F32) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            x = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __uint_as_float(kk[i]), __uint_as_float(qk[i]), x, 0, 0, 0);
                    } else {
                        x = ta_mfma<T>(kk, qk, x);
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++) s[n][t][r] = x[r];
            }
            // One column tile after the other: their operands together would
            // not fit the registers. And the copies that follow write where
            // these keys were read.
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Their exponentials, and the values weighted by them.
    auto weigh = [&]() {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float top = s[n][0][0];
#pragma unroll
            for (int j = 1; j < 4 * S::TILES; j++) top = fmaxf(top, s[n][j / 4][j % 4]);
            if (__any(top - m[n] > a.lag)) {
                top = fmaxf(m[n], lane_max4(top));
                const float f = exp2_hw((m[n] - (top == -INFINITY ? 0.0f : top)) * a.scale2);
                l[n] *= f;
#pragma unroll
                for (int e = 0; e < S::VE; e++) o[n][e] *= f;
                m[n] = top;
            }
            const float base = m[n] == -INFINITY ? 0.0f : m[n];
            uint32_t p[4];
            if constexpr (S::F32) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float x = exp2_hw((s[n][0][r] - base) * a.scale2);
                    l[n] += x;
                    p[r] = __float_as_uint(x);
                }
            } else {
                T h[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float x = exp2_hw(fmaf(s[n][j / 4][j % 4] - base, a.scale2, S::UP));
                    l[n] += x;
                    h[j] = (T)x;
                }
                __builtin_memcpy(p, h, 16);
            }
#pragma unroll
            for (int e = 0; e < S::VE; e++) o[n][e] = pv(e, p, o[n][e]);
            if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Chunk c's keys and values are in flight or here (cnv: how many of each
    // tile), the chunk after it is found (row, nv). Copies stand under no condition,
    // so that the compiler keeps count of them in its waits (past the end they read
    // nothing).
    uint32_t c = begin + kg * S::CK, cnv[S::TILES];
    auto advance = [&]() {
#pragma unroll
        for (int t = 0; t < S::TILES; t++) cnv[t] = nv[t];
        find(c + turn);
    };
    // Whether its keys are all there and committed.
    auto whole = [&]() {
        bool w = c + S::CK <= sq.past && cnv[0] == 16u;
        if constexpr (S::TILES > 1) w = w && cnv[1] == 16u;
        return w;
    };
    // A chunk that is not whole (the nodes', the last, one with a bad page): unseen
    // positions score -inf, and a node's values that are not finite become zeros, for
    // 0 times them would be NaN in rows that do not see the node. They join at the end.
    bool bad = false;
    auto mask = [&]() {
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t i = 4u * lk + r, p = c + 16u * t + i;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    // Selected, not branched over: the compiler lost the write of
                    // a branch here (ROCm 7.2, one f32 kernel).
                    const uint32_t j = p < sq.past ? 0u : p - sq.past;
                    const uint32_t ok =
                        sees_node(a, lwords[wave][16 * n + lm], lnode[wave][16 * n + lm],
                                  j < sq.nodes ? j : sq.nodes - 1u) |
                        (uint32_t)(p < sq.past);
                    s[n][t][r] = (ok & (uint32_t)(i < cnv[t])) ? s[n][t][r] : -INFINITY;
                }
#pragma unroll
                for (int x = 0; x < S::VP; x++)
#pragma unroll
                    for (int d = 0; d < S::VD; d++) {
                        const uint32_t fit = finite_part<T>(vr[t][r][x][d]);
                        const bool odd = p >= sq.past && fit != vr[t][r][x][d];
                        bad = bad || odd;
                        vr[t][r][x][d] = odd ? fit : vr[t][r][x][d];
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    find(c);
    if constexpr (RW == 1) {
        uint8_t *const k = kx + wave * S::KB, *const v = vx + wave * S::KB;
        auto chunk = [&]() {
            scores(k);
            load(kbase, k, 7u);
            read_v(v);
            if (!whole()) mask();
            weigh();
            __builtin_amdgcn_sched_barrier(0);     // the values have been read
            load(vbase, v, 0u);
            c += turn;
            advance();
        };
        load(kbase, k, 7u);
        load(vbase, v, 0u);
        advance();
        while (c < end) chunk();
    } else {
        const uint32_t mine = kg * S::KB;
        auto copy = [&](uint8_t *k, uint8_t *v) {
            load(kbase, k + mine, 7u);
            load(vbase, v + mine, 0u);
        };
        auto chunk = [&](const uint8_t *k, const uint8_t *v, uint8_t *next_k, uint8_t *next_v) {
            // The chunk has landed, and everybody is done with the one before.
            __builtin_amdgcn_s_waitcnt(0x0f70);    // vmcnt(0)
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            __builtin_amdgcn_sched_barrier(0);
            copy(next_k, next_v);
            scores(k + mine);
            read_v(v + mine);
            if (!whole()) mask();
            weigh();
            __builtin_amdgcn_sched_barrier(0);
            c += turn;
            advance();
        };
        copy(kx, vx);
        advance();
        // The same number of chunks, two by two, for every wave: past the end a chunk
        // is empty.
        for (uint32_t left = (end - begin + 2u * turn - 1u) / (2u * turn); left; left--) {
            chunk(kx, vx, ky, vy);
            chunk(ky, vy, kx, vx);
        }
    }

    // The waves' sums meet, a column tile at a time.
    // Place of dimension d (a multiple of 4, of the half in hand) of column `col` of
    // wave w's results.
    auto place = [&](uint32_t w, uint32_t col, uint32_t d) {
        return (float *)kx + (16u * w + col) * (HD / 2) +
               4u * ((d % (HD / 2) / 4u) ^ (col & 7u));
    };
    __builtin_amdgcn_s_waitcnt(0x0f70);                                 // no copy outlives the chunks' place
    if (__any(bad)) bad = true;
    __syncthreads();
    auto kept = [&](int i) { return (uint32_t)__builtin_amdgcn_readfirstlane(keep[i]); };
    const uint32_t id_ = kept(0), kvh_ = kept(1), wg0_ = kept(2), rows_ = kept(3), b_ = kept(5);
    const uint32_t begin_ = kept(6);
    const long long row0_ = (int32_t)kept(4);
#pragma unroll
    for (int h = 0; h < 2 * NT; h++) {
        const int n = h / 2;
        __syncthreads();                           // the chunks' place, or the last half's
        if (h % 2 == 0) {
            const float sum = lane_sum4(l[n]);
            if (lane == 0) lbad[wave] = bad;
            if (lk == 0) {
                lmax[wave][lm] = m[n];
                lsum[wave][lm] = sum;
            }
        }
        // Lane's dimensions: 16 CW c + CW (4 lk + r) + d.
#pragma unroll
        for (int x = 0; x < S::VP; x++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int d = 0; d < S::CW; d += 4) {
                    const uint32_t at = 16 * S::CW * x + S::CW * (4 * lk + r) + d;
                    if (at / (HD / 2) == h % 2)
                        *(float4 *)place(wave, lm, at) =
                            float4{o[n][x * S::CW + d][r], o[n][x * S::CW + d + 1][r],
                                   o[n][x * S::CW + d + 2][r], o[n][x * S::CW + d + 3][r]};
                }
        __syncthreads();
        // Each thread a run of four dimensions of a column.
        for (uint32_t i = threadIdx.x; i < 2u * HD * RW; i += 64u * S::W) {
            const uint32_t of = i / (2u * HD), col = i / (HD / 8u) % 16u;
            const uint32_t d = i % (HD / 8u) * 4u + h % 2 * (HD / 2u);
            const uint32_t rr = wg0_ + 16u * (NT * of + n) + col, nd = rr / a.group;
            const long long orow = row0_ + nd;
            if (rr >= rows_ || orow < 0 || orow >= (long long)a.n_rows) continue;
            float top = -INFINITY, all = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            uint32_t any_bad = 0u;
#pragma unroll
            for (int k = 0; k < KW; k++) {
                top = fmaxf(top, lmax[RW * k + of][col]);
                any_bad |= lbad[RW * k + of];
            }
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int k = 0; k < KW; k++) {
                const uint32_t w = RW * k + of;
                const float f = exp2_hw((lmax[w][col] - base) * a.scale2);
                const float4 x = *(const float4 *)place(w, col, d);
                all = fmaf(f, lsum[w][col], all);
                v[0] = fmaf(f, x.x, v[0]);
                v[1] = fmaf(f, x.y, v[1]);
                v[2] = fmaf(f, x.z, v[2]);
                v[3] = fmaf(f, x.w, v[3]);
            }
            const uint32_t head = kvh_ * a.group + rr - nd * a.group;
            if (any_bad) {
                // Infinities and NaN of the nodes this row sees: whatever their
                // share, the sum becomes theirs.
                for (uint32_t p = sq.past > begin_ ? sq.past : begin_; p < end; p++) {
                    unsigned long long r;
                    if (!sees_node(a, (size_t)orow * a.mask_words, nd, p - sq.past) ||
                        !cache_row(a, b_, p, r))
                        continue;
                    const T *x = (const T *)a.v + r * a.slot_stride + (size_t)kvh_ * HD + d;
                    for (int k = 0; k < 4; k++) {
                        const float y = (float)x[k];
                        if (!(fabsf(y) < INFINITY)) v[k] += y;
                    }
                }
            }
            if (a.slots > a.n_seqs) {
                const size_t at = (size_t)id_ * (16u * NT * RW) + (rr - wg0_);
                if (d == 0u) {
                    a.pm[at] = top;
                    a.pl[at] = all;
                }
                *(float4 *)(a.po + at * HD + d) = float4{v[0], v[1], v[2], v[3]};
            } else {
                const float inv = 1.0f / all;
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = all == 0.0f ? 0.0f : v[k] * inv;
                store4<true>((T *)a.out + (size_t)orow * a.out_stride + (size_t)head * HD + d, v);
            }
        }
    }
}

// The splits' partial sums to the output: a wave a (node, head). Grid (n_seqs,
// max_nodes, ceil(n_heads / 4)), block 256.
template <class T, int HD>
MYNAH_DEV void tree_join(const TreeArgs &a) {
    constexpr int E = HD / 64;
    const uint32_t b = blockIdx.x, nd = blockIdx.y;
    const uint32_t head = blockIdx.z * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const SeqSpan sq = seq_span(a, b);
    const long long row = sq.row0 + nd;
    if (nd >= sq.nodes || row < 0 || row >= (long long)a.n_rows || head >= a.n_heads) return;
    // A split's place in the partials, and how far the next split's is.
    const uint32_t kvh = head / a.group, rr = nd * a.group + head - kvh * a.group;
    const uint32_t part = rr / a.wg_rows;
    const bool one = a.n_seqs == 1u;
    const uint32_t first = one ? 0u : (uint32_t)scalar_i32(a.plan, 2u * b);
    const uint32_t splits = one ? a.slots : (uint32_t)scalar_i32(a.plan, 2u * b + 1u);
    const size_t step = (size_t)a.n_kv * a.groups * a.wg_rows;
    const size_t at = first * step + ((size_t)kvh * a.groups + part) * a.wg_rows +
                      (rr - part * a.wg_rows);
    // A split's maximum and sum to each lane, 64 of them at a time.
    float top = -INFINITY;
    for (uint32_t s = lane; s < splits; s += 64u) top = fmaxf(top, a.pm[s * step + at]);
    top = wave_max_dpp(top);
    const float base = top == -INFINITY ? 0.0f : top;
    float all = 0.0f, v[E];
#pragma unroll
    for (int i = 0; i < E; i++) v[i] = 0.0f;
    for (uint32_t s0 = 0u; s0 < splits; s0 += 64u) {
        const uint32_t n = splits - s0 < 64u ? splits - s0 : 64u;
        const size_t from = (s0 + lane) * step + at;
        const float w = lane < n ? exp2_hw((a.pm[from] - base) * a.scale2) : 0.0f;
        all += lane < n ? w * a.pl[from] : 0.0f;
        auto weight = [&](uint32_t s) {
            return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s));
        };
        const float *p = a.po + (s0 * step + at) * HD + E * lane;
        uint32_t s = 0u;
        for (; s + 8u <= n; s += 8u) {             // eight loads under way
            float x[8][E];
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int i = 0; i < E; i++) x[j][i] = p[(s + j) * step * HD + i];
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int i = 0; i < E; i++) v[i] = fmaf(weight(s + j), x[j][i], v[i]);
        }
        for (; s < n; s++)
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = fmaf(weight(s), p[s * step * HD + i], v[i]);
    }
    all = wave_sum(all);
    T *y = (T *)a.out + (size_t)row * a.out_stride + (size_t)head * HD + E * lane;
#pragma unroll
    for (int i = 0; i < E; i++) y[i] = (T)(all == 0.0f ? 0.0f : v[i] / all);
}

#define TREE_KERNEL(name, T, HD, NT, RW)                                                 \
    extern "C" __global__ void __launch_bounds__((64 * TaShape<T, HD>::W),               \
                                                 (TaShape<T, HD>::W / 4))                \
        mynah_tree_attn_##name##_##HD##_##NT##x##RW(TreeArgs a) {                        \
        tree_attn<T, HD, NT, RW>(a);                                                     \
    }
#define TREE_JOIN(name, T, HD)                                                           \
    extern "C" __global__ void __launch_bounds__(256) mynah_tree_join_##name##_##HD(     \
        TreeArgs a) { tree_join<T, HD>(a); }
TREE_KERNEL(f32, float, 64, 1, 1)
TREE_KERNEL(f32, float, 64, 1, 2)
TREE_KERNEL(f32, float, 128, 1, 1)
TREE_KERNEL(f32, float, 128, 1, 2)
TREE_KERNEL(f32, float, 256, 1, 1)
TREE_KERNEL(f32, float, 256, 1, 2)
#define TREE_KERNELS16(name, T) \
    TREE_KERNEL(name, T, 64, 1, 1)  \
    TREE_KERNEL(name, T, 64, 1, 2)  \
    TREE_KERNEL(name, T, 64, 2, 2)  \
    TREE_KERNEL(name, T, 64, 2, 4)  \
    TREE_KERNEL(name, T, 128, 1, 1) \
    TREE_KERNEL(name, T, 128, 1, 2) \
    TREE_KERNEL(name, T, 128, 2, 2) \
    TREE_KERNEL(name, T, 128, 2, 4) \
    TREE_KERNEL(name, T, 128, 2, 8) \
    TREE_KERNEL(name, T, 256, 1, 1) \
    TREE_KERNEL(name, T, 256, 1, 2) \
    TREE_KERNEL(name, T, 256, 1, 4)
TREE_KERNELS16(f16, _Float16)
TREE_KERNELS16(bf16, __bf16)
TREE_JOIN(f32, float, 64)
TREE_JOIN(f32, float, 128)
TREE_JOIN(f32, float, 256)
TREE_JOIN(f16, _Float16, 64)
TREE_JOIN(f16, _Float16, 128)
TREE_JOIN(f16, _Float16, 256)
TREE_JOIN(bf16, __bf16, 64)
TREE_JOIN(bf16, __bf16, 128)
TREE_JOIN(bf16, __bf16, 256)
