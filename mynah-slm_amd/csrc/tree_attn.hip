// tree_attn.hip — attention of drafted tokens over a key/value cache
// (include/mynah_attention.h, mynah_hip_tree_attention_dev).
//
// A key head's queries (its group of heads, of every node: row = node * group +
// head) are columns of 16 of the matrix instruction, keys its rows: S^T = K
// Q^T, so that a lane holds four keys' scores of one query, which is what the
// second product O^T = V^T P^T takes as its operand: the probabilities never
// leave their registers. Which key and which dimension an operand's place
// stands for is free as long as both operands agree, so K and V are read from
// memory in whole runs of 8 or 16 bytes a lane into the operands' registers;
// 16-bit V is turned by one v_perm per two values. No LDS in the loop and no
// barrier: each wave walks its own chunks of keys with its own running maximum
// and sum; the waves meet once at the end, workgroups in a second launch.
//
// SPDX-License-Identifier: MIT
#pragma once
#include "common.hip.h"
#include "elem.hip.h"

// Waves of a workgroup, each with its own keys (= MYNAH_TA_WAVES in
// runtime_internal.h).
#define TA_WAVES 4

struct TreeArgs {
    const void *q, *k, *v;
    void *out;
    size_t q_stride, out_stride, slot_stride, seq_slots;
    const int32_t *pages, *seq_start, *n_past;
    const uint32_t *mask;
    float *pm, *pl, *po;            // partials [split][n_rows * n_heads], (x head_dim)
    unsigned long long n_slots;
    uint32_t n_seqs, n_heads, n_kv, group, n_rows, page_log2, max_pages, mask_words;
    uint32_t max_nodes, max_kv, splits;
    float scale2;                   // scale * log2(e)
};

typedef float ta_v4f __attribute__((ext_vector_type(4)));
typedef _Float16 ta_v8h __attribute__((ext_vector_type(8)));
typedef __bf16 ta_v8b __attribute__((ext_vector_type(8)));

struct SeqSpan {
    long long row0;                 // first query row
    uint32_t nodes, past, kv;
};

// A sequence's rows and positions as the call bounds them.
MYNAH_DEV SeqSpan seq_span(const TreeArgs &a, uint32_t b) {
    SeqSpan s;
    s.row0 = a.seq_start[b];
    const long long n = (long long)a.seq_start[b + 1u] - s.row0;
    const int past = a.n_past[b];
    s.nodes = n <= 0 ? 0u : n < (long long)a.max_nodes ? (uint32_t)n : a.max_nodes;
    s.past = past > 0 ? (uint32_t)past : 0u;
    const unsigned long long kv = (unsigned long long)s.past + s.nodes;
    s.kv = kv < a.max_kv ? (uint32_t)kv : a.max_kv;
    return s;
}

MYNAH_DEV float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// What an element type and head size make of the operands.
template <class T, int HD>
struct TaShape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int TILES = F32 ? 1 : 2;         // 16-key tiles of a chunk
    static constexpr int CK = 16 * TILES;             // keys of a chunk
    static constexpr int KP = F32 ? HD / 16 : HD / 32; // 16-byte pieces of a lane's key
    static constexpr int VE = HD / 16;                // dimensions (O tiles) of a lane
    static constexpr int CW = F32 || HD == 64 ? 4 : 8; // of them side by side
    static constexpr int VP = VE / CW;                // pieces of a lane's value row
    static constexpr int VD = CW * (int)sizeof(T) / 4; // dwords of a piece
};

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

// A register of one f32 or two 16-bit values: whether it holds an infinity or
// NaN, and the register with zeros in their place.
template <class T>
MYNAH_DEV uint32_t finite_part(uint32_t d) {
    if constexpr (sizeof(T) == 4) return (d & 0x7f800000u) == 0x7f800000u ? 0u : d;
    constexpr uint32_t e = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    return ((d & e) == e ? 0u : d & 0xffffu) | (((d >> 16) & e) == e ? 0u : d & 0xffff0000u);
}
template <class T>
MYNAH_DEV bool not_finite(uint32_t d) { return finite_part<T>(d) != d; }

// Whether a query (node `node` of its sequence, its words of the mask from
// `words` on) sees node j, as 0 or 1.
MYNAH_DEV uint32_t sees_node(const TreeArgs &a, size_t words, uint32_t node, uint32_t j) {
    if (a.mask == nullptr) return j <= node;
    return (a.mask[words + j / 32u] >> (j & 31u)) & 1u;
}

// The cache row of position p of sequence b; false where it is not in the cache.
MYNAH_DEV bool cache_row(const TreeArgs &a, uint32_t b, uint32_t p, unsigned long long &row) {
    unsigned long long r = (unsigned long long)b * a.seq_slots + p;
    if (a.pages) {
        const int pg = a.pages[(size_t)b * a.max_pages + (p >> a.page_log2)];
        if (pg < 0) return false;
        r = ((unsigned long long)(uint32_t)pg << a.page_log2) + (p & ((1u << a.page_log2) - 1u));
    }
    row = r;
    return r < a.n_slots;
}

// Grid (n_seqs * n_kv, splits, row groups of 16 NT), block 64 TA_WAVES.
template <class T, int HD, int NT>
MYNAH_DEV void tree_attn(const TreeArgs &a) {
    using S = TaShape<T, HD>;
    __shared__ __attribute__((aligned(16))) float lo[TA_WAVES][16][HD + 4];
    __shared__ float lm_[TA_WAVES][16], ll_[TA_WAVES][16];
    __shared__ uint32_t lbad[TA_WAVES];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u, lm = lane & 15u, lk = lane >> 4;
    const uint32_t b = blockIdx.x / a.n_kv, kvh = blockIdx.x - b * a.n_kv, split = blockIdx.y;
    const SeqSpan sq = seq_span(a, b);
    const uint32_t rows = sq.nodes * a.group, rr0 = blockIdx.z * (16u * NT);
    if (rr0 >= rows) return;                       // uniform
    uint32_t per = (sq.kv + a.splits - 1u) / a.splits;
    per = (per + S::CK * TA_WAVES - 1u) / (S::CK * TA_WAVES) * (S::CK * TA_WAVES);
    const uint32_t begin = split * per < sq.kv ? split * per : sq.kv;
    const uint32_t end = sq.kv - begin < per ? sq.kv : begin + per;

    // This lane's query of each column tile.
    uint32_t qv[NT][S::KP][4], node[NT];
    size_t qwords[NT];              // its first word of the mask
#pragma unroll
    for (int n = 0; n < NT; n++) {
        // Columns that are no query (past the rows) take row 0 and hold zeros.
        const uint32_t rr = rr0 + 16u * n + lm, nd = rr / a.group;
        const long long qrow = sq.row0 + nd;
        const bool live = rr < rows && qrow >= 0 && qrow < (long long)a.n_rows;
        node[n] = nd;
        qwords[n] = live ? (size_t)qrow * a.mask_words : 0;
        const char *p = (const char *)a.q + ((live ? (size_t)qrow * a.q_stride : 0) +
                                             (size_t)(kvh * a.group + rr - nd * a.group) * HD) *
                                                sizeof(T);
#pragma unroll
        for (int c = 0; c < S::KP; c++) {
            const uint4 x = *(const uint4 *)(p + 64u * c + 16u * lk);
            qv[n][c][0] = live ? x.x : 0u;
            qv[n][c][1] = live ? x.y : 0u;
            qv[n][c][2] = live ? x.z : 0u;
            qv[n][c][3] = live ? x.w : 0u;
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
    uint32_t kr[S::TILES][S::KP][4], vr[S::TILES][4][S::VP][S::VD];
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
    // Rows past a tile's last are read as its last (of none, as row 0 of the
    // cache).
    auto load_k = [&]() {
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            const uint32_t most = nv[t] ? nv[t] - 1u : 0u;
            const char *p = kbase + row[t] * sb;
            const uint32_t at = (lm < most ? lm : most) * sb + 16u * lk;
#pragma unroll
            for (int c = 0; c < S::KP; c++) load_dwords<4>(p + (at + 64u * c), kr[t][c]);
        }
    };
    auto load_v = [&]() {
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            const uint32_t most = nv[t] ? nv[t] - 1u : 0u;
            const char *p = vbase + row[t] * sb;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t i = 4u * lk + r;
                const uint32_t at = (i < most ? i : most) * sb + lm * (uint32_t)(S::CW * sizeof(T));
#pragma unroll
                for (int c = 0; c < S::VP; c++)
                    load_dwords<S::VD>(p + (at + c * (uint32_t)(16 * S::CW * sizeof(T))),
                                       vr[t][r][c]);
            }
        }
    };
    // Probabilities (lane's keys) as the second product's operand, and that
    // product for tile e of the dimensions.
    struct Probs { uint32_t d[4]; };
    auto probs = [&](const float (&p)[S::TILES][4]) {
        Probs o;
        if constexpr (S::F32) {
#pragma unroll
            for (int r = 0; r < 4; r++) o.d[r] = __float_as_uint(p[0][r]);
        } else {
            T h[8];
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] = (T)p[j / 4][j % 4];
            __builtin_memcpy(o.d, h, 16);
        }
        return o;
    };
    auto pv = [&](int e, const Probs &p, ta_v4f acc) {
        const int c = e / S::CW;
        if constexpr (S::F32) {
#pragma unroll
            for (int r = 0; r < 4; r++)
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[0][r][c][e % 4]),
                                                           __uint_as_float(p.d[r]), acc, 0, 0, 0);
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
            return ta_mfma<T>(va, p.d, acc);
        }
    };
    bool bad = false;

    uint32_t c = begin + wave * S::CK;
    if (c < end) {
        find(c);
        load_k();
        load_v();
    }
    while (c < end) {
        const uint32_t next = c + S::CK * TA_WAVES;
        uint32_t cnv[S::TILES];
        bool whole = c + S::CK <= sq.past;
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            cnv[t] = nv[t];
            whole = whole && nv[t] == 16u;
        }
        // Scores: lane's query (column lm) against keys 4 lk + r of each tile.
        float s[NT][S::TILES][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int t = 0; t < S::TILES; t++) {
                ta_v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < S::KP; k++) {
                    if constexpr (S::F32) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            x = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __uint_as_float(kr[t][k][i]), __uint_as_float(qv[n][k][i]), x, 0,
                                0, 0);
                    } else {
                        x = ta_mfma<T>(kr[t][k], qv[n][k], x);
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++) s[n][t][r] = x[r] * a.scale2;
            }
        if (next < end) {
            find(next);
            load_k();
        }
        if (!whole) {
            // Unseen positions score -inf. Rows that are not there hold zeros,
            // and so do a node's values that are not finite: 0 times them would
            // be NaN in rows that do not see the node. They join at the end.
#pragma unroll
            for (int t = 0; t < S::TILES; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t i = 4u * lk + r, p = c + 16u * t + i;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        // Selected, not branched over: the compiler lost the
                        // write of a branch here (ROCm 7.2, one f32 kernel).
                        const uint32_t j = p < sq.past ? 0u : p - sq.past;
                        const uint32_t ok =
                            sees_node(a, qwords[n], node[n], j < sq.nodes ? j : sq.nodes - 1u) |
                            (uint32_t)(p < sq.past);
                        s[n][t][r] = (ok & (uint32_t)(i < cnv[t])) ? s[n][t][r] : -INFINITY;
                    }
#pragma unroll
                    for (int x = 0; x < S::VP; x++)
#pragma unroll
                        for (int d = 0; d < S::VD; d++) {
                            const bool odd = p >= sq.past && not_finite<T>(vr[t][r][x][d]);
                            bad = bad || (odd && i < cnv[t]);
                            if (i >= cnv[t]) vr[t][r][x][d] = 0u;
                            else if (odd) vr[t][r][x][d] = finite_part<T>(vr[t][r][x][d]);
                        }
                }
        }
        Probs pr[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < S::TILES; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) top = fmaxf(top, s[n][t][r]);
            top = fmaxf(m[n], lane_max4(top));
            const float base = top == -INFINITY ? 0.0f : top;
            if (__any(top > m[n])) {
                const float f = exp2_hw(m[n] - base);
                l[n] *= f;
#pragma unroll
                for (int e = 0; e < S::VE; e++) o[n][e] *= f;
            }
            m[n] = top;
#pragma unroll
            for (int t = 0; t < S::TILES; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    s[n][t][r] = exp2_hw(s[n][t][r] - base);
                    l[n] += s[n][t][r];
                }
            pr[n] = probs(s[n]);
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < S::VE; e++) o[n][e] = pv(e, pr[n], o[n][e]);
        if (next < end) load_v();
        c = next;
    }

    // The waves' sums meet, a column tile at a time.
    if (__any(bad)) bad = true;
    if (lane == 0) lbad[wave] = bad;
    const size_t heads_all = (size_t)a.n_rows * a.n_heads;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const float sum = lane_sum4(l[n]);
        if (n) __syncthreads();
        if (lk == 0) {
            lm_[wave][lm] = m[n];
            ll_[wave][lm] = sum;
        }
        // Lane's dimensions: 16 CW c + CW (4 lk + r) + d.
#pragma unroll
        for (int x = 0; x < S::VP; x++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int d = 0; d < S::CW; d++)
                    lo[wave][lm][16 * S::CW * x + S::CW * (4 * lk + r) + d] = o[n][x * S::CW + d][r];
        __syncthreads();
        // 16 threads a column, each every 16th run of four dimensions.
        const uint32_t col = threadIdx.x >> 4, ln = threadIdx.x & 15u;
        const uint32_t rr = rr0 + 16u * n + col, nd = rr / a.group;
        const long long orow = sq.row0 + nd;
        if (rr < rows && orow >= 0 && orow < (long long)a.n_rows) {
            float top = -INFINITY, w[TA_WAVES], all = 0.0f;
#pragma unroll
            for (int i = 0; i < TA_WAVES; i++) top = fmaxf(top, lm_[i][col]);
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int i = 0; i < TA_WAVES; i++) {
                w[i] = exp2_hw(lm_[i][col] - base);
                all = fmaf(w[i], ll_[i][col], all);
            }
            const uint32_t head = kvh * a.group + rr - nd * a.group;
            const float inv = a.splits > 1u ? 1.0f : all == 0.0f ? 0.0f : 1.0f / all;
            const size_t at = split * heads_all + (size_t)orow * a.n_heads + head;
            if (a.splits > 1u && ln == 0u) {
                a.pm[at] = top;
                a.pl[at] = all;
            }
            for (uint32_t d = 4u * ln; d < HD; d += 64u) {
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < TA_WAVES; i++)
#pragma unroll
                    for (int k = 0; k < 4; k++) v[k] = fmaf(w[i], lo[i][col][d + k], v[k]);
                if (lbad[0] | lbad[1] | lbad[2] | lbad[3]) {
                    // Infinities and NaN of the nodes this row sees: whatever
                    // their share, the sum becomes theirs.
                    for (uint32_t p = sq.past > begin ? sq.past : begin; p < end; p++) {
                        unsigned long long r;
                        if (!sees_node(a, (size_t)orow * a.mask_words, nd, p - sq.past) ||
                            !cache_row(a, b, p, r))
                            continue;
                        const T *x = (const T *)a.v + r * a.slot_stride + (size_t)kvh * HD + d;
                        for (int k = 0; k < 4; k++) {
                            const float y = (float)x[k];
                            if (!(fabsf(y) < INFINITY)) v[k] += y;
                        }
                    }
                }
                if (a.splits > 1u) {
                    *(float4 *)(a.po + at * HD + d) = float4{v[0], v[1], v[2], v[3]};
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) v[k] = all == 0.0f ? 0.0f : v[k] * inv;
                    store4<true>((T *)a.out + (size_t)orow * a.out_stride + (size_t)head * HD + d,
                                 v);
                }
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
    const size_t heads_all = (size_t)a.n_rows * a.n_heads;
    const size_t at = (size_t)row * a.n_heads + head;
    float top = -INFINITY;
    for (uint32_t s = 0; s < a.splits; s++) top = fmaxf(top, a.pm[s * heads_all + at]);
    const float base = top == -INFINITY ? 0.0f : top;
    float all = 0.0f, v[E];
#pragma unroll
    for (int i = 0; i < E; i++) v[i] = 0.0f;
    for (uint32_t s = 0; s < a.splits; s++) {
        const float w = exp2_hw(a.pm[s * heads_all + at] - base), ls = a.pl[s * heads_all + at];
        all = fmaf(w, ls, all);
        const float *p = a.po + (s * heads_all + at) * HD + E * lane;
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = fmaf(w, p[i], v[i]);
    }
    T *y = (T *)a.out + (size_t)row * a.out_stride + (size_t)head * HD + E * lane;
#pragma unroll
    for (int i = 0; i < E; i++) y[i] = (T)(all == 0.0f ? 0.0f : v[i] / all);
}

#define TREE_KERNEL(name, T, HD, NT, W)                                                  \
    extern "C" __global__ void __launch_bounds__(64 * TA_WAVES, W)                       \
        mynah_tree_attn_##name##_##HD##_##NT(TreeArgs a) { tree_attn<T, HD, NT>(a); }
#define TREE_JOIN(name, T, HD)                                                           \
    extern "C" __global__ void __launch_bounds__(256) mynah_tree_join_##name##_##HD(     \
        TreeArgs a) { tree_join<T, HD>(a); }
TREE_KERNEL(f32, float, 64, 1, 2)
TREE_KERNEL(f32, float, 64, 2, 2)
TREE_KERNEL(f32, float, 128, 1, 2)
TREE_KERNEL(f32, float, 128, 2, 2)
TREE_KERNEL(f32, float, 256, 1, 1)
#define TREE_KERNELS16(name, T)   \
    TREE_KERNEL(name, T, 64, 1, 2)  \
    TREE_KERNEL(name, T, 64, 2, 2)  \
    TREE_KERNEL(name, T, 64, 4, 2)  \
    TREE_KERNEL(name, T, 128, 1, 2) \
    TREE_KERNEL(name, T, 128, 2, 2) \
    TREE_KERNEL(name, T, 128, 4, 1) \
    TREE_KERNEL(name, T, 256, 1, 1) \
    TREE_KERNEL(name, T, 256, 2, 1)
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
