// kv8.hip — a key/value cache in 8 bits with a scale for each block of
// positions and head (include/mynah_cache.h): storing rows, and attention.
//
// SPDX-License-Identifier: MIT
#pragma once
#include "common.hip.h"
#include "elem.hip.h"
#include "tree_attn.hip"

enum { KV_I8 = 0, KV_E4M3 = 1 };

// ── rows into the cache ─────────────────────────────────────────────────────

struct Kv8StoreArgs {
    const void *x[2];               // new keys, new values
    size_t x_stride[2];
    uint8_t *c[2];
    float *s[2];
    const int32_t *seq_start, *n_past, *pages;
    size_t slot_stride, seq_slots;
    unsigned long long n_slots, units;
    uint32_t n_seqs, n_kv, n_rows, page_log2, max_pages, block_log2, blocks, max_nodes, max_kv;
    uint32_t format;
};

MYNAH_DEV float kv8_scale(float amax, uint32_t format) {
    if (format == KV_I8) return amax / 127.0f;
    const uint32_t q = __float_as_uint(amax / 448.0f);       // normal: amax >= 2^-100
    return __uint_as_float((q + 0x7fffffu) & 0x7f800000u);
}

// Four codes of x times inv.
MYNAH_DEV uint32_t kv8_codes(const float *x, float inv, uint32_t format) {
    float y[4];
    const float most = format == KV_I8 ? 127.0f : 448.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        y[i] = x[i] * inv;
        y[i] = y[i] != y[i] ? 0.0f : fminf(fmaxf(y[i], -most), most);
    }
    if (format == KV_I8) {
        uint32_t d = 0u;
#pragma unroll
        for (int i = 0; i < 4; i++) d |= ((uint32_t)(int)rintf(y[i]) & 0xffu) << (8 * i);
        return d;
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}

// The values of four codes.
MYNAH_DEV void kv8_values(uint32_t d, uint32_t format, float *x) {
    if (format == KV_I8) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (float)(int8_t)(d >> (8 * i));
    } else {
        x[0] = __builtin_amdgcn_cvt_f32_fp8((int)d, 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8((int)d, 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8((int)d, 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8((int)d, 3);
    }
}

// One workgroup of W waves takes one block of positions of a sequence, one head, of
// keys or of values, so that a block's scale has one owner and no result depends on
// an order. New values stay in registers between the largest and the rounding, up to HOLD runs of
// eight a thread; further ones are read twice. Grid: units, heads fastest; block 64 W.
template <class T, int HD, int W, int HOLD>
MYNAH_DEV void kv8_store(const Kv8StoreArgs &a) {
    constexpr uint32_t LPR = HD / 8, RPS = 64 * W / LPR; // lanes of a row, rows a step
    __shared__ float top[W];
    unsigned long long u = blockIdx.x;
    const uint32_t h = (uint32_t)(u % a.n_kv);
    u /= a.n_kv;
    const uint32_t kv = (uint32_t)(u & 1u);
    u >>= 1;
    const uint32_t i = (uint32_t)(u % a.blocks), b = (uint32_t)(u / a.blocks);
    const long long row0 = a.seq_start[b], n = a.seq_start[b + 1u] - row0;
    const uint32_t past = a.n_past[b] > 0 ? (uint32_t)a.n_past[b] : 0u;
    const uint32_t nodes = n <= 0 ? 0u : n < (long long)a.max_nodes ? (uint32_t)n : a.max_nodes;
    const unsigned long long all = (unsigned long long)past + nodes;
    const uint32_t end = all < a.max_kv ? (uint32_t)all : a.max_kv;
    const uint32_t bs = 1u << a.block_log2;
    const unsigned long long first64 = (((unsigned long long)past >> a.block_log2) + i) << a.block_log2;
    if (first64 >= end || past >= end) return;
    const uint32_t first = (uint32_t)first64, from = first < past ? past : first;
    const uint32_t upto = end - first < bs ? end : first + bs;
    unsigned long long slot = (unsigned long long)b * a.seq_slots + first;
    if (a.pages) {
        const int pg = a.pages[(size_t)b * a.max_pages + (first >> a.page_log2)];
        if (pg < 0) return;
        slot = ((unsigned long long)(uint32_t)pg << a.page_log2) + (first & ((1u << a.page_log2) - 1u));
    }
    if (slot >= a.n_slots) return;               // whole blocks: n_slots is so many
    float *scale = a.s[kv] + (slot >> a.block_log2) * a.n_kv + h;
    uint8_t *const codes = a.c[kv] + slot * a.slot_stride + h * HD;
    const uint32_t lr = threadIdx.x / LPR, e = threadIdx.x % LPR * 8u;
    const T *x = (const T *)a.x[kv] + h * HD + e;
    const size_t xs = a.x_stride[kv];
    // Row p's values, zeros where it has none.
    auto read = [&](uint32_t p, float *v) {
        const long long r = row0 + (long long)(p - past);
        const bool there = p < upto && r >= 0 && r < (long long)a.n_rows;
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = 0.0f;
        if (there) {
            load4<true>(x + (size_t)r * xs, v);
            load4<true>(x + (size_t)r * xs + 4, v + 4);
        }
        return there;
    };
    float m = 7.888609052210118e-31f;            // 2^-100
    auto largest = [&](const float *v) {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float t = fabsf(v[k]);
            m = fmaxf(m, t < INFINITY ? t : 0.0f);
        }
    };
    const float was = *scale;
    const float old = first < past && was > 0.0f && was < INFINITY ? was : 0.0f;
    float held[HOLD][8];
    bool there[HOLD];
#pragma unroll
    for (int k = 0; k < HOLD; k++) there[k] = read(from + lr + k * RPS, held[k]);
#pragma unroll
    for (int k = 0; k < HOLD; k++) largest(held[k]);
    for (uint32_t p = from + lr + HOLD * RPS; p < upto; p += RPS) {
        float v[8];
        read(p, v);
        largest(v);
    }
    m = wave_max_dpp(m);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63u) == 0u) top[threadIdx.x >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; w++) m = fmaxf(m, top[w]);
    }
    const float fresh = kv8_scale(m, a.format);
    const float now = first < past ? fmaxf(fresh, old) : fresh;
    const float inv = 1.0f / now;
    auto write = [&](uint32_t p, const float *v, float f) {
        *(uint2 *)(codes + (size_t)(p - first) * a.slot_stride + e) =
            uint2{kv8_codes(v, f, a.format), kv8_codes(v + 4, f, a.format)};
    };
#pragma unroll
    for (int k = 0; k < HOLD; k++)
        if (there[k]) write(from + lr + k * RPS, held[k], inv);
    for (uint32_t p = from + lr + HOLD * RPS; p < upto; p += RPS) {
        float v[8];
        if (read(p, v)) write(p, v, inv);
    }
    if (first >= past || now != old) {
        const float ratio = old / now;
        for (uint32_t p = first + lr; p < past; p += RPS) {
            const uint2 c = *(const uint2 *)(codes + (size_t)(p - first) * a.slot_stride + e);
            float v[8];
            kv8_values(c.x, a.format, v);
            kv8_values(c.y, a.format, v + 4);
            write(p, v, ratio);
        }
        if (threadIdx.x == 0u) *scale = now;
    }
}

#define KV8_STORE(name, T, HD)                                                               \
    extern "C" __global__ void __launch_bounds__(64) mynah_kv8_store_##name##_##HD##_1(      \
        Kv8StoreArgs a) { kv8_store<T, HD, 1, 1>(a); }                                       \
    extern "C" __global__ void __launch_bounds__(256) mynah_kv8_store_##name##_##HD##_4(     \
        Kv8StoreArgs a) { kv8_store<T, HD, 4, 4>(a); }
#define KV8_STORES(name, T) KV8_STORE(name, T, 64) KV8_STORE(name, T, 128) KV8_STORE(name, T, 256)
KV8_STORES(f32, float)
KV8_STORES(f16, _Float16)
KV8_STORES(bf16, __bf16)

// ── attention ───────────────────────────────────────────────────────────────
//
// As the tree attention of wider caches: a key head's queries are columns of 16
// of the matrix instruction, keys its rows, S^T = K Q^T and O^T = V^T P^T, so a
// lane's scores are the second product's operand. Codes are widened, exactly, to
// the 16-bit type of the product: keys to bf16, or to f16 for f16 queries; values to
// bf16, whose range holds a probability times any scale. What 16 bits do not hold
// of the other operand goes into further products: f32 queries and weights are
// three bf16 numbers each, weights of f16 calls two. The scales of a tile of 16 keys
// are one number each: the keys' joins the exponent's factor (one fma a score),
// the values' multiplies the probabilities.

struct Kv8Args {
    TreeArgs t;                     // k and v codes; scale2 1, for the join of log2 references
    const float *ks, *vs;
    uint32_t block_log2;
    float scale2;                   // |scale| log2(e)
};

typedef uint32_t kv8_v4u __attribute__((ext_vector_type(4)));
typedef uint32_t kv8_v2u __attribute__((ext_vector_type(2)));

typedef __attribute__((address_space(4))) const float kv8_const_f32;
MYNAH_DEV float scalar_f32(const float *p, size_t i) {
    return ((kv8_const_f32 *)(uintptr_t)p)[i];
}

template <class V>
MYNAH_DEV uint32_t as_u32(V v) {
    static_assert(sizeof(V) == 4, "");
    uint32_t d;
    __builtin_memcpy(&d, &v, 4);
    return d;
}

// Four codes as four bf16 numbers, in order: both formats' values are among them.
template <int F>
MYNAH_DEV void kv8_bf16(uint32_t c, uint32_t &lo, uint32_t &hi) {
    if constexpr (F == KV_E4M3) {
        lo = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, false));
        hi = as_u32(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, true));
    } else {
        uint32_t f[4];
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __float_as_uint((float)(int8_t)(c >> (8 * i)));
        lo = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);
        hi = __builtin_amdgcn_perm(f[3], f[2], 0x07060302u);
    }
}

// Four codes as four f16 numbers. Of an integer: 0x6400 + u is 1024 + u for a
// byte u, here the code plus 128.
template <int F>
MYNAH_DEV void kv8_f16(uint32_t c, uint32_t &lo, uint32_t &hi) {
    if constexpr (F == KV_E4M3) {
        lo = as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false));
        hi = as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, true));
    } else {
        typedef _Float16 v2h __attribute__((ext_vector_type(2)));
        const uint32_t u = c ^ 0x80808080u;
        uint32_t d[2] = {__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u),
                         __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            v2h h;
            __builtin_memcpy(&h, &d[i], 4);
            h -= (_Float16)1152.0f;
            __builtin_memcpy(&d[i], &h, 4);
        }
        lo = d[0];
        hi = d[1];
    }
}

// Bytes that are e4m3's NaN as zeros.
MYNAH_DEV uint32_t kv8_no_nan(uint32_t d) {
    const uint32_t n = ((d & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;   // bit 7 of such a byte
    return d & ~((n >> 7) * 0xffu);
}

template <class T, int HD>
struct Kv8Shape {
    static constexpr bool F32 = sizeof(T) == 4, F16 = __is_same(T, _Float16);
    static constexpr int QN = F32 ? 3 : 1;              // numbers that a query value is
    static constexpr int PN = F32 ? 3 : F16 ? 2 : 1;    // ... that a weight is
    static constexpr int TILES = HD == 256 ? 2 : 4;     // 16-key tiles of a chunk
    static constexpr int CK = 16 * TILES;
    static constexpr int KP = HD / 64;                  // 16-byte pieces of a lane's key
    static constexpr int VE = HD / 16;                  // dimensions (O tiles) of a lane
    static constexpr int VD = HD / 64;                  // dwords of a lane's value row
    static constexpr int W = 8;
};

// Two f32 numbers cut to bf16, and what is left of them.
MYNAH_DEV uint32_t kv8_cut(float &x, float &y) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    x -= __uint_as_float(a & 0xffff0000u);
    y -= __uint_as_float(b & 0xffff0000u);
    return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

MYNAH_DEV uint32_t kv8_round(float x, float y) {        // to bf16
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    return as_u32(v2b{(__bf16)x, (__bf16)y});
}

// A workgroup's W waves take chunks of CK keys in turn, for the same 16 queries,
// straight from memory into registers: a chunk's keys are under way while the one
// before is weighed, its values while its scores are made. The waves' results meet
// at the end. Grid slots * n_kv * groups (of 16 query rows), block 64 W; the order
// of workgroups as in tree_attn.
template <class T, int F, int HD>
MYNAH_DEV void kv8_attn(const Kv8Args &g) {
    using S = Kv8Shape<T, HD>;
    const TreeArgs &a = g.t;
    __shared__ __attribute__((aligned(16))) float part[S::W * 16 * HD / 2];
    __shared__ float lmax[S::W][16], lsum[S::W][16];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u, lm = lane & 15u, lk = lane >> 4;
    uint32_t id = blockIdx.x;
    const uint32_t even = gridDim.x & ~7u;
    if (id < even) id = (id & 7u) * (even >> 3) + (id >> 3);
    const uint32_t head_id = id / a.groups, slot = head_id / a.n_kv;
    const uint32_t kvh = head_id - slot * a.n_kv, grp = id - head_id * a.groups;
    const uint32_t turn = S::CK * S::W;
    SlotShare share = {slot, 0u, ~0u};
    if (a.slots > a.n_seqs) {                      // uniform
        if (a.n_seqs == 1u) share = {0u, slot, 0u};
        else if (!share_slots(a, slot, turn, kvh == 0u && grp == 0u, share)) return;
    }
    const uint32_t b = __builtin_amdgcn_readfirstlane(share.b);
    const uint32_t split = __builtin_amdgcn_readfirstlane(share.split);
    const SeqSpan sq = seq_span(a, b);
    const uint32_t rows = sq.nodes * a.group, wg0 = grp * 16u;
    if (wg0 >= rows) return;                       // uniform
    uint32_t per = __builtin_amdgcn_readfirstlane(share.per);
    if (per == 0u) {
        per = (sq.kv + a.slots - 1u) / a.slots;
        per = (per + turn - 1u) / turn * turn;
    }
    const unsigned long long from = (unsigned long long)split * per;
    const uint32_t begin = from < sq.kv ? (uint32_t)from : sq.kv;
    const uint32_t end = sq.kv - begin < per ? sq.kv : begin + per;

    // The lane's query as operands: piece h of 16 dimensions is 16 (lk + 4 h) ..,
    // half j of it one step of the product.
    const uint32_t rr = wg0 + lm, node = rr / a.group;
    const long long qrow = sq.row0 + node;
    const bool live = rr < rows && qrow >= 0 && qrow < (long long)a.n_rows;
    const size_t words = live ? (size_t)qrow * a.mask_words : 0;
    uint32_t qv[S::QN][2 * S::KP][4];
    {
        const T *q = (const T *)a.q + (live ? (size_t)qrow * a.q_stride : 0) +
                     (size_t)(kvh * a.group + rr - node * a.group) * HD;
#pragma unroll
        for (int k = 0; k < 2 * S::KP; k++) {
            const T *p = q + 16u * (lk + 4u * (k / 2)) + 8u * (k % 2);
            uint32_t d[S::F32 ? 8 : 4];
            *(uint4 *)d = *(const uint4 *)p;
            if constexpr (S::F32) *(uint4 *)(d + 4) = *(const uint4 *)(p + 4);
#pragma unroll
            for (int i = 0; i < (S::F32 ? 8 : 4); i++) d[i] = live ? d[i] ^ a.flip : 0u;
            if constexpr (S::F32) {
                float v[8];
                __builtin_memcpy(v, d, 32);
#pragma unroll
                for (int t = 0; t < 3; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) qv[t][k][i] = kv8_cut(v[2 * i], v[2 * i + 1]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) qv[0][k][i] = d[i];
            }
        }
    }
    float m = -INFINITY, l = 0.0f;
    ta_v4f o[S::VE];
#pragma unroll
    for (int e = 0; e < S::VE; e++) o[e] = ta_v4f{0.0f, 0.0f, 0.0f, 0.0f};

    // Tiles of the next chunk: the first cache row, how many of the 16 there are,
    // their scales (the keys' times the call's, in log2 units).
    const uint32_t sb = (uint32_t)a.slot_stride;
    const uint8_t *kbase = (const uint8_t *)a.k + (size_t)kvh * HD;
    const uint8_t *vbase = (const uint8_t *)a.v + (size_t)kvh * HD;
    unsigned long long row[S::TILES];
    uint32_t nv[S::TILES], cnv[S::TILES];
    float ks[S::TILES], vs[S::TILES], cks[S::TILES], cvs[S::TILES];
    auto find = [&](uint32_t c) {
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            const uint32_t p = c + 16u * t;
            row[t] = 0;
            nv[t] = 0;
            ks[t] = vs[t] = 0.0f;
            unsigned long long r;
            if (p >= end || !cache_row(a, b, p, r)) continue;
            row[t] = r;
            nv[t] = end - p < 16u ? end - p : 16u;   // n_slots is whole blocks
            const size_t at = (size_t)(r >> g.block_log2) * a.n_kv + kvh;
            ks[t] = scalar_f32(g.ks, at);
            vs[t] = scalar_f32(g.vs, at);
        }
    };
    kv8_v4u kr[S::TILES][S::KP];
    uint32_t vr[S::TILES][4][S::VD];
    // Rows past a tile's last are out of its buffer's range, are not read and
    // become zeros.
    auto rsrc = [&](const uint8_t *base, int t) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)(base + row[t] * sb), 0, nv[t] * sb,
                                                 0x00020000);
    };
    auto load_k = [&]() {
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
#pragma unroll
            for (int h = 0; h < S::KP; h++)
                kr[t][h] = __builtin_amdgcn_raw_buffer_load_b128(
                    rsrc(kbase, t), __umul24(lm, sb) + 16u * lk, 64 * h, 0);
    };
    auto load_v = [&]() {
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t at = __umul24(4u * lk + r, sb) + S::VE * lm;
                if constexpr (S::VD == 1) {
                    vr[t][r][0] = __builtin_amdgcn_raw_buffer_load_b32(rsrc(vbase, t), at, 0, 0);
                } else if constexpr (S::VD == 2) {
                    const kv8_v2u x = __builtin_amdgcn_raw_buffer_load_b64(rsrc(vbase, t), at, 0, 0);
                    vr[t][r][0] = x[0];
                    vr[t][r][1] = x[1];
                } else {
                    const kv8_v4u x = __builtin_amdgcn_raw_buffer_load_b128(rsrc(vbase, t), at, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) vr[t][r][i] = x[i];
                }
            }
    };
    uint32_t c = begin + wave * S::CK;
    auto advance = [&]() {
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            cnv[t] = nv[t];
            const float k = ks[t] < INFINITY ? ks[t] : 0.0f;      // NaN: 0 by fmaxf
            cks[t] = fminf(fmaxf(k * g.scale2, 1e-30f), 3.402823466e38f);
            cvs[t] = vs[t] > 0.0f && vs[t] < INFINITY ? vs[t] : 0.0f;
        }
        find(c + turn);
    };
    find(c);
    load_k();
    load_v();
    advance();
    while (c < end) {
        float s[S::TILES][4];
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            ta_v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 2 * S::KP; k++) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint32_t d = kr[t][k / 2][2 * (k % 2) + i];
                    if constexpr (S::F16) kv8_f16<F>(d, w[2 * i], w[2 * i + 1]);
                    else kv8_bf16<F>(d, w[2 * i], w[2 * i + 1]);
                }
#pragma unroll
                for (int n = S::QN - 1; n >= 0; n--) {
                    if constexpr (S::F16) x = ta_mfma<_Float16>(w, qv[n][k], x);
                    else x = ta_mfma<__bf16>(w, qv[n][k], x);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) s[t][r] = x[r];
        }
        load_k();
        bool whole = c + S::CK <= sq.past;
#pragma unroll
        for (int t = 0; t < S::TILES; t++) whole = whole && cnv[t] == 16u;
        if (!whole) {
            // The nodes' chunk, the last, one with a bad page: unseen positions score
            // -inf, and a node's values that are NaN become zeros.
#pragma unroll
            for (int t = 0; t < S::TILES; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t i = 4u * lk + r, p = c + 16u * t + i;
                    const uint32_t j = p < sq.past ? 0u : p - sq.past;
                    const uint32_t ok = sees_node(a, words, node, j < sq.nodes ? j : sq.nodes - 1u) |
                                        (uint32_t)(p < sq.past);
                    s[t][r] = (ok & (uint32_t)(i < cnv[t])) ? s[t][r] : -INFINITY;
                    if constexpr (F == KV_E4M3)
#pragma unroll
                        for (int d = 0; d < S::VD; d++)
                            vr[t][r][d] = p < sq.past ? vr[t][r][d] : kv8_no_nan(vr[t][r][d]);
                }
        }
        // References are in log2 units; fma takes a score's difference to its column's
        // in one rounding. They lag by up to 2^8 in the probabilities.
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
            top = fmaxf(top, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])) * cks[t]);
        if (__any(top - m > 8.0f)) {
            top = fmaxf(m, lane_max4(top));
            const float f = exp2_hw(m - (top == -INFINITY ? 0.0f : top));
            l *= f;
#pragma unroll
            for (int e = 0; e < S::VE; e++) o[e] *= f;
            m = top;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        uint32_t w[S::TILES / 2][S::PN][4];
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            float p[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                p[r] = exp2_hw(fmaf(s[t][r], cks[t], -base));
                l += p[r];
                p[r] *= cvs[t];
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int n = 0; n < S::PN; n++)
                    w[t / 2][n][2 * (t % 2) + i] = n == S::PN - 1
                                                       ? kv8_round(p[2 * i], p[2 * i + 1])
                                                       : kv8_cut(p[2 * i], p[2 * i + 1]);
        }
        // Values: four keys' bytes of one dimension side by side, then widened.
#pragma unroll
        for (int u = 0; u < S::TILES / 2; u++)
#pragma unroll
            for (int d = 0; d < S::VD; d++) {
                uint32_t y[2][4];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const uint32_t(&x)[4][S::VD] = vr[2 * u + t];
                    const uint32_t p0 = __builtin_amdgcn_perm(x[1][d], x[0][d], 0x05010400u);
                    const uint32_t p1 = __builtin_amdgcn_perm(x[1][d], x[0][d], 0x07030602u);
                    const uint32_t p2 = __builtin_amdgcn_perm(x[3][d], x[2][d], 0x05010400u);
                    const uint32_t p3 = __builtin_amdgcn_perm(x[3][d], x[2][d], 0x07030602u);
                    y[t][0] = __builtin_amdgcn_perm(p2, p0, 0x05040100u);
                    y[t][1] = __builtin_amdgcn_perm(p2, p0, 0x07060302u);
                    y[t][2] = __builtin_amdgcn_perm(p3, p1, 0x05040100u);
                    y[t][3] = __builtin_amdgcn_perm(p3, p1, 0x07060302u);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t va[4];
                    kv8_bf16<F>(y[0][e], va[0], va[1]);
                    kv8_bf16<F>(y[1][e], va[2], va[3]);
#pragma unroll
                    for (int n = S::PN - 1; n >= 0; n--)
                        o[4 * d + e] = ta_mfma<__bf16>(va, w[u][n], o[4 * d + e]);
                }
            }
        load_v();
        c += turn;
        advance();
    }

    // The waves' sums meet, half of the dimensions at a time. Lane's dimensions:
    // VE (4 lk + r) + e.
    const float sum = lane_sum4(l);
    if (lk == 0) {
        lmax[wave][lm] = m;
        lsum[wave][lm] = sum;
    }
    auto place = [&](uint32_t w, uint32_t col, uint32_t d) {
        return part + (16u * w + col) * (HD / 2) + 4u * ((d % (HD / 2) / 4u) ^ (col & 7u));
    };
#pragma unroll
    for (int h = 0; h < 2; h++) {
        __syncthreads();
        if (lk / 2u == (uint32_t)h)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < S::VE; e += 4)
                    *(float4 *)place(wave, lm, S::VE * (4u * lk + r) + e) =
                        float4{o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]};
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 2u * HD; i += 64u * S::W) {
            const uint32_t col = i / (HD / 8u), d = i % (HD / 8u) * 4u + h * (HD / 2u);
            const uint32_t r = wg0 + col, nd = r / a.group;
            const long long orow = sq.row0 + nd;
            if (r >= rows || orow < 0 || orow >= (long long)a.n_rows) continue;
            float best = -INFINITY, all = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < S::W; w++) best = fmaxf(best, lmax[w][col]);
            const float base = best == -INFINITY ? 0.0f : best;
#pragma unroll
            for (int w = 0; w < S::W; w++) {
                const float f = exp2_hw(lmax[w][col] - base);
                const float4 x = *(const float4 *)place(w, col, d);
                all = fmaf(f, lsum[w][col], all);
                v[0] = fmaf(f, x.x, v[0]);
                v[1] = fmaf(f, x.y, v[1]);
                v[2] = fmaf(f, x.z, v[2]);
                v[3] = fmaf(f, x.w, v[3]);
            }
            if (a.slots > a.n_seqs) {
                const size_t at = (size_t)id * 16u + col;
                if (d == 0u) {
                    a.pm[at] = best;
                    a.pl[at] = all;
                }
                *(float4 *)(a.po + at * HD + d) = float4{v[0], v[1], v[2], v[3]};
            } else {
                const float inv = 1.0f / all;
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = all == 0.0f ? 0.0f : v[k] * inv;
                store4<true>((T *)a.out + (size_t)orow * a.out_stride +
                                 (size_t)(kvh * a.group + r - nd * a.group) * HD + d, v);
            }
        }
    }
}

#define KV8_ATTN(name, T, fmt, F, HD)                                                        \
    extern "C" __global__ void __launch_bounds__((64 * Kv8Shape<T, HD>::W), 2)               \
        mynah_kv8_attn_##name##_##fmt##_##HD(Kv8Args a) { kv8_attn<T, F, HD>(a); }
#define KV8_ATTNS(name, T, HD) \
    KV8_ATTN(name, T, i8, KV_I8, HD) KV8_ATTN(name, T, e4m3, KV_E4M3, HD)
KV8_ATTNS(f32, float, 64)
KV8_ATTNS(f32, float, 128)
KV8_ATTNS(f32, float, 256)
KV8_ATTNS(f16, _Float16, 64)
KV8_ATTNS(f16, _Float16, 128)
KV8_ATTNS(f16, _Float16, 256)
KV8_ATTNS(bf16, __bf16, 64)
KV8_ATTNS(bf16, __bf16, 128)
KV8_ATTNS(bf16, __bf16, 256)
