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
    unsigned long long n_slots;
    uint32_t n_seqs, n_kv, n_rows, page_log2, max_pages, block_log2, blocks, max_nodes, max_kv;
    uint32_t format, ragged;
};

// Units of a ragged batch: sequence b's blocks are numbered from (rows there before its
// own) / block + 2 b on, which leaves room for its rows / block + 2 of them, all that so many
// rows touch; a row is there in [0, n_rows), and a sequence's first block is its first such
// row's. The sequence of unit u is the last that begins at or before it, found by 64 lanes
// at a time. (Numbered by the longest sequence, a prompt of 8000 tokens beside 255
// single ones has 32,000 blocks, of which 380 are there.)
MYNAH_DEV uint32_t kv8_sequence(const Kv8StoreArgs &a, unsigned long long u, uint32_t &i) {
    const uint32_t lane = threadIdx.x & 63u;
    auto begins = [&](uint32_t b) {
        const int32_t row = a.seq_start[b], there = row < (int32_t)a.n_rows ? row : (int32_t)a.n_rows;
        return (unsigned long long)((uint32_t)(there > 0 ? there : 0) >> a.block_log2) + 2u * b;
    };
    uint32_t from = 0u, n = a.n_seqs;              // among from .. from + n - 1
    while (n > 1u) {
        const uint32_t step = (n + 63u) / 64u, b = from + lane * step;
        const bool low = lane * step < n && begins(b) <= u;
        const uint32_t upto = (uint32_t)__builtin_popcountll(__ballot(low));
        const uint32_t at = upto ? (upto - 1u) * step : 0u;        // none: before the first's
        from += at;
        n = n - at < step ? n - at : step;
    }
    from = __builtin_amdgcn_readfirstlane(from);
    const unsigned long long b0 = begins(from);
    i = u - b0 < a.blocks ? (uint32_t)(u - b0) : a.blocks;         // before or past its own: no block
    return from;
}

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
// an order. New values stay in registers between the largest and the rounding, up to
// HOLD runs of eight a thread; further ones are read twice. What bounds it: memory for
// a prompt (8190 bf16 tokens of 8 heads of 128 to e4m3, 50 MB, 13.7 us, 3.7 TB/s), for
// single tokens the launch and its reads one after the other (3.0-3.9 us, 256 tokens of
// as many sequences 4.5). Grid: units, heads fastest; block 64 W.
template <class T, int HD, int W, int HOLD>
MYNAH_DEV void kv8_store(const Kv8StoreArgs &a) {
    constexpr uint32_t LPR = HD / 8, RPS = 64 * W / LPR; // lanes of a row, rows a step
    __shared__ float top[W];
    unsigned long long u = blockIdx.x;
    const uint32_t h = (uint32_t)(u % a.n_kv);
    u /= a.n_kv;
    const uint32_t kv = (uint32_t)(u & 1u);
    u >>= 1;
    uint32_t i = a.ragged ? 0u : (uint32_t)(u % a.blocks);
    const uint32_t b = a.ragged ? kv8_sequence(a, u, i) : (uint32_t)(u / a.blocks);
    if (i >= a.blocks) return;                     // uniform
    const long long row0 = a.seq_start[b], n = a.seq_start[b + 1u] - row0;
    const uint32_t past = a.n_past[b] > 0 ? (uint32_t)a.n_past[b] : 0u;
    const uint32_t nodes = n <= 0 ? 0u : n < (long long)a.max_nodes ? (uint32_t)n : a.max_nodes;
    const unsigned long long all = (unsigned long long)past + nodes;
    const uint32_t end = all < a.max_kv ? (uint32_t)all : a.max_kv;
    const uint32_t bs = 1u << a.block_log2;
    // Rows before row 0, whose blocks a ragged batch does not number.
    const uint32_t skip = a.ragged && row0 < 0 ? (-row0 < (long long)nodes ? (uint32_t)-row0 : nodes) : 0u;
    const unsigned long long first64 =
        ((((unsigned long long)past + skip) >> a.block_log2) + i) << a.block_log2;
    if (first64 >= end || past >= end) return;
    const uint32_t first = (uint32_t)first64, from = first < past ? past : first;
    const uint32_t upto = end - first < bs ? end : first + bs;
    // A block none of whose rows are there keeps its scale.
    const long long r0 = row0 + (long long)(from - past);
    if (r0 >= (long long)a.n_rows || r0 + (long long)(upto - from) <= 0) return;
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
// three bf16 numbers each, weights of f16 calls two, and of bf16 calls two where rows are
// few: memory bounds those (32 queries over up to 16,384 positions 134 us both ways, 256
// over up to 2048 134 for 132). With many rows a bf16 call's weight is one number, 8 bits as
// its result has: a second one takes 399 us for 292 of a prompt of 2048 behind 6144, and
// halves the square of the error, which is the weights' and the result's rounding alike.
// The scales of a tile of 16 keys are one number each: the keys' joins the exponent's
// factor (one fma a score), the values' multiplies the probabilities.

struct Kv8Args {
    TreeArgs t;                     // k and v codes; scale2 1, for the join of log2 references
    const float *ks, *vs;
    uint32_t block_log2;
    float scale2;                   // |scale| log2(e)
};

typedef uint32_t kv8_v4u __attribute__((ext_vector_type(4)));
typedef uint32_t kv8_v2u __attribute__((ext_vector_type(2)));

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

// Bytes that are e4m3's NaN as zeros (of either sign), of those with bit 7 of `which`.
MYNAH_DEV uint32_t kv8_no_nan(uint32_t d, uint32_t which) {
    const uint32_t n = ((d & 0x7f7f7f7fu) + 0x01010101u) & which;
    return d & ~(n - (n >> 7));
}

template <class T, int HD, int NT = 1>
struct Kv8Shape {
    static constexpr bool F32 = sizeof(T) == 4, F16 = __is_same(T, _Float16);
    static constexpr int QN = F32 ? 3 : 1;              // numbers that a query value is
    static constexpr int PN = F32 ? 3 : 2;              // ... that a weight is
    static constexpr int TILES = HD * NT >= 256 ? 2 : 4; // 16-key tiles of a chunk
    static constexpr int CK = 16 * TILES;
    static constexpr int KP = HD / 64;                  // 16-byte pieces of a lane's key
    static constexpr int VE = HD / 16;                  // dimensions (O tiles) of a lane
    static constexpr int VD = HD / 64;                  // dwords of a lane's value row
    static constexpr int W = 4;                         // (= KV8_WAVES in kv8.c)
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

// The eight dimensions at q of a query as operands: step k of each of its numbers.
template <class T, int QN, int K>
MYNAH_DEV void kv8_query(const T *q, bool live, uint32_t flip, uint32_t (&qv)[QN][K][4], int k) {
    constexpr int D = sizeof(T) == 4 ? 8 : 4;
    uint32_t d[D];
    *(uint4 *)d = *(const uint4 *)q;
    if constexpr (D == 8) *(uint4 *)(d + 4) = *(const uint4 *)(q + 4);
#pragma unroll
    for (int i = 0; i < D; i++) d[i] = live ? d[i] ^ flip : 0u;
    if constexpr (D == 8) {
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

// A column's scores of TILES tiles, four a lane, become weights in two steps. First
// its reference, m, follows the largest; sum l and outputs o with it. References are
// in log2 units and lag by up to 2^8 in the probabilities.
template <int NT, int TILES, int VE>
MYNAH_DEV void kv8_refer(const float (&s)[NT][TILES][4], const float (&ks)[TILES], float (&m)[NT],
                         float (&l)[NT], ta_v4f (&o)[NT][VE]) {
    float top[NT];
    bool grown = false;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        top[n] = -INFINITY;
#pragma unroll
        for (int t = 0; t < TILES; t++)
            top[n] = fmaxf(top[n], fmaxf(fmaxf(s[n][t][0], s[n][t][1]),
                                         fmaxf(s[n][t][2], s[n][t][3])) * ks[t]);
        grown = grown || top[n] - m[n] > 8.0f;
    }
    if (!__any(grown)) return;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const float to = fmaxf(m[n], lane_max4(top[n]));
        const float f = exp2_hw(m[n] - (to == -INFINITY ? 0.0f : to));
        l[n] *= f;
#pragma unroll
        for (int e = 0; e < VE; e++) o[n][e] *= f;
        m[n] = to;
    }
}
// Then a tile's four scores become weights, rounded as two dwords of each of their PN
// numbers: fma takes a score's difference to the reference in one rounding.
template <int PN>
MYNAH_DEV void kv8_weigh(const float (&s)[4], float ks, float vs, float m, float &l,
                         uint32_t (&w)[PN][4], int half) {
    const float base = m == -INFINITY ? 0.0f : m;
    float p[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        p[r] = exp2_hw(fmaf(s[r], ks, -base));
        l += p[r];
        p[r] *= vs;
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int n = 0; n < PN; n++)
            w[n][2 * half + i] =
                n == PN - 1 ? kv8_round(p[2 * i], p[2 * i + 1]) : kv8_cut(p[2 * i], p[2 * i + 1]);
}

// Which of the CK <= 64 positions from c on (uniform) a query sees, as bits: node
// `node` of its sequence, its words of the mask from `words` on. Positions past the
// sequence's last are for the caller to leave out.
MYNAH_DEV uint64_t kv8_sees(const TreeArgs &a, size_t words, uint32_t node, uint32_t past,
                            uint32_t c) {
    const long long off = (long long)c - past;     // the first one's node
    if (!a.mask) {
        const long long n = (long long)node + 1 - off;
        return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1u;
    }
    auto word = [&](uint32_t i) -> uint64_t { return i < a.mask_words ? a.mask[words + i] : 0u; };
    if (off < 0) {
        const uint32_t n = off < -64 ? 64u : (uint32_t)-off;
        return n >= 64u ? ~0ull : (word(0) | word(1) << 32) << n | ((1ull << n) - 1u);
    }
    const uint32_t i = (uint32_t)off / 32u, sh = (uint32_t)off % 32u;
    const uint64_t low = word(i) | word(i + 1u) << 32;
    return sh ? low >> sh | word(i + 2u) << (64u - sh) : low;
}
// Bits of the positions that tiles have, lane t's of n rows.
template <int TILES>
MYNAH_DEV uint64_t kv8_there(uint32_t n) {
    uint64_t b = 0u;
#pragma unroll
    for (int t = 0; t < TILES; t++)
        b |= (uint64_t)((1u << __builtin_amdgcn_readlane(n, t)) - 1u) << (16 * t);
    return b;
}
// Scores of positions without their bit (the lane's first at bit 0) become -inf.
template <int TILES>
MYNAH_DEV void kv8_hide(float (&s)[TILES][4], uint64_t bits) {
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[t][r] = bits >> (16 * t + r) & 1u ? s[t][r] : -INFINITY;
}

// Four rows of four bytes, turned.
MYNAH_DEV void kv8_turn(const uint32_t (&x)[4], uint32_t (&y)[4]) {
    const uint32_t p0 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u);
    const uint32_t p1 = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
    const uint32_t p2 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
    const uint32_t p3 = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
    y[0] = __builtin_amdgcn_perm(p2, p0, 0x05040100u);
    y[1] = __builtin_amdgcn_perm(p2, p0, 0x07060302u);
    y[2] = __builtin_amdgcn_perm(p3, p1, 0x05040100u);
    y[3] = __builtin_amdgcn_perm(p3, p1, 0x07060302u);
}

// Four rows of four codes, x[row], as bf16 columns: y[column] has rows 0 and 1, 2 and 3.
// An integer's conversion takes its byte from any place, so nothing has to be turned:
// 46.1 -> 45.8 us for 32 bf16 queries over 4000 positions each, 61.6 -> 60.5 for 8 f16
// queries over 130,000.
template <int F>
MYNAH_DEV void kv8_columns(const uint32_t (&x)[4], uint32_t (&y)[4][2]) {
    if constexpr (F == KV_I8) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t f[4];
#pragma unroll
            for (int r = 0; r < 4; r++) f[r] = __float_as_uint((float)(int8_t)(x[r] >> (8 * i)));
            y[i][0] = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);
            y[i][1] = __builtin_amdgcn_perm(f[3], f[2], 0x07060302u);
        }
    } else {
        uint32_t d[4];
        kv8_turn(x, d);
#pragma unroll
        for (int i = 0; i < 4; i++) kv8_bf16<F>(d[i], y[i][0], y[i][1]);
    }
}

// Where a chunk's tiles of 16 positions lie: each lane has tile lane % TILES, and hands
// it out by readlane. What a chunk needs is read ahead in two steps, its pages' ids,
// then, from those, its scales, so that no wave waits for one read after the other.
// (As scalars the tiles took 200 scalar instructions a chunk and spilled.)
MYNAH_DEV uint32_t lane_of(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
MYNAH_DEV float lane_of(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

struct Kv8Tile {
    unsigned long long row;         // the first cache row
    uint32_t n;                     // how many of the 16 there are
};
template <int TILES>
struct Kv8Walk {
    const Kv8Args &g;
    uint32_t b, kvh, end, at;       // sequence, key head, positions' end, the lane's 16 t
    __device__ __forceinline__ Kv8Walk(const Kv8Args &g_, uint32_t b_, uint32_t kvh_, uint32_t end_)
        : g(g_), b(b_), kvh(kvh_), end(end_), at(threadIdx.x % TILES * 16u) {}
    __device__ __forceinline__ int32_t page(uint32_t c) const {
        if (!g.t.pages) return 0;
        const uint32_t p = c + at < end ? c + at : end - 1u;
        return g.t.pages[(size_t)b * g.t.max_pages + (p >> g.t.page_log2)];
    }
    __device__ __forceinline__ Kv8Tile tile(uint32_t c, int32_t id) const {
        const uint32_t p = c + at, low = p & ((1u << g.t.page_log2) - 1u);
        Kv8Tile x;
        x.row = g.t.pages ? ((unsigned long long)(uint32_t)id << g.t.page_log2) + low
                          : (unsigned long long)b * g.t.seq_slots + p;
        const bool there = p < end && id >= 0 && x.row < g.t.n_slots;   // whole blocks
        x.row = there ? x.row : 0u;
        x.n = !there ? 0u : end - p < 16u ? end - p : 16u;
        return x;
    }
    __device__ __forceinline__ void scales(const Kv8Tile &x, float &k, float &v) const {
        const size_t i = (size_t)(x.row >> g.block_log2) * g.t.n_kv + kvh;
        k = g.ks[i];
        v = g.vs[i];
    }
    // As the products take them: the keys' times the call's, in log2 units; 0 unless
    // positive and finite. The keys' is f32's least number in place of 0, so that -inf
    // stays what it is: 2^-149 of sums below 2^127 is 2^-22 of a score in log2 units.
    // Below f32's normal numbers a factor is off by half of that, as much again.
    __device__ __forceinline__ void settle(float k, float v, float (&ks)[TILES],
                                           float (&vs)[TILES]) const {
        k = fminf(fmaxf((k < INFINITY ? k : 0.0f) * g.scale2, 0x1p-149f), 3.402823466e38f);
        v = v > 0.0f && v < INFINITY ? v : 0.0f;
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            ks[t] = lane_of(k, t);
            vs[t] = lane_of(v, t);
        }
    }
    // The buffer of tile t (uniform) of rows of sb bytes: rows past its last are out of
    // range, are not read and become zeros.
    __device__ __forceinline__ auto buffer(const uint8_t *base, uint32_t sb, const Kv8Tile &x,
                                           int t) const {
        const unsigned long long row =
            (unsigned long long)lane_of((uint32_t)(x.row >> 32), t) << 32 | lane_of((uint32_t)x.row, t);
        return __builtin_amdgcn_make_buffer_rsrc((void *)(base + row * sb), 0, lane_of(x.n, t) * sb,
                                                 0x00020000);
    }
};

// A workgroup's W waves take chunks of CK keys in turn, for the same 16 NT queries,
// straight from memory into registers: a chunk's keys are under way while the one
// before is weighed, its values while its scores are made. The waves' results meet
// at the end. Four waves and two workgroups a CU, so that one's start and end stand
// beside the other's stream (one of eight: 170 us for 134, below). What bounds it:
// memory, as far as two waves a SIMD keep copies under way (widening an e4m3 chunk is
// 430 vector instructions, of i8 690, a quarter of the time). Measured: 32 sequences of
// up to 16,384 positions, one bf16 token each, 554 MB, 134 us, 4.1 TB/s; 8 f16 nodes
// over 130,009 i8 positions (266 MB) 67-74 us, 3.6-4.0 TB/s; 256 bf16 tokens over up to
// 2048 i8 positions (537 MB) 134 us; one f32 token over 513 12.1 us in two launches.
// Grid slots * n_kv * groups (of 16 NT query rows), block 64 W; the order of
// workgroups as in tree_attn.
template <class T, int F, int HD, int NT>
MYNAH_DEV void kv8_attn(const Kv8Args &g) {
    using S = Kv8Shape<T, HD, NT>;
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
    const uint32_t rows = sq.nodes * a.group, wg0 = grp * (16u * NT);
    if (wg0 >= rows) return;                       // uniform
    uint32_t per = __builtin_amdgcn_readfirstlane(share.per);
    if (per == 0u) {
        per = (sq.kv + a.slots - 1u) / a.slots;
        per = (per + turn - 1u) / turn * turn;
    }
    const unsigned long long from = (unsigned long long)split * per;
    const uint32_t begin = from < sq.kv ? (uint32_t)from : sq.kv;
    const uint32_t end = sq.kv - begin < per ? sq.kv : begin + per;

    // The lane's queries as operands: piece h of 16 dimensions is 16 (lk + 4 h) ..,
    // half j of it one step of the product.
    uint32_t node[NT], qv[NT][S::QN][2 * S::KP][4];
    size_t words[NT];
    float m[NT], l[NT];
    ta_v4f o[NT][S::VE];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const uint32_t rr = wg0 + 16u * j + lm;
        node[j] = rr / a.group;
        const long long qrow = sq.row0 + node[j];
        const bool live = rr < rows && qrow >= 0 && qrow < (long long)a.n_rows;
        words[j] = live ? (size_t)qrow * a.mask_words : 0;
        const T *q = (const T *)a.q + (live ? (size_t)qrow * a.q_stride : 0) +
                     (size_t)(kvh * a.group + rr - node[j] * a.group) * HD;
#pragma unroll
        for (int k = 0; k < 2 * S::KP; k++)
            kv8_query<T>(q + 16u * (lk + 4u * (k / 2)) + 8u * (k % 2), live, a.flip, qv[j], k);
        m[j] = -INFINITY;
        l[j] = 0.0f;
#pragma unroll
        for (int e = 0; e < S::VE; e++) o[j][e] = ta_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const uint32_t sb = (uint32_t)a.slot_stride;
    const uint8_t *kbase = (const uint8_t *)a.k + (size_t)kvh * HD;
    const uint8_t *vbase = (const uint8_t *)a.v + (size_t)kvh * HD;
    const Kv8Walk<S::TILES> walk(g, b, kvh, end);
    Kv8Tile x;                                     // of the chunk to be loaded
    int32_t ahead;                                 // the page of the one after it
    float ks[S::TILES], vs[S::TILES], nks, nvs;
    kv8_v4u kr[S::TILES][S::KP];
    uint32_t vr[S::TILES][4][S::VD];
    // Rows past a tile's last are out of its buffer's range, are not read and
    // become zeros.
    auto load_k = [&]() {
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            const auto kb = walk.buffer(kbase, sb, x, t);
#pragma unroll
            for (int h = 0; h < S::KP; h++)
                kr[t][h] = __builtin_amdgcn_raw_buffer_load_b128(
                    kb, __umul24(lm, sb) + 16u * lk, 64 * h, 0);
        }
    };
    auto load_v = [&]() {
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            const auto vb = walk.buffer(vbase, sb, x, t);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t at = __umul24(4u * lk + r, sb) + S::VE * lm;
                if constexpr (S::VD == 1) {
                    vr[t][r][0] = __builtin_amdgcn_raw_buffer_load_b32(vb, at, 0, 0);
                } else if constexpr (S::VD == 2) {
                    const kv8_v2u x = __builtin_amdgcn_raw_buffer_load_b64(vb, at, 0, 0);
                    vr[t][r][0] = x[0];
                    vr[t][r][1] = x[1];
                } else {
                    const kv8_v4u x = __builtin_amdgcn_raw_buffer_load_b128(vb, at, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) vr[t][r][i] = x[i];
                }
            }
        }
    };
    uint32_t c = begin + wave * S::CK, n;
    x = walk.tile(c, walk.page(c));
    ahead = walk.page(c + turn);
    load_k();
    load_v();
    walk.scales(x, nks, nvs);
    // The chunk at c becomes the current one, what the next ones need is read.
    auto advance = [&]() {
        walk.settle(nks, nvs, ks, vs);
        n = x.n;
        x = walk.tile(c + turn, ahead);
        walk.scales(x, nks, nvs);
        ahead = walk.page(c + 2u * turn);
    };
    while (c < end) {
        advance();
        float s[NT][S::TILES][4];
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            ta_v4f acc[NT];
#pragma unroll
            for (int j = 0; j < NT; j++) acc[j] = ta_v4f{0.0f, 0.0f, 0.0f, 0.0f};
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
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int i = S::QN - 1; i >= 0; i--) {
                        if constexpr (S::F16) acc[j] = ta_mfma<_Float16>(w, qv[j][i][k], acc[j]);
                        else acc[j] = ta_mfma<__bf16>(w, qv[j][i][k], acc[j]);
                    }
            }
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[j][t][r] = acc[j][r];
        }
        load_k();
        if (c + S::CK > sq.past || __any(n != 16u)) {
            // The nodes' chunk, the last, one with a bad page: unseen positions score
            // -inf, and a node's values that are NaN become zeros.
            const uint64_t there = kv8_there<S::TILES>(n);
#pragma unroll
            for (int j = 0; j < NT; j++)
                kv8_hide(s[j], (kv8_sees(a, words[j], node[j], sq.past, c) & there) >> (4u * lk));
            if constexpr (F == KV_E4M3)
#pragma unroll
                for (int t = 0; t < S::TILES; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int d = 0; d < S::VD; d++)
                            vr[t][r][d] = kv8_no_nan(
                                vr[t][r][d], c + 16u * t + 4u * lk + r < sq.past ? 0u : 0x80808080u);
        }
        uint32_t w[NT][S::TILES / 2][S::PN][4];
        kv8_refer(s, ks, m, l, o);
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int t = 0; t < S::TILES; t++)
                kv8_weigh(s[j][t], ks[t], vs[t], m[j], l[j], w[j][t / 2], t % 2);
        // Values: four keys' bytes of one dimension side by side, then widened.
#pragma unroll
        for (int u = 0; u < S::TILES / 2; u++)
#pragma unroll
            for (int d = 0; d < S::VD; d++) {
                uint32_t y[2][4][2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const uint32_t x[4] = {vr[2 * u + t][0][d], vr[2 * u + t][1][d],
                                           vr[2 * u + t][2][d], vr[2 * u + t][3][d]};
                    kv8_columns<F>(x, y[t]);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t va[4] = {y[0][e][0], y[0][e][1], y[1][e][0], y[1][e][1]};
#pragma unroll
                    for (int j = 0; j < NT; j++)
#pragma unroll
                        for (int i = S::PN - 1; i >= 0; i--)
                            o[j][4 * d + e] = ta_mfma<__bf16>(va, w[j][u][i], o[j][4 * d + e]);
                }
            }
        load_v();
        c += turn;
    }

    // The waves' sums meet, a column tile and half of the dimensions at a time. Lane's
    // dimensions: VE (4 lk + r) + e.
    auto place = [&](uint32_t w, uint32_t col, uint32_t d) {
        return part + (16u * w + col) * (HD / 2) + 4u * ((d % (HD / 2) / 4u) ^ (col & 7u));
    };
#pragma unroll
    for (int h = 0; h < 2 * NT; h++) {
        constexpr int HALF = HD / 2;
        const int j = h / 2;
        __syncthreads();
        if (h % 2 == 0) {
            const float sum = lane_sum4(l[j]);
            if (lk == 0) {
                lmax[wave][lm] = m[j];
                lsum[wave][lm] = sum;
            }
        }
        if (lk / 2u == (uint32_t)(h % 2))
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < S::VE; e += 4)
                    *(float4 *)place(wave, lm, S::VE * (4u * lk + r) + e) =
                        float4{o[j][e][r], o[j][e + 1][r], o[j][e + 2][r], o[j][e + 3][r]};
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 2u * HD; i += 64u * S::W) {
            const uint32_t col = i / (HD / 8u), d = i % (HD / 8u) * 4u + h % 2 * HALF;
            const uint32_t r = wg0 + 16u * j + col, nd = r / a.group;
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
                const size_t at = (size_t)id * (16u * NT) + 16u * j + col;
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

// ── many rows ───────────────────────────────────────────────────────────────
//
// A prompt's rows: the workgroup's waves share a chunk of CK keys, each with 16 NT
// rows of its own. Every code is widened once a workgroup: a chunk's codes come into
// registers while one before is computed, and leave for the LDS as bf16 (keys of f16
// calls f16), the values turned so that a lane reads eight keys of one dimension. Keys
// are a chunk ahead of values, so that the products of the next chunk's scores stand
// beside this one's exponentials. Two buffers of each, one barrier a chunk. Places in
// the LDS are 16-byte pieces, swapped so that 16 lanes of an access meet no bank twice.
//
// What bounds it: vector instructions (0.63 of the issue slots: 32 exponentials, their
// sums and roundings, 32 codes to widen a lane and chunk) beside the products (0.39 of
// the matrix cores' time); the LDS is busy 0.34. Then a chain's rows: a workgroup a CU
// stops at the last position its rows see, and the last one's sets the time. 2048 bf16
// tokens behind 6144 i8 positions, 32 heads, 8 of keys (7168 positions in the mean, 8192
// for the last rows): 289-331 us by box, 0.73-0.83 PFLOP/s, where a large product reaches
// 1.28; 2048 tokens of a new prompt (1 to 32 chunks) 86-92 us; f16 queries 385 us (their
// weights are two numbers), f32 584 (queries and weights three), on a box where bf16
// takes 289.
template <class T, int HD>
struct Kv8Wide {
    using S = Kv8Shape<T, HD>;
    static constexpr int W = 8;
    static constexpr int NT = S::F32 || HD == 256 ? 1 : 2;  // column tiles of a wave
    static constexpr int ROWS = 16 * NT * W;
    static constexpr int PN = S::F32 ? 3 : S::F16 ? 2 : 1;  // numbers that a weight is
    static constexpr int CK = HD == 256 ? 32 : 64, TILES = CK / 16;
    static constexpr int KS = HD / 32;              // steps of a score's product
    static constexpr int LB = HD == 64 ? 8 : 16;    // bytes of a thread's keys
    static constexpr int PR = CK / 8;               // pieces of a dimension's keys
    // Steps by which LDS reads lead their products; f16's second number a weight leaves
    // registers for two.
    static constexpr int AHEAD = S::F16 && HD == 128 ? 2 : 3;
};

template <class T, int F, int HD>
MYNAH_DEV void kv8_wide(const Kv8Args &g) {
    using S = Kv8Shape<T, HD>;
    using Z = Kv8Wide<T, HD>;
    constexpr int NT = Z::NT, TILES = Z::TILES;
    const TreeArgs &a = g.t;
    __shared__ uint4 kl[2][Z::CK * HD / 8], vl[2][Z::CK * HD / 8];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u, lm = lane & 15u, lk = lane >> 4;
    uint32_t id = blockIdx.x;
    const uint32_t even = gridDim.x & ~7u;
    if (id < even) id = (id & 7u) * (even >> 3) + (id >> 3);
    const uint32_t head_id = id / a.groups, slot = head_id / a.n_kv;
    const uint32_t kvh = head_id - slot * a.n_kv, grp = id - head_id * a.groups;
    SlotShare share = {slot, 0u, ~0u};
    if (a.slots > a.n_seqs) {                      // uniform
        if (a.n_seqs == 1u) share = {0u, slot, 0u};
        else if (!share_slots(a, slot, Z::CK, kvh == 0u && grp == 0u, share)) return;
    }
    const uint32_t b = __builtin_amdgcn_readfirstlane(share.b);
    const uint32_t split = __builtin_amdgcn_readfirstlane(share.split);
    const SeqSpan sq = seq_span(a, b);
    const uint32_t rows = sq.nodes * a.group, wg0 = grp * Z::ROWS;
    if (wg0 >= rows) return;                       // uniform
    uint32_t per = __builtin_amdgcn_readfirstlane(share.per);
    if (per == 0u) {
        per = (sq.kv + a.slots - 1u) / a.slots;
        per = (per + Z::CK - 1u) / Z::CK * Z::CK;
    }
    const unsigned long long from = (unsigned long long)split * per;
    const uint32_t begin = from < sq.kv ? (uint32_t)from : sq.kv;
    uint32_t end = sq.kv - begin < per ? sq.kv : begin + per;
    // The last position that a chain's rows see, of the workgroup and of the wave.
    const bool chain = a.mask == nullptr;
    const uint32_t w0 = wg0 + 16u * NT * wave;
    auto sees_upto = [&](uint32_t r) {
        const unsigned long long p = (unsigned long long)sq.past + (r < rows ? r : rows - 1u) / a.group + 1u;
        return p < end ? (uint32_t)p : end;
    };
    uint32_t mine = end;
    if (chain) {
        mine = w0 < rows ? sees_upto(w0 + 16u * NT - 1u) : begin;
        const uint32_t all = sees_upto(wg0 + Z::ROWS - 1u);
        end = all > begin ? all : begin;
    }
    const uint32_t first_node = (w0 < rows ? w0 : rows - 1u) / a.group;

    // Each wave's own: its columns' nodes, and their first words of the mask. In
    // registers they would spill.
    __shared__ uint32_t lnode[Z::W][16 * NT], lwords[Z::W][16 * NT];
    uint32_t qv[NT][S::QN][Z::KS][4];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t rr = w0 + 16u * n + lm;
        const uint32_t nd = rr / a.group;
        const long long qrow = sq.row0 + nd;
        const bool live = rr < rows && qrow >= 0 && qrow < (long long)a.n_rows;
        lnode[wave][16 * n + lm] = nd;
        lwords[wave][16 * n + lm] = live ? (uint32_t)qrow * a.mask_words : 0u;
        const T *q = (const T *)a.q + (live ? (size_t)qrow * a.q_stride : 0) +
                     (size_t)(kvh * a.group + rr - nd * a.group) * HD;
#pragma unroll
        for (int k = 0; k < Z::KS; k++) kv8_query<T>(q + 32u * k + 8u * lk, live, a.flip, qv[n], k);
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

    // A thread's part of a chunk: LB bytes of key tk, and four keys from 4 tv on of
    // four dimensions from td on.
    const uint32_t tk = threadIdx.x / (HD / Z::LB), tp = threadIdx.x % (HD / Z::LB);
    const uint32_t tv = threadIdx.x / (HD / 4), td = threadIdx.x % (HD / 4) * 4u;
    const bool has_v = 64 * Z::W == Z::CK / 4 * HD / 4 || tv < Z::CK / 4;
    const uint32_t sb = (uint32_t)a.slot_stride;
    const uint8_t *kbase = (const uint8_t *)a.k + (size_t)kvh * HD;
    const uint8_t *vbase = (const uint8_t *)a.v + (size_t)kvh * HD;
    uint32_t kc[4], vc[4];
    const Kv8Walk<TILES> walk(g, b, kvh, end);
    Kv8Tile x[2];                                  // of the next chunk, and the one after it
    int32_t ahead;                                 // the page of the third
    float ks[TILES], vs[TILES], nks[2], nvs[2];    // scales of the current one; of the next two
    uint32_t rows_now;                             // rows of the current one's tiles
    auto load_k = [&](const Kv8Tile &x) {
        const auto kb = walk.buffer(kbase, sb, x, __builtin_amdgcn_readfirstlane(tk / 16u));
        const uint32_t at = __umul24(tk & 15u, sb) + Z::LB * tp;
        if constexpr (Z::LB == 16) {
            const kv8_v4u x = __builtin_amdgcn_raw_buffer_load_b128(kb, at, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) kc[i] = x[i];
        } else {
            const kv8_v2u x = __builtin_amdgcn_raw_buffer_load_b64(kb, at, 0, 0);
            kc[0] = x[0];
            kc[1] = x[1];
        }
    };
    auto load_v = [&](const Kv8Tile &x) {
        if (!has_v) return;
        const auto vb = walk.buffer(vbase, sb, x, __builtin_amdgcn_readfirstlane(tv / 4u));
        const uint32_t at = __umul24(4u * tv & 15u, sb) + td;
#pragma unroll
        for (int r = 0; r < 4; r++)
            vc[r] = __builtin_amdgcn_raw_buffer_load_b32(vb, at + r * sb, 0, 0);
    };
    // Widened into the LDS. Key k's piece p (eight dimensions) lies at place p ^ swap(k)
    // of its row; keys 16 t + 4 i .. + 3 of dimension d are half t & 1 of piece 4 (t / 2)
    // + i of d's row, at place piece ^ turn(d).
    auto swap = [](uint32_t k) { return HD == 64 ? (k >> 1) & 7u : k & 15u; };
    auto turn = [](uint32_t d) { return Z::PR == 8 ? (d >> 1) & 7u : (d >> 2) & 3u; };
    // f16 calls have no registers for where a thread writes, and find it anew each time.
    auto anew = [](uint32_t v) {
        if constexpr (S::F16 && HD == 128) asm volatile("" : "+v"(v));
        return v;
    };
    auto widen_k = [&](int buf) {
        // Piece LB / 8 tp of key tk.
        const uint32_t i = anew(threadIdx.x), tk = i / (HD / Z::LB), tp = i % (HD / Z::LB);
        const uint32_t to = tk * (HD / 8) + ((Z::LB / 8 * tp) ^ swap(tk));
#pragma unroll
        for (int p = 0; p < Z::LB / 8; p++) {
            uint4 w;
            if constexpr (S::F16) {
                kv8_f16<F>(kc[2 * p], w.x, w.y);
                kv8_f16<F>(kc[2 * p + 1], w.z, w.w);
            } else {
                kv8_bf16<F>(kc[2 * p], w.x, w.y);
                kv8_bf16<F>(kc[2 * p + 1], w.z, w.w);
            }
            kl[buf][to ^ p] = w;                   // LB / 8 tp is even where p is not 0 alone
        }
    };
    auto widen_v = [&](uint32_t c, int buf) {
        if (!has_v) return;
        // td's half piece, in halves (turn(td + 2) is turn(td) ^ 1 for eight pieces a
        // row, and turn(td) for four).
        const uint32_t id = anew(threadIdx.x), tv = id / (HD / 4), td = id % (HD / 4) * 4u;
        const uint32_t to = 2u * (td * Z::PR + ((tv / 8u * 4u + (tv & 3u)) ^ turn(td))) + (tv / 4u & 1u);
        const auto put = [&](int i, uint2 w) {
            ((uint2 *)vl[buf])[(Z::PR == 8 ? to ^ (i & 2) : to) + 2 * i * Z::PR] = w;
        };
        // f16 kernels have the most to hold: 401 us -> 384 without the turn, where bf16's
        // 289 stay and f32's 584 become 590.
        if constexpr (F == KV_I8 && S::F16) {
            uint32_t y[4][2];
            kv8_columns<F>(vc, y);
#pragma unroll
            for (int i = 0; i < 4; i++) put(i, uint2{y[i][0], y[i][1]});
        } else {
            uint32_t y[4];
            kv8_turn(vc, y);
            if constexpr (F == KV_E4M3) {          // a node's NaN is 0
                const uint32_t p = c + 4u * tv, old = sq.past > p ? sq.past - p : 0u;
                const uint32_t nodes = old < 4u ? 0x80808080u << (8u * old) : 0u;
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = kv8_no_nan(y[i], nodes);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint2 w;
                kv8_bf16<F>(y[i], w.x, w.y);
                put(i, w);
            }
        }
    };

    // The lane's places: of piece 4 k + lk of key lm, and of 4 u + lk of dimension lm.
    constexpr int KA = HD == 64 ? 2 : 4;
    uint32_t kat[KA];
#pragma unroll
    for (int k = 0; k < KA; k++) kat[k] = lm * (HD / 8) + ((4u * k + lk) ^ swap(lm));
    uint32_t vat[TILES / 2];
#pragma unroll
    for (int u = 0; u < TILES / 2; u++) vat[u] = lm * Z::PR + ((4u * u + lk) ^ turn(lm));
    float s[2][NT][TILES][4];
    constexpr int SQ = TILES * Z::KS, SV = TILES / 2 * S::VE;  // steps of the two products
    auto key = [&](int buf, int i) {                           // a step's operands
        return kl[buf][kat[i % Z::KS % KA] + 16 * (i / Z::KS) * (HD / 8) + 4 * KA * (i % Z::KS / KA)];
    };
    auto value = [&](int buf, int i) { return vl[buf][vat[i / S::VE] + 16 * (i % S::VE) * Z::PR]; };
    // Step i of a chunk's scores: tile i / KS, dimensions 32 (i % KS) ..
    auto score = [&](float (&to)[NT][TILES][4], const uint4 &kk, int i) {
        const uint32_t w[4] = {kk.x, kk.y, kk.z, kk.w};
        const int t = i / Z::KS, k = i % Z::KS;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            ta_v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (k)
#pragma unroll
                for (int r = 0; r < 4; r++) x[r] = to[n][t][r];
#pragma unroll
            for (int j = S::QN - 1; j >= 0; j--) {
                if constexpr (S::F16) x = ta_mfma<_Float16>(w, qv[n][j][k], x);
                else x = ta_mfma<__bf16>(w, qv[n][j][k], x);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) to[n][t][r] = x[r];
        }
    };
    // Chunk c, whose scores are s[buf] and whose values are in buffer `buf`. The scores
    // of the next one, whose keys are in the other, are made beside its exponentials,
    // and the codes that have come are widened beside its second product, step by
    // step: the compiler by itself puts all products behind all else. Operands are
    // read AHEAD steps ahead.
    constexpr int AHEAD = Z::AHEAD, RING = AHEAD + 1;
    auto compute = [&](uint32_t c, int buf) {
        if (c + Z::CK > sq.past + (chain ? first_node : 0u) || __any(rows_now != 16u)) {
            const uint64_t there = kv8_there<TILES>(rows_now);
#pragma unroll
            for (int n = 0; n < NT; n++)
                kv8_hide(s[buf][n], (kv8_sees(a, lwords[wave][16 * n + lm], lnode[wave][16 * n + lm],
                                              sq.past, c) & there) >> (4u * lk));
        }
        uint4 op[RING];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) op[i] = key(1 - buf, i);
        kv8_refer(s[buf], ks, m, l, o);
        uint32_t w[NT][TILES / 2][Z::PN][4];
        constexpr int G = NT * TILES;              // tiles of all columns
#pragma unroll
        for (int i = 0; i < SQ; i++) {
            op[(i + AHEAD) % RING] = i + AHEAD < SQ ? key(1 - buf, i + AHEAD) : value(buf, i + AHEAD - SQ);
            score(s[1 - buf], op[i % RING], i);
#pragma unroll
            for (int j = i * G / SQ; j < (i + 1) * G / SQ; j++)
                kv8_weigh(s[buf][j % NT][j / NT], ks[j / NT], vs[j / NT], m[j % NT], l[j % NT],
                          w[j % NT][j / NT / 2], j / NT % 2);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < SV; i++) {
            const int at = SQ + i;
            if (i + AHEAD < SV) op[(at + AHEAD) % RING] = value(buf, i + AHEAD);
            const uint4 vv = op[at % RING];
            const uint32_t va[4] = {vv.x, vv.y, vv.z, vv.w};
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = Z::PN - 1; j >= 0; j--)
                    o[n][i % S::VE] = ta_mfma<__bf16>(va, w[n][i / S::VE][j], o[n][i % S::VE]);
            if (i == SV / 4) widen_k(buf);
            if (i == SV / 2) widen_v(c + Z::CK, 1 - buf);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    x[0] = walk.tile(begin, walk.page(begin));
    x[1] = walk.tile(begin + Z::CK, walk.page(begin + Z::CK));
    ahead = walk.page(begin + 2u * Z::CK);
    load_k(x[0]);
    load_v(x[0]);
    walk.scales(x[0], nks[0], nvs[0]);
    walk.scales(x[1], nks[1], nvs[1]);
    widen_k(0);
    load_k(x[1]);
    widen_v(begin, 0);
    widen_k(1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SQ; i++) score(s[0], key(0, i), i);
    __syncthreads();
    for (uint32_t c = begin; c < end; c += 2u * Z::CK) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t at = c + h * Z::CK;
            load_v(x[1]);
            walk.settle(nks[0], nvs[0], ks, vs);
            rows_now = x[0].n;
            x[0] = x[1];
            x[1] = walk.tile(at + 2u * Z::CK, ahead);
            load_k(x[1]);
            nks[0] = nks[1];
            nvs[0] = nvs[1];
            walk.scales(x[1], nks[1], nvs[1]);
            ahead = walk.page(at + 3u * Z::CK);
            if (at < mine) {
                compute(at, h);
            } else {
                widen_k(h);
                widen_v(at + Z::CK, 1 - h);
            }
            __syncthreads();
        }
    }

#pragma unroll
    for (int n = 0; n < NT; n++) {
        const float all = lane_sum4(l[n]);
        const uint32_t rr = w0 + 16u * n + lm;
        const uint32_t nd = rr / a.group;
        const long long orow = sq.row0 + nd;
        if (rr >= rows || orow < 0 || orow >= (long long)a.n_rows) continue;
        const size_t at = (size_t)id * Z::ROWS + (rr - wg0);
        const bool joined = a.slots > a.n_seqs;
        if (joined && lk == 0u) {
            a.pm[at] = m[n];
            a.pl[at] = all;
        }
        const float inv = 1.0f / all;
        T *y = (T *)a.out + (size_t)orow * a.out_stride +
               (size_t)(kvh * a.group + rr - nd * a.group) * HD;
#pragma unroll
        for (int e = 0; e < S::VE; e++) {
            const uint32_t d = 16u * e + 4u * lk;
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = joined ? o[n][e][r] : all == 0.0f ? 0.0f : o[n][e][r] * inv;
            if (joined) *(float4 *)(a.po + at * HD + d) = float4{v[0], v[1], v[2], v[3]};
            else store4<true>(y + d, v);
        }
    }
}

#define KV8_ATTN(name, T, fmt, F, HD, NT, WAVES)                                             \
    extern "C" __global__ void __launch_bounds__((64 * Kv8Shape<T, HD, NT>::W), WAVES)       \
        mynah_kv8_attn_##name##_##fmt##_##HD##_##NT(Kv8Args a) { kv8_attn<T, F, HD, NT>(a); }
#define KV8_WIDE(name, T, fmt, F, HD)                                                        \
    extern "C" __global__ void __launch_bounds__((64 * Kv8Wide<T, HD>::W), 2)                \
        mynah_kv8_wide_##name##_##fmt##_##HD(Kv8Args a) { kv8_wide<T, F, HD>(a); }
// Two waves a SIMD; one of f32 queries of 256 values, which take 96 registers.
#define KV8_ATTNS(name, T, fmt, F)                                              \
    KV8_ATTN(name, T, fmt, F, 64, 1, 2) KV8_ATTN(name, T, fmt, F, 64, 2, 2)     \
    KV8_ATTN(name, T, fmt, F, 128, 1, 2) KV8_ATTN(name, T, fmt, F, 128, 2, 2)   \
    KV8_ATTN(name, T, fmt, F, 256, 1, (sizeof(T) == 4 ? 1 : 2))                 \
    KV8_WIDE(name, T, fmt, F, 64) KV8_WIDE(name, T, fmt, F, 128) KV8_WIDE(name, T, fmt, F, 256)
KV8_ATTNS(f32, float, i8, KV_I8)
KV8_ATTNS(f32, float, e4m3, KV_E4M3)
KV8_ATTNS(f16, _Float16, i8, KV_I8)
KV8_ATTNS(f16, _Float16, e4m3, KV_E4M3)
KV8_ATTNS(bf16, __bf16, i8, KV_I8)
KV8_ATTNS(bf16, __bf16, e4m3, KV_E4M3)
