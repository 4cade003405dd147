// logits.hip — rules on a batch's logits (include/mynah_generate.h,
// mynah_hip_logits_dev): penalties for repeated tokens, biases, grammar masks.
//
// A workgroup takes LG_CH tokens of one row. Their logits are under way while it
// counts, in the LDS, how often each occurs in the row's history (every workgroup of
// a row reads all of it), and which bias is each one's: integer sums and maxima, so
// that no result depends on an order.
//
// What bounds it: memory, then the lists' latency and the LDS. 192 rows of 151,936, bf16 to
// f32, histories of 2049 to 4096 tokens, biases, grammars (178 MB) 60-65 us by box, 2.7-3.0
// TB/s, 36 with no rule at all (4.9 TB/s), with the histories alone 60, biases 41, grammars
// 38; with inputs in the last-level cache 41-44, and 27 with no rule. Half or twice the
// tokens a workgroup took 57 and 56 us for 47 in an earlier form.
//
// SPDX-License-Identifier: MIT
#pragma once
#include "common.hip.h"
#include "elem.hip.h"

struct LogitsArgs {
    const void *x;
    void *y;
    size_t x_stride, y_stride;
    const int32_t *hist;
    const int64_t *hist_start;
    const float *repeat, *freq, *presence;
    const int32_t *bias_id;
    const float *bias;
    const int64_t *bias_start;
    const uint32_t *allowed;
    const int32_t *mask_row;
    uint32_t vocab, chunks, mask_words, n_masks, each, vec;
};

#define LG_T 512u
#define LG_CH 8192u                 // tokens of a workgroup (= MYNAH_LOGITS_CH)

// An element that no kernel writes while this one runs, by a scalar load.
template <class V>
MYNAH_DEV V scalar_at(const V *p, size_t i) {
    typedef __attribute__((address_space(4))) const V C;
    return ((C *)(uintptr_t)p)[i];
}

MYNAH_DEV float penalised(float l, uint32_t count, float rep, float freq, float pres,
                          uint32_t each) {
#pragma clang fp contract(off)
    for (uint32_t k = each ? count : 1u; k; k--) {
        const float was = l;
        l = l > 0.0f ? l / rep : l * rep;
        l -= freq * (float)count;
        l -= pres;
        if (l == was) break;                       // and so would be every further one
    }
    return l;
}

// Entries from..to of a list of ids, LG_N a thread at a time: f(token of the chunk,
// entry) for those that fall in it. The first LG_N of a thread are read once.
#define LG_N 8u
struct LogitsList {
    const int32_t *ids;
    int64_t from, to;
    uint32_t c0, n, held[LG_N];
    __device__ __forceinline__ void read(int64_t base, uint32_t (&t)[LG_N]) const {
#pragma unroll
        for (uint32_t j = 0; j < LG_N; j++) {
            const int64_t k = base + threadIdx.x + LG_T * j;
            t[j] = k < to ? (uint32_t)ids[k] - c0 : ~0u;
        }
    }
    __device__ __forceinline__ void open(const int32_t *ids_, int64_t from_, int64_t to_,
                                         uint32_t c0_, uint32_t n_) {
        ids = ids_;
        from = from_;
        to = to_;
        c0 = c0_;
        n = n_;
        read(from, held);
    }
    template <class G>
    __device__ __forceinline__ void each(G &&f) const {
#pragma unroll
        for (uint32_t j = 0; j < LG_N; j++)
            if (held[j] < n) f(held[j], (uint32_t)(threadIdx.x + LG_T * j));
        for (int64_t base = from + LG_N * LG_T; base < to; base += LG_N * LG_T) {
            uint32_t t[LG_N];
            read(base, t);
#pragma unroll
            for (uint32_t j = 0; j < LG_N; j++)
                if (t[j] < n) f(t[j], (uint32_t)(base - from + threadIdx.x + LG_T * j));
        }
    }
};

// Grid chunks * rows, block LG_T.
template <class T, class O>
MYNAH_DEV void logits(const LogitsArgs &a) {
#pragma clang fp contract(off)
    constexpr uint32_t N = LG_CH / (4u * LG_T);    // runs of four tokens of a thread
    // How often a token occurs; then, counted from 1, which bias it gets.
    __shared__ __attribute__((aligned(16))) uint32_t info[LG_CH];
    const uint32_t r = blockIdx.x / a.chunks, c0 = (blockIdx.x - r * a.chunks) * LG_CH;
    const uint32_t n = a.vocab - c0 < LG_CH ? a.vocab - c0 : LG_CH, tid = threadIdx.x;
    // The row's own first, then what depends on them and the logits, all at once: of
    // seven reads one after the other a workgroup took 13 us.
    const float rep = a.repeat ? scalar_at(a.repeat, r) : 1.0f;
    const float freq = a.freq ? scalar_at(a.freq, r) : 0.0f;
    const float pres = a.presence ? scalar_at(a.presence, r) : 0.0f;
    int64_t h0 = 0, h1 = 0, b0 = 0, b1 = 0, m = -1;
    if (a.hist) {
        h0 = scalar_at(a.hist_start, r);
        h1 = scalar_at(a.hist_start, r + 1u);
    }
    if (a.bias_id) {
        b0 = scalar_at(a.bias_start, r);
        b1 = scalar_at(a.bias_start, r + 1u);
    }
    if (a.allowed) m = a.mask_row ? scalar_at(a.mask_row, r) : (int64_t)r;
    const T *x = (const T *)a.x + (size_t)r * a.x_stride + c0;
    O *y = (O *)a.y + (size_t)r * a.y_stride + c0;
    if (rep == 1.0f && freq == 0.0f && pres == 0.0f) h1 = h0;
    const bool count = h1 > h0, bias = b1 > b0;    // uniform
    const bool masked = m >= 0 && m < (int64_t)a.n_masks;
    LogitsList seen, wanted;
    seen.open(a.hist, h0, h1, c0, n);
    wanted.open(a.bias_id, b0, b1, c0, n);
    // Lists first, so that nobody who waits for them waits for the logits.
    Elem4<T> raw[N];
#pragma unroll
    for (uint32_t k = 0; k < N; k++) {
        const uint32_t i = 4u * (tid + LG_T * k);
        if (a.vec && i + 4u <= n) {
            raw[k] = *(const Elem4<T> *)(x + i);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++) raw[k].e[j] = i + j < n ? x[i + j] : (T)0.0f;
        }
    }
    const uint32_t *allowed = a.allowed + (masked ? (size_t)m * a.mask_words + c0 / 32u : 0);
    uint32_t words[N];
#pragma unroll
    for (uint32_t k = 0; k < N; k++) {
        const uint32_t i = 4u * (tid + LG_T * k);
        words[k] = masked && i < n ? allowed[i / 32u] : ~0u;
    }
    if (count || bias) {
#pragma unroll
        for (uint32_t k = 0; k < N; k++) *(uint4 *)&info[4u * (tid + LG_T * k)] = uint4{0u, 0u, 0u, 0u};
        __syncthreads();
    }
    if (count) {
        seen.each([&](uint32_t t, uint32_t) { atomicAdd(&info[t], 1u); });
        __syncthreads();
    }
    float v[N][4];
#pragma unroll
    for (uint32_t k = 0; k < N; k++)
#pragma unroll
        for (uint32_t j = 0; j < 4u; j++) v[k][j] = (float)raw[k].e[j];
    if (count) {
#pragma unroll
        for (uint32_t k = 0; k < N; k++) {
            const uint4 c4 = *(const uint4 *)&info[4u * (tid + LG_T * k)];
            const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
            if (c4.x | c4.y | c4.z | c4.w) {
                if (bias) *(uint4 *)&info[4u * (tid + LG_T * k)] = uint4{0u, 0u, 0u, 0u};
#pragma unroll
                for (uint32_t j = 0; j < 4u; j++)
                    if (c[j]) v[k][j] = penalised(v[k][j], c[j], rep, freq, pres, a.each);
            }
        }
    }
    if (bias) {
        if (count) __syncthreads();
        // A bias by its place in the row's list; of several the last.
        wanted.each([&](uint32_t t, uint32_t k) { atomicMax(&info[t], k + 1u); });
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < N; k++) {
            const uint4 w4 = *(const uint4 *)&info[4u * (tid + LG_T * k)];
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
            if (w4.x | w4.y | w4.z | w4.w)
#pragma unroll
                for (uint32_t j = 0; j < 4u; j++)
                    if (w[j]) v[k][j] += a.bias[b0 + (w[j] - 1u)];
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < N; k++) {
        const uint32_t i = 4u * (tid + LG_T * k);
        if (i >= n) break;
        const uint32_t word = words[k] >> (i % 32u);
#pragma unroll
        for (uint32_t j = 0; j < 4u; j++) v[k][j] = (word >> j) & 1u ? v[k][j] : -INFINITY;
        if (a.vec && i + 4u <= n) {
            store4<true>(y + i, v[k]);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++)
                if (i + j < n) y[i + j] = (O)v[k][j];
        }
    }
}

#define LOGITS(name, T, out, O)                                                     \
    extern "C" __global__ void __launch_bounds__(LG_T, 8) mynah_logits_##name##_##out( \
        LogitsArgs a) { logits<T, O>(a); }
#define LOGITS_OF(name, T) \
    LOGITS(name, T, f32, float) LOGITS(name, T, f16, _Float16) LOGITS(name, T, bf16, __bf16)
LOGITS_OF(f32, float)
LOGITS_OF(f16, _Float16)
LOGITS_OF(bf16, __bf16)
