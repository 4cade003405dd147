// logits.hip — rules on a batch's logits (include/mynah_generate.h,
// mynah_hip_logits_dev): penalties for repeated tokens, biases, grammar masks.
//
// A workgroup takes LG_CH tokens of one row. Their logits are under way while it
// counts, in the LDS, how often each occurs in the row's history (every workgroup of
// a row reads all of it), and which bias is each one's: integer sums and maxima, so that no result
// depends on an order.
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

// Grid chunks * rows, block LG_T.
template <class T, class O>
MYNAH_DEV void logits(const LogitsArgs &a) {
#pragma clang fp contract(off)
    constexpr uint32_t N = LG_CH / (4u * LG_T);    // runs of four tokens of a thread
    __shared__ uint32_t counts[LG_CH], biased[LG_CH];
    const uint32_t r = blockIdx.x / a.chunks, c0 = (blockIdx.x - r * a.chunks) * LG_CH;
    const uint32_t n = a.vocab - c0 < LG_CH ? a.vocab - c0 : LG_CH, tid = threadIdx.x;
    const T *x = (const T *)a.x + (size_t)r * a.x_stride + c0;
    O *y = (O *)a.y + (size_t)r * a.y_stride + c0;
    float v[N][4];
#pragma unroll
    for (uint32_t k = 0; k < N; k++) {
        const uint32_t i = 4u * (tid + LG_T * k);
        if (a.vec && i + 4u <= n) {
            load4<true>(x + i, v[k]);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++) v[k][j] = i + j < n ? (float)x[i + j] : 0.0f;
        }
    }
    const float rep = a.repeat ? a.repeat[r] : 1.0f, freq = a.freq ? a.freq[r] : 0.0f;
    const float pres = a.presence ? a.presence[r] : 0.0f;
    int64_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    if (a.hist && !(rep == 1.0f && freq == 0.0f && pres == 0.0f)) {
        h0 = a.hist_start[r];
        h1 = a.hist_start[r + 1u];
    }
    if (a.bias_id) {
        b0 = a.bias_start[r];
        b1 = a.bias_start[r + 1u];
    }
    const bool count = h1 > h0, bias = b1 > b0;    // uniform
    if (count || bias) {
        for (uint32_t i = tid; i < LG_CH; i += LG_T) counts[i] = biased[i] = 0u;
        __syncthreads();
        for (int64_t k = h0 + tid; k < h1; k += LG_T) {
            const uint32_t t = (uint32_t)a.hist[k] - c0;
            if (t < n) atomicAdd(&counts[t], 1u);
        }
        // A bias by its place in the row's list, one up; of several the last.
        for (int64_t k = b0 + tid; k < b1; k += LG_T) {
            const uint32_t t = (uint32_t)a.bias_id[k] - c0;
            if (t < n) atomicMax(&biased[t], (uint32_t)(k - b0) + 1u);
        }
        __syncthreads();
    }
    const int64_t m = a.allowed ? (a.mask_row ? a.mask_row[r] : (int64_t)r) : -1;
    const bool masked = m >= 0 && m < (int64_t)a.n_masks;
    const uint32_t *allowed = a.allowed + (masked ? (size_t)m * a.mask_words + c0 / 32u : 0);
#pragma unroll
    for (uint32_t k = 0; k < N; k++) {
        const uint32_t i = 4u * (tid + LG_T * k);
        if (i >= n) break;
        if (count || bias) {
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++) {
                const uint32_t c = counts[i + j], at = biased[i + j];
                if (c) v[k][j] = penalised(v[k][j], c, rep, freq, pres, a.each);
                if (at) v[k][j] += a.bias[b0 + at - 1];
            }
        }
        const uint32_t word = masked ? allowed[i / 32u] >> (i % 32u) : ~0u;
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
    extern "C" __global__ void __launch_bounds__(LG_T) mynah_logits_##name##_##out( \
        LogitsArgs a) { logits<T, O>(a); }
#define LOGITS_OF(name, T) \
    LOGITS(name, T, f32, float) LOGITS(name, T, f16, _Float16) LOGITS(name, T, bf16, __bf16)
LOGITS_OF(f32, float)
LOGITS_OF(f16, _Float16)
LOGITS_OF(bf16, __bf16)
