// draft.hip — the small kernels around a verification step of drafted tokens
// (mynah_hip_qwen3_verify, mynah_hip_qwen3_accept).
//
// SPDX-License-Identifier: MIT
#pragma once
#include "common.hip.h"

// The greedy choice of each row of logits (argmax_key's order). Grid (rows),
// block 1024: a row of n floats is read once, four values a thread at a time;
// n a multiple of 4. Bound by the latency of one workgroup's loads, little next to
// the head that made the rows.
extern "C" __global__ void __launch_bounds__(1024)
mynah_argmax_rows(const float *__restrict__ x, uint32_t n, uint32_t *__restrict__ ids) {
    __shared__ unsigned long long best[16];
    const float4 *row = (const float4 *)(x + (size_t)blockIdx.x * n);
    unsigned long long key = 0ull;
    for (uint32_t i = threadIdx.x; i < n / 4u; i += 1024u) {
        const float4 v = row[i];
        const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned long long k = argmax_key(f[j], 4u * i + j);
            key = k > key ? k : key;
        }
    }
    key = wave_max_u64(key);
    if ((threadIdx.x & 63u) == 0u) best[threadIdx.x >> 6] = key;
    __syncthreads();
    if (threadIdx.x != 0u) return;
    for (int w = 1; w < 16; w++) key = best[w] > key ? best[w] : key;
    ids[blockIdx.x] = ~(uint32_t)key;
}

// Rows base + path[i] of every layer's keys and values to rows base + i, i < n,
// path rising: a thread moves its own four columns in order, so a row is read
// before a later one takes its place. Grid (ceil(kv_dim / 256), layers, 2 for keys
// and values), block 64.
extern "C" __global__ void __launch_bounds__(64)
mynah_kv_compact(float *__restrict__ k, float *__restrict__ v, const int32_t *__restrict__ path,
                 uint32_t n, uint32_t base, uint32_t kv_dim, size_t per_layer) {
    const uint32_t col = (blockIdx.x * 64u + threadIdx.x) * 4u;
    if (col >= kv_dim) return;
    float *c = (blockIdx.z ? v : k) + blockIdx.y * per_layer + (size_t)base * kv_dim + col;
    for (uint32_t i = 0; i < n; i++) {
        const uint32_t from = (uint32_t)path[i];
        if (from != i)
            *(float4 *)(c + (size_t)i * kv_dim) = *(const float4 *)(c + (size_t)from * kv_dim);
    }
}
