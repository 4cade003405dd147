// fp8.hip — products in 8-bit floating point (e4m3, no infinities, largest
// value 448) with one f32 scale for each 128 values of an activation row and
// each 128 x 128 block of the weights (include/kernels_hip.h):
//   y[t][r] = sum_b xs[t][b] ws[r / 128][b] sum_{k in block b} xq[t][k] w[r][k]
// The inner sum of a block starts from zero on the matrix cores; the two scales
// multiply it in f32 as it joins the running sum.
//
// SPDX-License-Identifier: MIT
#pragma once
#include "common.hip.h"
#include "elem.hip.h"

#define FP8_B 128u

typedef int fp8_v8i __attribute__((ext_vector_type(8)));
typedef float fp8_v4f __attribute__((ext_vector_type(4)));

// ── activations to e4m3 ────────────────────────────────────────────────────
// Per block: amax = max(max |x|, 2^-100), xs = amax * f32(1 / 448), xq = e4m3(x *
// (448 * (1 / amax))), each operation rounded to f32, e4m3 to nearest, ties to
// even. 16 lanes a block, 8 values a lane; a NaN
// stays NaN, an infinity makes its block's scale infinite (and its product
// NaN). What bounds it: HBM (or the launch, for few tokens).
template <class T>
MYNAH_DEV void fp8_quantize(const T *x, size_t x_stride, uint32_t cols, uint32_t nb,
                            unsigned long long blocks, uint8_t *xq, float *xs) {
    const unsigned long long unit = (unsigned long long)blockIdx.x * 16u + (threadIdx.x >> 4);
    if (unit >= blocks) return;                  // whole 16-lane groups
    const unsigned long long t = unit / nb;
    const uint32_t b = (uint32_t)(unit - t * nb), l = threadIdx.x & 15u;
    const uint32_t e = b * FP8_B + 8u * l;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (e < cols) {                              // cols is a multiple of 16
        load4<true>(x + t * x_stride + e, v);
        load4<true>(x + t * x_stride + e + 4u, v + 4);
    }
    float m = 7.888609052210118e-31f;            // 2^-100
#pragma unroll
    for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[i]));
    m = fmaxf(m, dpp_f<0xB1>(m));
    m = fmaxf(m, dpp_f<0x4E>(m));
    m = fmaxf(m, dpp_f<0x124>(m));
    m = fmaxf(m, dpp_f<0x128>(m));
    const float inv = 448.0f * (1.0f / m);
    if (e < cols) {
        uint2 q;
        int w = 0;
        w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
        q.x = (uint32_t)w;
        w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, w, true);
        q.y = (uint32_t)w;
        *(uint2 *)(xq + t * cols + e) = q;
    }
    if (l == 0) xs[unit] = m * (1.0f / 448.0f);
}

#define FP8_QUANT_KERNEL(name, T)                                                            \
    extern "C" __global__ void __launch_bounds__(256) mynah_fp8_quantize_##name(             \
        const T *x, size_t x_stride, uint32_t cols, uint32_t nb, unsigned long long blocks,  \
        uint8_t *xq, float *xs) {                                                            \
        fp8_quantize<T>(x, x_stride, cols, nb, blocks, xq, xs);                              \
    }
FP8_QUANT_KERNEL(f32, float)
FP8_QUANT_KERNEL(f16, _Float16)
FP8_QUANT_KERNEL(bf16, __bf16)

// ── few tokens: the weights streamed once ─────────────────────────────────
// A workgroup of four waves holds 16 weight rows x 16 NT tokens and splits the
// blocks of the rows over its waves, whose sums meet in LDS (wave order, so the
// same bits every time). Weight rows are the MFMA's rows, tokens its columns:
// lane l gets of row (token) l % 16 the 16 bytes at 16 (l / 16) and at 64 + 16
// (l / 16) of a block, the same places of both operands, so each load of a wave
// takes 64 contiguous bytes of 16 rows, straight into the operand's registers;
// its results are token l % 16, rows 4 (l / 16) + 0..3.
// What bounds it: HBM, the weights being read once.
struct Fp8Chunk { uint4 lo, hi; };
MYNAH_DEV Fp8Chunk fp8_chunk(const uint8_t *row, uint32_t k) {
    return Fp8Chunk{*(const uint4 *)(row + k), *(const uint4 *)(row + k + 64u)};
}
// A last block's, at columns k + lane and k + lane + 64 of a row that starts
// `lane` bytes before `row`: zeros past its end.
MYNAH_DEV Fp8Chunk fp8_chunk_tail(const uint8_t *row, uint32_t k, uint32_t lane, uint32_t cols) {
    Fp8Chunk c = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (k + lane < cols) c.lo = *(const uint4 *)(row + k);
    if (k + lane + 64u < cols) c.hi = *(const uint4 *)(row + k + 64u);
    return c;
}

// e4m3 values as bf16, which holds each exactly: eight of them.
typedef __bf16 fp8_v8b __attribute__((ext_vector_type(8)));
MYNAH_DEV fp8_v8b fp8_wide(uint32_t x, uint32_t y) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.0f, false);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.0f, true);
    return fp8_v8b{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// A block's inner sums with f32 accumulation: v_mfma_f32_16x16x32_bf16 of the
// values as bf16 (against 64 bits 9e-9 of the result over N(0, 1) blocks; the
// 8-bit instructions align their products to the largest first: 1.5e-5, half
// an f16 rounding's 32nd part but 200 of f32's).
MYNAH_DEV fp8_v4f fp8_block_exact(const Fp8Chunk &a, const Fp8Chunk &x) {
    fp8_v4f c = {0.0f, 0.0f, 0.0f, 0.0f};
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_wide(a.lo.x, a.lo.y),
                                                fp8_wide(x.lo.x, x.lo.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_wide(a.lo.z, a.lo.w),
                                                fp8_wide(x.lo.z, x.lo.w), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_wide(a.hi.x, a.hi.y),
                                                fp8_wide(x.hi.x, x.hi.y), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_wide(a.hi.z, a.hi.w),
                                                   fp8_wide(x.hi.z, x.hi.w), c, 0, 0, 0);
}

template <int NT, class T>
MYNAH_DEV void fp8_few(const uint8_t *w, const float *ws, const uint8_t *xq, const float *xs,
                       T *y, uint32_t rows, uint32_t cols, uint32_t tokens, uint32_t nb) {
    __shared__ __attribute__((aligned(16))) float part[4][NT][64][4];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u, lm = lane & 15u, lk = lane >> 4;
    const uint32_t r0 = blockIdx.x * 16u, t0 = blockIdx.y * (16u * NT);
    const uint8_t *wr = w + (size_t)(r0 + lm < rows ? r0 + lm : rows - 1u) * cols + 16u * lk;
    const float *wsr = ws + (size_t)(r0 / FP8_B) * nb;
    const uint8_t *xr[NT];
    const float *xsr[NT];
    fp8_v4f acc[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t t = t0 + 16u * n + lm < tokens ? t0 + 16u * n + lm : tokens - 1u;
        xr[n] = xq + (size_t)t * cols + 16u * lk;
        xsr[n] = xs + (size_t)t * nb;
        acc[n] = fp8_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    auto join = [&](uint32_t b, const Fp8Chunk &a, const Fp8Chunk (&x)[NT]) {
        const float sw = wsr[b];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float s = sw * xsr[n][b];
            const fp8_v4f c = fp8_block_exact(a, x[n]);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[n][i] = fmaf(s, c[i], acc[n][i]);
        }
    };
    const uint32_t full = cols / FP8_B;
    for (uint32_t b = wave; b < full; b += 4u) {
        const Fp8Chunk a = fp8_chunk(wr, b * FP8_B);
        Fp8Chunk x[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) x[n] = fp8_chunk(xr[n], b * FP8_B);
        join(b, a, x);
    }
    if (full < nb && (full & 3u) == wave) {
        const uint32_t k = full * FP8_B;
        const Fp8Chunk a = fp8_chunk_tail(wr, k, 16u * lk, cols);
        Fp8Chunk x[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) x[n] = fp8_chunk_tail(xr[n], k, 16u * lk, cols);
        join(full, a, x);
    }
#pragma unroll
    for (int n = 0; n < NT; n++) *(fp8_v4f *)part[wave][n][lane] = acc[n];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 256u * NT; i += 256u) {
        const uint32_t n = i >> 8, tk = (i >> 4) & 15u, rr = i & 15u;
        const uint32_t l = (rr >> 2) * 16u + tk, e = rr & 3u;
        const float v = ((part[0][n][l][e] + part[1][n][l][e]) + part[2][n][l][e]) +
                        part[3][n][l][e];
        const uint32_t t = t0 + 16u * n + tk;
        if (t < tokens && r0 + rr < rows) y[(size_t)t * rows + r0 + rr] = (T)v;
    }
}

#define FP8_FEW_KERNEL(nt, name, T)                                                          \
    extern "C" __global__ void __launch_bounds__(256) mynah_fp8_few##nt##_##name(            \
        const uint8_t *w, const float *ws, const uint8_t *xq, const float *xs, T *y,         \
        uint32_t rows, uint32_t cols, uint32_t tokens, uint32_t nb) {                        \
        fp8_few<nt, T>(w, ws, xq, xs, y, rows, cols, tokens, nb);                            \
    }
FP8_FEW_KERNEL(1, f32, float)
FP8_FEW_KERNEL(1, f16, _Float16)
FP8_FEW_KERNEL(1, bf16, __bf16)
FP8_FEW_KERNEL(2, f32, float)
FP8_FEW_KERNEL(2, f16, _Float16)
FP8_FEW_KERNEL(2, bf16, __bf16)
FP8_FEW_KERNEL(4, f32, float)
FP8_FEW_KERNEL(4, f16, _Float16)
FP8_FEW_KERNEL(4, bf16, __bf16)
