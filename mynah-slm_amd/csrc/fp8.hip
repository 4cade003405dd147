// fp8.hip — products in 8-bit floating point (e4m3, no infinities, largest
// value 448) with one f32 scale for each 128 values of an activation row and
// each 128 x 128 block of the weights (include/kernels_hip.h):
//   y[t][r] = sum_b xs[t][b] ws[r / 128][b] sum_{k in block b} xq[t][k] w[r][k]
// The inner sum of a block starts from zero on the matrix cores, in f32; the two
// scales multiply it in f32 as it joins the running sum.
//
// SPDX-License-Identifier: MIT
#pragma once
#include "common.hip.h"
#include "elem.hip.h"

#define FP8_B 128u

typedef float fp8_v4f __attribute__((ext_vector_type(4)));

// ── activations to e4m3 ────────────────────────────────────────────────────
// Per block: amax = max(max |x|, 2^-100), xs = amax * f32(1 / 448), xq = e4m3(x *
// (448 * (1 / amax))), each operation rounded to f32, e4m3 to nearest, ties to
// even. 16 lanes a block, 8 values a lane; a NaN
// stays NaN, an infinity makes its block's scale infinite (and its product
// NaN). What bounds it: HBM, or the launch for few tokens (37 x 2560 bf16: 2.4 us).
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
// What bounds it: HBM, the weights being read once (9728 x 2560, one token, f32 out:
// 6.4 us a call, 3.9 TB/s), and for more tokens the loads of few workgroups (4096 x
// 2560, 37 tokens, bf16 out: 256 of them, 8.0 us).
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
// A block's inner sums in f32: v_mfma_f32_16x16x32_bf16 of the values as bf16
// (against 64 bits 9e-9 of the result over N(0, 1) blocks). The 8-bit matrix
// instructions have up to twice the rate and hold less: of each eight products they
// cut every one to a multiple of the largest one's power of two times 2^-13 to
// 2^-14 (448 x 448 and its negative leave nothing of six products of 4 beside them).
// What that costs: 9728 x 2560, 8192 tokens, bf16 out 383 us (1.07 PFLOP/s, where a
// large bf16 library product reaches 1.2), 201 us with the 8-bit instructions.
MYNAH_DEV fp8_v4f fp8_block(const Fp8Chunk &a, const Fp8Chunk &x) {
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
            const fp8_v4f c = fp8_block(a, x[n]);
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
    extern "C" __global__ void __launch_bounds__(256, 2) mynah_fp8_few##nt##_##name(            \
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

// ── many tokens: tiles through LDS ────────────────────────────────────────
// A workgroup of WR x WT waves takes 16 MT WR weight rows x 16 NT WT tokens; each
// step it copies one block (128 columns) of its rows and tokens, and their
// scales, straight from memory into LDS, ST buffers, so that ST - 1 steps'
// copies are in flight while one is summed; one barrier a step. Weight rows are
// the MFMA's rows, so a lane holds four rows of one token and its two scales are
// one factor a tile.
// A row's 16-byte chunk c lies at place c ^ (row % 8), so that the copies read
// whole rows and the operand reads (16 rows, one chunk) meet no bank twice. The
// buffers are LDS objects of their own: of one object the compiler makes every
// operand read wait for the newest copy.
typedef __attribute__((address_space(3))) void fp8_lds_void;

template <int WR, int WT, int MT, int NT> struct Fp8Tile {
    static constexpr int NW = WR * WT, ROWS = 16 * MT * WR, TOK = 16 * NT * WT;
    static constexpr int COPIES = (ROWS + TOK) / 8 / NW;   // of a wave, 1 KiB each
    static constexpr int XS = (ROWS + TOK) * 128;          // tokens' scales, then rows'
    static constexpr int WS = XS + 256 * NW, BYTES = WS + 256 * NW;
};

// s_waitcnt vmcnt(N), and a barrier that no memory access crosses (the fences of
// one wave's scope cost nothing; __syncthreads would wait for every copy).
template <int N> MYNAH_DEV void fp8_wait() {
    __builtin_amdgcn_s_waitcnt((N & 15) | 0x70 | 0xf00 | ((N >> 4) << 14));
}
MYNAH_DEV void fp8_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_sched_barrier(0);
}

template <int WR, int WT, int MT, int NT, int ST, class T>
MYNAH_DEV void fp8_tile(const uint8_t *w, const float *ws, const uint8_t *xq, const float *xs,
                        T *y, uint32_t rows, uint32_t cols, uint32_t tokens, uint32_t nb,
                        uint32_t tiles_r) {
    using P = Fp8Tile<WR, WT, MT, NT>;
    static_assert((P::ROWS / 8) % P::NW == 0 && (P::TOK / 8) % P::NW == 0 &&
                      P::TOK <= 64 * P::NW && P::TOK / P::NW % 16 == 0 &&
                      16 * NT % (P::TOK / P::NW) == 0, "copies");
    __shared__ __attribute__((aligned(16))) uint8_t s0[P::BYTES], s1[P::BYTES];
    __shared__ __attribute__((aligned(16))) uint8_t s2[ST > 2 ? P::BYTES : 16];
    __shared__ __attribute__((aligned(16))) uint8_t s3[ST > 3 ? P::BYTES : 16];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u, lm = lane & 15u, lk = lane >> 4;
    // Workgroups go to the 8 XCDs in turn: each XCD takes a run of tiles, in
    // columns of four token tiles, so that what runs on it at one time shares
    // rows and tokens in its L2 (9728 x 2560, 8192 tokens: 400 -> 383 us against
    // runs of one token tile).
    uint32_t id = blockIdx.x;
    const uint32_t whole = gridDim.x & ~7u;
    if (id < whole) id = (id & 7u) * (whole >> 3) + (id >> 3);
    const uint32_t tiles_t = gridDim.x / tiles_r, g0 = id / (4u * tiles_r) * 4u;
    const uint32_t gs = tiles_t - g0 < 4u ? tiles_t - g0 : 4u, in = id - g0 * tiles_r;
    const uint32_t R0 = (in / gs) * P::ROWS, T0 = (g0 + in % gs) * P::TOK;
    const uint32_t r0 = 16u * MT * (wave % WR), t0 = 16u * NT * (wave / WR);

    // Buffers end with their matrix (or where 32 bits do): a copy from NONE on is
    // out of range, reads nothing and leaves zeros.
    constexpr uint32_t NONE = 0xfffffff0u;
    uint32_t at[P::COPIES];
    const uint32_t chunk = (lane & 7u) ^ (lane >> 3), rmost = rows - 1u - R0,
                   tmost = tokens - 1u - T0;
    constexpr int WC = P::COPIES * P::ROWS / (P::ROWS + P::TOK);   // of them weights
#pragma unroll
    for (int i = 0; i < P::COPIES; i++) {
        const uint32_t r = 8u * (P::NW * i + wave) + (lane >> 3);
        const uint32_t q = i < WC ? r : r - P::ROWS, most = i < WC ? rmost : tmost;
        at[i] = (q < most ? q : most) * cols + 16u * chunk;
    }
    // A wave's share of the tokens' scales: its first TOK / NW lanes.
    constexpr uint32_t SHARE = P::TOK / P::NW;
    const uint32_t ts = SHARE * wave + lane;
    const uint32_t xat = lane < SHARE ? (ts < tmost ? ts : tmost) * nb * 4u : NONE;
    const uint32_t wat = ((R0 + (r0 < rmost ? r0 : rmost)) / FP8_B - R0 / FP8_B) * nb * 4u;
    auto rsrc = [](const void *p, size_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0,
                                                 bytes < NONE ? (uint32_t)bytes : NONE, 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t rw = rsrc(w + (size_t)R0 * cols, (size_t)(rows - R0) * cols),
                                 rx = rsrc(xq + (size_t)T0 * cols, (size_t)(tokens - T0) * cols),
                                 rxs = rsrc(xs + (size_t)T0 * nb, (size_t)(tokens - T0) * nb * 4),
                                 rws = rsrc(ws + (size_t)(R0 / FP8_B) * nb,
                                            (size_t)((rows - 1u) / FP8_B - R0 / FP8_B + 1u) * nb *
                                                4);
    constexpr int OPS = P::COPIES + 2;           // VMEM operations of a wave's step
    auto copy = [&](uint32_t b, uint8_t *p) {
        const uint32_t off = b * FP8_B + 16u * chunk < cols ? 0u : NONE;
        const uint32_t soff = b < nb ? 0u : NONE;
        // The range check compares an offset with the buffer's size less the block's
        // place, which past the last block would be below zero.
        const uint32_t place = b < nb ? b : 0u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rxs, (fp8_lds_void *)(p + P::XS + 256u * wave),
                                                 4, xat | soff, 4u * place, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rws, (fp8_lds_void *)(p + P::WS + 256u * wave),
                                                 4, wat | soff, 4u * place, 0, 0);
#pragma unroll
        for (int i = 0; i < P::COPIES; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                i < WC ? rw : rx, (fp8_lds_void *)(p + 1024u * (P::NW * i + wave)), 16,
                at[i] | off, FP8_B * place, 0, 0);
    };
    const uint32_t a0 = (r0 + lm) * FP8_B + 16u * (lk ^ (lm & 7u));
    const uint32_t b0 = (P::ROWS + t0 + lm) * FP8_B + 16u * (lk ^ (lm & 7u));

    fp8_v4f acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) acc[m][n] = fp8_v4f{0.0f, 0.0f, 0.0f, 0.0f};

    auto step = [&](const uint8_t *p) {
        auto operand = [&](uint32_t o) {
            return Fp8Chunk{*(const uint4 *)(p + o), *(const uint4 *)(p + (o ^ 64u))};
        };
        const float scale = *(const float *)(p + P::WS + 256u * wave);
        const uint8_t *sp = p + P::XS + 256u * (t0 / SHARE) + 4u * lm;
        Fp8Chunk a[MT], x[2];
#pragma unroll
        for (int m = 0; m < MT; m++) a[m] = operand(a0 + 2048u * m);
        x[0] = operand(b0);
        // A token tile's sums join, and the next one's operand is read, while
        // its products run.
        fp8_v4f c[2][MT];
        float f[2];
#pragma unroll
        for (int n = 0; n <= NT; n++) {
            if (n < NT) {
                if (n + 1 < NT) x[(n + 1) & 1] = operand(b0 + 2048u * (n + 1));
                f[n & 1] = scale * *(const float *)(sp + 256u * (16u * n / SHARE) +
                                                    4u * (16u * n % SHARE));
#pragma unroll
                for (int m = 0; m < MT; m++) c[n & 1][m] = fp8_block(a[m], x[n & 1]);
            }
            if (n > 0) {
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        acc[m][n - 1][i] =
                            fmaf(f[(n - 1) & 1], c[(n - 1) & 1][m][i], acc[m][n - 1][i]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Block b, in buffer `now`: its copies have landed (those of the ST - 2 blocks
    // after it may be under way), everybody is done with the buffer before it,
    // `old`, which takes block b + ST - 1's. Copies and waits stand under no
    // condition (past the last block the copies read nothing): over a branch the
    // compiler loses count of them and waits for all.
    auto turn = [&](uint32_t b, uint8_t *old, const uint8_t *now) {
        fp8_wait<(ST - 2) * OPS>();
        fp8_barrier();
        copy(b + ST - 1u, old);
        __builtin_amdgcn_sched_barrier(0);
        step(now);
    };
    copy(0u, s0);
    if constexpr (ST > 2) copy(1u, s1);
    if constexpr (ST > 3) copy(2u, s2);
    // Turns of s0, s1, ... ST at a time, then those left (a loop that could end
    // between them keeps a copy of the sums for each end).
    auto first = [&](uint32_t b) {
        if constexpr (ST == 2) turn(b, s1, s0);
        else if constexpr (ST == 3) turn(b, s2, s0);
        else turn(b, s3, s0);
    };
    uint32_t b = 0;
    for (; b + ST <= nb; b += ST) {
        first(b);
        turn(b + 1u, s0, s1);
        if constexpr (ST > 2) turn(b + 2u, s1, s2);
        if constexpr (ST > 3) turn(b + 3u, s2, s3);
    }
    if (b < nb) {
        first(b);
        if constexpr (ST > 2) {
            if (b + 1u < nb) turn(b + 1u, s0, s1);
        }
        if constexpr (ST > 3) {
            if (b + 2u < nb) turn(b + 2u, s1, s2);
        }
    }
    fp8_wait<0>();                               // no copy outlives the workgroup
    // Out through LDS, a wave its own part, so that stores are whole runs of a
    // token's rows: 16-byte chunk c of token t at place c ^ (t % CH).
    constexpr int ROW = 16 * MT * (int)sizeof(T), CH = ROW / 16, E = 16 / (int)sizeof(T);
    constexpr int PART = 16 * NT * ROW, FIT = P::BYTES / PART;
    static_assert(FIT * ST >= P::NW, "the tile's results fit the buffers");
    fp8_barrier();
    uint8_t *o;
    if (wave < FIT) o = s0 + PART * wave;
    else if (wave < 2 * FIT) o = s1 + PART * (wave - FIT);
    else if (wave < 3 * FIT) o = s2 + PART * (wave - 2 * FIT);
    else o = s3 + PART * (wave - 3 * FIT);
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const uint32_t t = 16u * n + lm, e = 16u * m + 4u * lk;
            const uint32_t c = (e / E) ^ (t & (CH - 1u));
            const float v[4] = {acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]};
            store4<true>((T *)(o + t * ROW + 16u * c) + e % E, v);
        }
    const bool wide = rows % E == 0 && ((uintptr_t)y & 15u) == 0;
#pragma unroll 4
    for (uint32_t i = lane; i < 16u * NT * CH; i += 64u) {
        const uint32_t t = i / CH, c = i % CH, r = R0 + r0 + E * c;
        if (T0 + t0 + t >= tokens || r >= rows) continue;
        const uint4 x = *(const uint4 *)(o + t * ROW + 16u * (c ^ (t & (CH - 1u))));
        T *yo = y + (size_t)(T0 + t0 + t) * rows + r;
        if (wide) {
            *(uint4 *)yo = x;
        } else {
            T v[E];
            __builtin_memcpy(v, &x, 16);
#pragma unroll
            for (int k = 0; k < E; k++)
                if (r + k < rows) yo[k] = v[k];
        }
    }
}

#define FP8_TILE_KERNEL(tile, WR, WT, MT, NT, ST, W, name, T)                                   \
    extern "C" __global__ void __launch_bounds__(64 * WR * WT, W) mynah_fp8_##tile##_##name( \
        const uint8_t *w, const float *ws, const uint8_t *xq, const float *xs, T *y,         \
        uint32_t rows, uint32_t cols, uint32_t tokens, uint32_t nb, uint32_t tiles_r) {      \
        fp8_tile<WR, WT, MT, NT, ST, T>(w, ws, xq, xs, y, rows, cols, tokens, nb, tiles_r);  \
    }
#define FP8_TILE_KERNELS(tile, WR, WT, MT, NT, ST, W)            \
    FP8_TILE_KERNEL(tile, WR, WT, MT, NT, ST, W, f32, float)       \
    FP8_TILE_KERNEL(tile, WR, WT, MT, NT, ST, W, f16, _Float16)    \
    FP8_TILE_KERNEL(tile, WR, WT, MT, NT, ST, W, bf16, __bf16)
FP8_TILE_KERNELS(64x64, 2, 2, 2, 2, 4, 2)
FP8_TILE_KERNELS(64x128, 2, 2, 2, 4, 3, 2)
FP8_TILE_KERNELS(128x128, 2, 2, 4, 4, 2, 2)
FP8_TILE_KERNELS(128x128w, 4, 2, 2, 4, 4, 2)
