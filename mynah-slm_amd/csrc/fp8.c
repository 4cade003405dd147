/* fp8.c — host side of the 8-bit floating point product (fp8.hip,
 * include/kernels_hip.h): argument checks and the choice of a kernel.
 *
 * SPDX-License-Identifier: MIT */
#include "kernels_hip.h"
#include "mynah_attention.h"
#include "runtime_internal.h"

#include <stdlib.h>

#define BLOCK 128u

static int type_index(int type) {
    return type == MYNAH_F32 ? 0 : type == MYNAH_F16 ? 1 : type == MYNAH_BF16 ? 2 : -1;
}

static int check_shape(int type, size_t cols, size_t tokens) {
    if (type_index(type) < 0) {
        mynah_set_error("fp8: type %d is not f32, f16 or bf16", type);
        return -1;
    }
    if (cols == 0 || cols % 16 != 0 || cols > 0x7fffff00u || tokens == 0 ||
        tokens > 0x7fffffffu) {
        mynah_set_error("fp8: %zu columns, %zu tokens: columns a multiple of 16 and at least one "
                        "token are needed", cols, tokens);
        return -1;
    }
    return 0;
}

int mynah_hip_fp8_quantize_dev(int type, const void *x, size_t x_stride, size_t tokens,
                               size_t cols, uint8_t *xq, float *xs, void *stream) {
    if (x == NULL || xq == NULL || xs == NULL) {
        mynah_set_error("null argument");
        return -1;
    }
    if (check_shape(type, cols, tokens) != 0) return -1;
    const size_t size = type == MYNAH_F32 ? 4 : 2;
    if (x_stride < cols || x_stride > SIZE_MAX / 8 / tokens) {
        mynah_set_error("fp8: bad row stride");
        return -1;
    }
    if (((uintptr_t)x & 15u) != 0 || (x_stride * size) % 16 != 0 || ((uintptr_t)xq & 15u) != 0 ||
        ((uintptr_t)xs & 3u) != 0) {
        mynah_set_error("fp8: rows and quantised values must be 16-byte aligned");
        return -1;
    }
    uint32_t c32 = (uint32_t)cols, nb = (uint32_t)((cols + BLOCK - 1) / BLOCK);
    unsigned long long blocks = (unsigned long long)tokens * nb;
    if ((blocks + 15) / 16 > MYNAH_MOST_WGS(256)) {
        mynah_set_error("fp8: too many values for one launch");
        return -1;
    }
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    void *args[] = {&x, &x_stride, &c32, &nb, &blocks, &xq, &xs};
    return mynah_launch(d, MYNAH_K_FP8_QUANT + type_index(type), (unsigned)((blocks + 15) / 16), 1,
                        256, 0, mynah_stream_or_default(d, stream), args);
}

/* The tiled kernels, in the kernel ids' order: how many workgroups a CU holds, and
 * the microseconds of a step (a block of 128 columns) with one a CU and with all of
 * them, measured on MI355X as the slope from 10 to 40 blocks at 256 workgroups and at
 * 2,048 (bf16 outputs; f32 ones within 3 %). Two of the 4-wave 128 x 128 tile share a
 * CU (1.86 us for both); alone on it the 8-wave one is the faster (0.97 against 1.05
 * where 128 CUs have one). */
typedef struct {
    uint32_t rows, toks, waves, per_cu;
    float one, all;
} fp8_tile;
static const fp8_tile fp8_tiles[4] = {{64, 64, 4, 2, 0.43f, 0.69f},
                                      {64, 128, 4, 2, 0.66f, 1.14f},
                                      {128, 128, 4, 2, 1.06f, 1.86f},
                                      {128, 128, 8, 1, 1.05f, 1.05f}};

/* Microseconds of the streaming kernel for 17 to 64 tokens, launch and all: rounds
 * of 16 weight rows a CU, a step longer with every token. Up to 16 tokens it is
 * taken in any case. Measured against the fastest tile, bf16 out: 1024 x 2560, 17
 * tokens 4.9 for 11.2 us, 64 tokens 8.9 for 11.3; 4096 x 2560, 64 tokens 9.3 for 11.5;
 * 9728 x 2560, 16 tokens 9.5, 17 tokens 10.9 for 11.5, 24 tokens 12.4 for 11.6, 64 tokens
 * 22.3 for 11.8; 2560 x 9728, 64 tokens 27.3 for 34.6. */
static double fp8_few_us(size_t rows, size_t tokens, size_t cols, uint32_t cus) {
    const double rounds = (double)(((rows + 15) / 16 + cus - 1) / cus);
    return 2.4 + rounds * (double)((cols + BLOCK - 1) / BLOCK) * (0.085 + 0.0038 * (double)tokens);
}

/* The tile of least estimated time for a product, or NULL for the streaming
 * kernel: whole rounds of resident workgroups, then a last one. Four steps stand
 * for the start and the end of a workgroup, 1.5 us for the launch. The tiles address
 * their rows in 32 bits. MYNAH_FP8_TILE=0..3 forces one. */
static const fp8_tile *fp8_plan(size_t rows, size_t tokens, size_t cols, uint32_t cus) {
    if (tokens <= 16 || cols > (size_t)1 << 23) return NULL;
    const char *env = getenv("MYNAH_FP8_TILE");
    if (env != NULL && env[0] >= '0' && env[0] <= '3' && env[1] == '\0')
        return &fp8_tiles[env[0] - '0'];
    const fp8_tile *best = NULL;
    double best_us = 0.0;
    for (int i = 0; i < 4; i++) {
        const fp8_tile *t = &fp8_tiles[i];
        const uint64_t wgs = (uint64_t)((rows + t->rows - 1) / t->rows) *
                             (uint64_t)((tokens + t->toks - 1) / t->toks);
        const uint64_t slots = (uint64_t)cus * t->per_cu, left = wgs % slots;
        double us = (double)(wgs / slots) * t->all;
        if (left) us += left <= cus ? t->one : t->all;
        us *= (double)((cols + BLOCK - 1) / BLOCK + 4);
        if (best == NULL || us < best_us) {
            best = t;
            best_us = us;
        }
    }
    if (tokens <= 64 && fp8_few_us(rows, tokens, cols, cus) <= best_us + 1.5) return NULL;
    return best;
}

int mynah_hip_fp8_matmat_dev(const uint8_t *w, const float *ws, size_t rows, size_t cols,
                             const uint8_t *xq, const float *xs, int type, void *y,
                             size_t tokens, void *stream) {
    if (w == NULL || ws == NULL || xq == NULL || xs == NULL || y == NULL) {
        mynah_set_error("null argument");
        return -1;
    }
    if (check_shape(type, cols, tokens) != 0) return -1;
    if (rows == 0 || (rows + 15) / 16 > MYNAH_MOST_WGS(256) || tokens > SIZE_MAX / 8 / rows) {
        mynah_set_error("fp8: bad row count");
        return -1;
    }
    const size_t size = type == MYNAH_F32 ? 4 : 2;
    if (((uintptr_t)w & 15u) != 0 || ((uintptr_t)xq & 15u) != 0 || ((uintptr_t)ws & 3u) != 0 ||
        ((uintptr_t)xs & 3u) != 0 || (uintptr_t)y % size != 0) {
        mynah_set_error("fp8: 8-bit operands must be 16-byte aligned, the others to their size");
        return -1;
    }
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    uint32_t r32 = (uint32_t)rows, c32 = (uint32_t)cols, t32 = (uint32_t)tokens,
             nb = (uint32_t)((cols + BLOCK - 1) / BLOCK);
    hipStream_t st = mynah_stream_or_default(d, stream);
    const int t = type_index(type);
    const fp8_tile *tl = fp8_plan(rows, tokens, cols, (uint32_t)d->cus);
    if (tl != NULL) {
        uint32_t tr = (uint32_t)((rows + tl->rows - 1) / tl->rows);
        const uint64_t wgs = (uint64_t)tr * ((tokens + tl->toks - 1) / tl->toks);
        if (wgs <= MYNAH_MOST_WGS(64 * tl->waves)) {
            void *args[] = {&w, &ws, &xq, &xs, &y, &r32, &c32, &t32, &nb, &tr};
            return mynah_launch(d, MYNAH_K_FP8_TILE + 3 * (int)(tl - fp8_tiles) + t, (unsigned)wgs, 1,
                                64 * tl->waves, 0, st, args);
        }
    }
    void *args[] = {&w, &ws, &xq, &xs, &y, &r32, &c32, &t32, &nb};
    const int v = tokens <= 16 ? 0 : tokens <= 32 ? 1 : 2;
    const uint32_t per = 16u << v;
    const size_t tiles = (tokens + per - 1) / per;
    if (tiles > 65535) {
        mynah_set_error("fp8: too many tokens for one launch");
        return -1;
    }
    return mynah_launch(d, MYNAH_K_FP8_FEW1 + 3 * v + t, (unsigned)((rows + 15) / 16),
                        (unsigned)tiles, 256, 0, st, args);
}
