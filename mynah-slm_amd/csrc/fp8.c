/* fp8.c — host side of the 8-bit floating point product (fp8.hip,
 * include/kernels_hip.h): argument checks and the choice of a kernel.
 *
 * SPDX-License-Identifier: MIT */
#include "kernels_hip.h"
#include "mynah_attention.h"
#include "runtime_internal.h"

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
    if ((blocks + 15) / 16 > 0x7fffffffu) {
        mynah_set_error("fp8: too many values for one launch");
        return -1;
    }
    mynah_device *d = mynah_dev();
    if (d == NULL) return -1;
    void *args[] = {&x, &x_stride, &c32, &nb, &blocks, &xq, &xs};
    return mynah_launch(d, MYNAH_K_FP8_QUANT + type_index(type), (unsigned)((blocks + 15) / 16), 1,
                        256, 0, mynah_stream_or_default(d, stream), args);
}

int mynah_hip_fp8_matmat_dev(const uint8_t *w, const float *ws, size_t rows, size_t cols,
                             const uint8_t *xq, const float *xs, int type, void *y,
                             size_t tokens, void *stream) {
    if (w == NULL || ws == NULL || xq == NULL || xs == NULL || y == NULL) {
        mynah_set_error("null argument");
        return -1;
    }
    if (check_shape(type, cols, tokens) != 0) return -1;
    if (rows == 0 || rows > 0x7fffff00u || tokens > SIZE_MAX / 8 / rows) {
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
    void *args[] = {&w, &ws, &xq, &xs, &y, &r32, &c32, &t32, &nb};
    const int v = tokens <= 16 ? 0 : tokens <= 32 ? 1 : 2;
    const uint32_t per = 16u << v;
    const size_t tiles = (tokens + per - 1) / per;
    if (tiles > 65535) {
        mynah_set_error("fp8: too many tokens for one launch");
        return -1;
    }
    return mynah_launch(d, MYNAH_K_FP8_FEW1 + 3 * v + type_index(type),
                        (unsigned)((rows + 15) / 16), (unsigned)tiles, 256, 0, st, args);
}
