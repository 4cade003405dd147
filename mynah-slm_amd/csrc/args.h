/* args.h — what the host sides of the operators share: refusals, element
 * types, sizes that fit.
 *
 * SPDX-License-Identifier: MIT */
#ifndef MYNAH_ARGS_H
#define MYNAH_ARGS_H

#include "mynah_attention.h"
#include "runtime_internal.h"

static inline int refuse(const char *what) {
    mynah_set_error("%s", what);
    return -1;
}

static inline size_t elem_size(int type) {
    return type == MYNAH_F32 ? 4u : type == MYNAH_F16 || type == MYNAH_BF16 ? 2u : 0u;
}

static inline int type_index(int type) {
    return type == MYNAH_F32 ? 0 : type == MYNAH_F16 ? 1 : 2;
}

/* Whether `n` rows `stride` apart, of `len` elements each, fit the address
 * space in bytes. */
static inline int fits(size_t n, size_t stride, size_t len, size_t size) {
    return stride <= (SIZE_MAX / 4 / size) / n && len <= SIZE_MAX / 4 / size;
}

static inline uint32_t log2_of(uint32_t power) { return (uint32_t)__builtin_ctz(power); }
static inline int is_power(uint32_t n) { return n != 0 && (n & (n - 1)) == 0; }

#endif
