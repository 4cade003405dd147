// rope.hip — rotary positions, and the norms of query and key heads with the
// rotation and the cache store in the same pass (include/mynah_attention.h).
//
// SPDX-License-Identifier: MIT
#pragma once
#include "common.hip.h"
#include "elem.hip.h"

// One row set of a launch: heads of `in` (strides in elements) to `out`, whose
// row is the token's, or its slot's where slotted. Host mirror: mynah_rope_seg
// (runtime_internal.h).
struct RopeSeg {
    const void *in;
    void *out;
    size_t in_token, in_head, out_token, out_head;
    const float *norm;
    uint32_t heads, rotate, slotted, pad;
};
struct RopeArgs {
    RopeSeg seg[3];
    const double *freqs;
    const int32_t *pos, *slots;
    unsigned long long units;       // tokens * groups
    uint32_t n_slots, hd, rot, lanes_log2, groups, heads;
    float eps, mscale;
};

// cos and sin of the angle p * f, scaled. The product and its reduction to an
// eighth of a turn either side of a quarter are in double (a position of 2^31
// keeps its angle to 2^-22 radians), the rest in f32: with |x| <= pi / 4 the
// Taylor sums below end within 2e-9 (sin, next term x^11 / 11!) and 1.2e-10 (cos,
// x^12 / 12!) of the functions, under their f32 rounding.
MYNAH_DEV void turn(double p, double f, float mscale, float &c, float &s) {
    const double rev = p * f * 0.15915494309189535;       // 1 / (2 pi)
    const double r = rev - __builtin_rint(rev);
    const double q = __builtin_rint(4.0 * r);
    const float x = (float)(__builtin_fma(-0.25, q, r) * 6.283185307179586);
    const float z = x * x;
    float sn = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    sn = fmaf(z, sn, 8.3333333e-3f);
    sn = fmaf(z, sn, -1.6666667e-1f);
    sn = fmaf(x * z, sn, x);
    float cs = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    cs = fmaf(z, cs, -1.3888889e-3f);
    cs = fmaf(z, cs, 4.1666667e-2f);
    cs = fmaf(z, cs, -0.5f);
    cs = fmaf(z, cs, 1.0f);
    const int k = (int)q;
    const float a = (k & 1) ? sn : cs, b = (k & 1) ? cs : sn;
    c = mscale * (k == 0 || k == -1 ? a : -a);
    s = mscale * (k == 0 || k == 1 ? b : -b);
}

// A head is 2^lanes_log2 lanes, lane l holding pairs 4 l .. 4 l + 3 as two runs
// of four values (inactive past head_dim / 8): with half pairs of the rotated
// part the runs start at 4 l and rot / 2 + 4 l, otherwise they are the eight
// values from 8 l on. A slot of lanes keeps one token's cos and sin over the
// heads g, g + groups, ... of its group.
// What bounds it: HBM on long inputs, the launch and one chain of dependent
// loads (position, frequency, row) on single tokens. Measured, MI355X: 8192 tokens of
// 32 heads of 128 bf16 (134 MB) 41 us, 3.3 TB/s (a copy of the size 26; 27 where
// the last-level cache holds them), 2047 tokens of 40 f32 heads with norms to bf16
// rows 18.2 us, one token 4 us. One head a lane took 46 us (an angle for each), rows
// loaded two or four ahead of their use 52.
template <class TI, class TO, bool HALF, bool VEC>
MYNAH_DEV void rope_rows(const RopeArgs &a) {
    const uint32_t ll = a.lanes_log2, l = threadIdx.x & ((1u << ll) - 1u);
    const unsigned long long unit =
        (unsigned long long)blockIdx.x * (blockDim.x >> ll) + (threadIdx.x >> ll);
    if (unit >= a.units) return;                 // whole slots, and no barrier below
    const unsigned long long t = unit / a.groups;
    const uint32_t g = (uint32_t)(unit - t * a.groups);
    const bool on = 8u * l < a.hd;
    const uint32_t half = a.rot >> 1;
    const bool turns = on && 4u * l < half;
    const uint32_t e0 = HALF && turns ? 4u * l : 8u * l;
    const uint32_t e1 = HALF && turns ? half + 4u * l : 8u * l + 4u;
    float c[4] = {1.0f, 1.0f, 1.0f, 1.0f}, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (turns) {
        const double p = a.pos ? (double)a.pos[t] : (double)t;
#pragma unroll
        for (int i = 0; i < 4; i++) turn(p, a.freqs[4u * l + i], a.mscale, c[i], s[i]);
    }
    long long slot = (long long)t;
    if (a.slots) slot = a.slots[t];
    const bool stored = slot >= 0 && slot < (long long)a.n_slots;
    for (uint32_t h = g; h < a.heads; h += a.groups) {
        uint32_t k = 0, hs = h;
        while (k < 2u && hs >= a.seg[k].heads) hs -= a.seg[k++].heads;
        const RopeSeg &sg = a.seg[k];
        if (sg.slotted && !stored) continue;
        const TI *x = (const TI *)sg.in + t * sg.in_token + hs * sg.in_head;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = 0.0f;
        if (on) {
            load4<VEC>(x + e0, v);
            load4<VEC>(x + e1, v + 4);
        }
        if (sg.norm) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(v[i], v[i], ss);
            for (uint32_t m = 1; m < (1u << ll); m <<= 1) ss += __shfl_xor(ss, m, 64);
            const float r = 1.0f / sqrtf(ss / (float)a.hd + a.eps);
            if (on) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[i] = v[i] * r * sg.norm[e0 + i];
                    v[4 + i] = v[4 + i] * r * sg.norm[e1 + i];
                }
            }
        }
        if (!on) continue;
        if (sg.rotate && turns) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float &x0 = HALF ? v[i] : v[2 * i], &x1 = HALF ? v[4 + i] : v[2 * i + 1];
                const float y0 = x0 * c[i] - x1 * s[i];
                x1 = x1 * c[i] + x0 * s[i];
                x0 = y0;
            }
        }
        TO *y = (TO *)sg.out + (sg.slotted ? (size_t)slot : (size_t)t) * sg.out_token +
                hs * sg.out_head;
        store4<VEC>(y + e0, v);
        store4<VEC>(y + e1, v + 4);
    }
}

#define ROPE_KERNEL(name, TI, TO)                                                       \
    extern "C" __global__ void __launch_bounds__(256) mynah_rope_##name(RopeArgs a,     \
                                                                        uint32_t mode) { \
        if (mode == 3u) rope_rows<TI, TO, true, true>(a);                               \
        else if (mode == 2u) rope_rows<TI, TO, true, false>(a);                         \
        else if (mode == 1u) rope_rows<TI, TO, false, true>(a);                         \
        else rope_rows<TI, TO, false, false>(a);                                        \
    }
ROPE_KERNEL(f32_f32, float, float)
ROPE_KERNEL(f32_f16, float, _Float16)
ROPE_KERNEL(f32_bf16, float, __bf16)
ROPE_KERNEL(f16_f32, _Float16, float)
ROPE_KERNEL(f16_f16, _Float16, _Float16)
ROPE_KERNEL(f16_bf16, _Float16, __bf16)
ROPE_KERNEL(bf16_f32, __bf16, float)
ROPE_KERNEL(bf16_f16, __bf16, _Float16)
ROPE_KERNEL(bf16_bf16, __bf16, __bf16)
