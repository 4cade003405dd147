"""An 8-bit cache with its calls, what they should leave, and how far off they
may be, for the operators' tests (include/mynah_cache.h)."""
from __future__ import annotations

import numpy as np

import elem_lib as E

U = E.U
I8, E4M3 = 0, 1
MOST = {I8: np.float32(127), E4M3: np.float32(448)}
LEAST = np.float32(2.0 ** -100)


def values(codes, f):
    return codes.view(np.int8).astype(np.float64) if f == I8 else E.E4M3[codes]


def scale_of(amax, f):
    """f32, as the operator's definition rounds it."""
    q = np.maximum(np.float32(amax), LEAST) / MOST[f]
    if f == I8:
        return q
    m, e = np.frexp(q)
    return np.ldexp(np.float32(1), np.where(m > 0.5, e, e - 1)).astype(np.float32)


def codes_of(x, inv, f):
    with np.errstate(over="ignore", invalid="ignore"):
        y = np.asarray(x, np.float32) * np.float32(inv)
    y = np.where(np.isnan(y), np.float32(0), np.clip(y, -MOST[f], MOST[f]))
    return np.rint(y).astype(np.int8).view(np.uint8) if f == I8 else E.to_e4m3(y)


class Kv8:
    """A ragged batch over a contiguous or paged 8-bit cache.

    lens: [(committed positions, new tokens)] of the sequences; mask "chain" (none
    given), "tree" (random ancestors) or an array [rows][words] of uint32."""

    def __init__(self, M, lens, heads, kvh, hd, t, f, block=16, page=0, mask="chain", seed=0,
                 extra_rows=0, max_nodes=None, max_kv=None, pad=0, scale=None):
        self.M, self.lens, self.heads, self.kvh, self.hd = M, lens, heads, kvh, hd
        self.t, self.f, self.block, self.page, self.pad = t, f, block, page, pad
        rng = self.rng = np.random.default_rng(seed)
        n = len(lens)
        self.past = np.array([p for p, _ in lens], np.int32)
        self.nodes = np.array([k for _, k in lens], np.int32)
        self.start = np.concatenate([[0], np.cumsum(self.nodes)]).astype(np.int32)
        self.rows = max(1, int(self.start[-1]) + extra_rows)
        self.max_nodes = max_nodes or max(1, int(self.nodes.max()))
        self.max_kv = max_kv or max(1, int((self.past + self.nodes).max()))
        self.words = -(-self.max_nodes // 32)
        if page:
            self.max_pages = -(-self.max_kv // page)
            self.slots = n * self.max_pages * page
            self.pages = rng.permutation(n * self.max_pages).astype(np.int32)
            self.pages = self.pages.reshape(n, self.max_pages)
            self.seq_slots = 0
        else:
            self.seq_slots = -(-self.max_kv // block) * block
            self.slots, self.pages, self.max_pages = n * self.seq_slots, None, 0
        self.ss = kvh * hd + pad
        self.xs = kvh * hd + pad
        self.qs = heads * hd + pad
        nb = self.slots // block
        self.k = rng.integers(0, 256, (self.slots, self.ss)).astype(np.uint8)
        self.v = rng.integers(0, 256, (self.slots, self.ss)).astype(np.uint8)
        if f == E4M3:
            for c in (self.k, self.v):
                c[(c & 127) == 127] = 5
        # Codes of any size: scales that make values of about 1.
        typical = 70.0 if f == I8 else 40.0
        self.ks, self.vs = (np.exp(0.6 * rng.standard_normal((2, nb, kvh))) / typical).astype(np.float32)
        if f == E4M3:
            self.ks, self.vs = (np.exp2(np.rint(np.log2(s))).astype(np.float32)
                                for s in (self.ks, self.vs))
        self.q = E.encode(0.7 * rng.standard_normal((self.rows, self.qs)), t)
        self.kx = E.encode(rng.standard_normal((self.rows, self.xs)), t)
        self.vx = E.encode(rng.standard_normal((self.rows, self.xs)), t)
        self.scale = hd ** -0.5 if scale is None else scale
        self.mask = None if isinstance(mask, str) else mask
        if isinstance(mask, str) and mask == "tree":
            self.mask = np.zeros((self.rows, self.words), np.uint32)
            for b in range(n):
                for i in range(self.nodes[b]):
                    row = self.start[b] + i
                    parent = int(rng.integers(-1, i)) if i else -1
                    if parent >= 0:
                        self.mask[row] = self.mask[self.start[b] + parent]
                    if i < 32 * self.words:
                        self.mask[row, i // 32] |= np.uint32(1 << (i % 32))
        self.d = None

    # ── calls ────────────────────────────────────────────────────────────────

    def upload(self):
        B = self.M.DeviceBuffer.from_array
        self.out0 = E.encode(np.full((self.rows, self.qs), 11.0), self.t)
        self.d = {n: B(getattr(self, n)) for n in ("q", "k", "v", "ks", "vs", "kx", "vx", "start",
                                                   "past")}
        self.d["out"] = B(self.out0)
        for n in ("pages", "mask"):
            if getattr(self, n) is not None:
                self.d[n] = B(getattr(self, n))

    def at(self, n):
        return self.d[n].ptr if n in self.d else None

    def cache(self):
        return self.M.Kv8Cache(
            format=self.f, n_kv_heads=self.kvh, head_dim=self.hd, block=self.block, k=self.at("k"),
            v=self.at("v"), slot_stride=self.ss, n_slots=self.slots, k_scale=self.at("ks"),
            v_scale=self.at("vs"), seq_slots=self.seq_slots, pages=self.at("pages"),
            page_size=self.page, max_pages=self.max_pages)

    def store_args(self, **change):
        v = dict(cache=self.cache(), type=self.t, n_seqs=len(self.lens), k=self.at("kx"),
                 v=self.at("vx"), k_stride=self.xs, v_stride=self.xs, n_rows=self.rows,
                 seq_start=self.at("start"), n_past=self.at("past"), max_nodes=self.max_nodes,
                 max_kv=self.max_kv)
        return self.M.Kv8Store(**{**v, **change})

    def attn_args(self, **change):
        v = dict(cache=self.cache(), type=self.t, n_seqs=len(self.lens), n_heads=self.heads,
                 q=self.at("q"), q_stride=self.qs, out=self.at("out"), out_stride=self.qs,
                 n_rows=self.rows, seq_start=self.at("start"), n_past=self.at("past"),
                 mask=self.at("mask"), mask_words=self.words, max_nodes=self.max_nodes,
                 max_kv=self.max_kv, scale=self.scale)
        return self.M.Kv8Attention(**{**v, **change})

    def store(self, stream=None, **change):
        self.upload()
        self.M.kv8_store_dev(self.store_args(**change), stream)
        self.M.check(self.M.lib.mynah_hip_sync(stream), "sync")
        return self.stored()

    def stored(self):
        return {n: self.d[n].download(getattr(self, n).dtype, getattr(self, n).size)
                .reshape(getattr(self, n).shape) for n in ("k", "v", "ks", "vs")}

    def attend(self, stream=None, **change):
        self.upload()
        a = self.attn_args(**change)
        n = self.M.kv8_attention_workspace(a)
        self.ws = self.M.DeviceBuffer.from_array(np.full(n, 0xFF, np.uint8))   # NaN, stale
        self.M.kv8_attention_dev(a, self.ws.ptr, n, stream)
        self.M.check(self.M.lib.mynah_hip_sync(stream), "sync")
        return self.raw()

    def raw(self):
        return self.d["out"].download(E.NP[self.t], self.q.size).reshape(self.q.shape)

    # ── what they should leave ───────────────────────────────────────────────

    def cache_rows(self, b, n):
        """Rows of positions 0 .. n - 1; -1 where there is none."""
        p = np.arange(n)
        if self.page:
            pg = self.pages[b, p // self.page].astype(np.int64)
            at = np.where(pg < 0, -1, pg * self.page + p % self.page)
        else:
            at = b * self.seq_slots + p
        return np.where(at < self.slots, at, -1)

    def expected_store(self):
        """The cache after the call: every byte of it."""
        out = {n: getattr(self, n).copy() for n in ("k", "v", "ks", "vs")}
        for b, (past, _) in enumerate(self.lens):
            past, nodes = max(past, 0), min(int(self.nodes[b]), self.max_nodes)
            end = min(past + nodes, self.max_kv)
            if end <= past:
                continue
            rows = self.cache_rows(b, end)
            for first in range(past // self.block * self.block, end, self.block):
                lo, hi = max(first, past), min(first + self.block, end)
                if rows[lo] < 0:
                    continue
                src = self.start[b] + np.arange(lo, hi) - past
                there = (src >= 0) & (src < self.rows)
                src, dst = src[there], rows[lo:hi][there]
                blk = rows[lo] // self.block
                for c, s, x in (("k", "ks", self.kx), ("v", "vs", self.vx)):
                    x = E.decode(x[src], self.t).astype(np.float32)[:, :self.kvh * self.hd]
                    x = x.reshape(-1, self.kvh, self.hd)
                    amax = np.where(np.isfinite(x), np.abs(x), 0).max((0, 2), initial=0)
                    new, old = scale_of(amax, self.f), out[s][blk].copy()
                    old = np.where((old > 0) & np.isfinite(old), old, np.float32(0))
                    if first < past:
                        new = np.maximum(new, old)
                        kept = rows[first:past]
                        was = out[c][kept][:, :self.kvh * self.hd].reshape(-1, self.kvh, self.hd)
                        again = codes_of(values(was, self.f), (old / new)[:, None], self.f)
                        again = np.where((old == new)[:, None], was, again)
                        out[c][kept, :self.kvh * self.hd] = again.reshape(len(kept), -1)
                    out[s][blk] = new
                    put = codes_of(x, (np.float32(1) / new)[:, None], self.f)
                    out[c][dst, :self.kvh * self.hd] = put.reshape(len(dst), -1)
        return out

    def check_store(self, got, what=""):
        want = self.expected_store()
        for n in ("ks", "vs"):
            assert np.array_equal(got[n], want[n], equal_nan=True), (what, n)
        for n in ("k", "v"):
            a, b = got[n].copy(), want[n].copy()
            if self.f == E4M3:                         # zeros of either sign
                a[a == 128], b[b == 128] = 0, 0
            assert np.array_equal(a, b), (what, n, np.argwhere(a != b)[:4].tolist())

    def expected(self):
        """(out [rows][heads][hd], bound, which rows are written). Per output, with A =
        sum p |v|. Codes are exact; a score is a sum of hd products in f32 (of f32
        queries 3 hd) and the exponent takes four more roundings of its size (scale,
        log2 e, the block's scale, the difference): off by at most d = (QN hd + 8) u scale
        |q| . |k| (its largest over the row), and exp follows: 2 d A + 6 u A. Sums over n
        positions, of PN products each, add PN n u A. A weight is one bf16 number of
        bf16 calls (a half step, 2^-8 A), two of f16 ones (2^-8 cut, then 2^-8: 2^-16
        A), three of f32 ones (exact). Below f32's (and bf16's) smallest normal number the
        exponential and the products hold nothing: a probability, or a part of a
        weight, under 2^-126 counts as 0, which takes n 2^-126 (largest |v| + PN largest
        |code|) at most (a column whose one large probability has the code 0)."""
        QN = 3 if self.t == E.F32 else 1
        PN = {E.F32: 3, E.F16: 2, E.BF16: 1}[self.t]
        cut = {E.F32: 0.0, E.F16: 2.0 ** -16, E.BF16: 2.0 ** -8}[self.t]
        out = np.zeros((self.rows, self.heads, self.hd))
        tol = np.zeros_like(out)
        live = np.zeros(self.rows, bool)
        group = self.heads // self.kvh

        def cache(c, s):
            s = np.where((s > 0) & np.isfinite(s), s, 0).astype(np.float64)
            x = values(c[:, :self.kvh * self.hd], self.f).reshape(-1, self.kvh, self.hd)
            return x * np.repeat(s, self.block, 0)[..., None]
        k, v = cache(self.k, self.ks), cache(self.v, self.vs)
        q = E.decode(self.q, self.t)[:, :self.heads * self.hd].reshape(-1, self.heads, self.hd)
        for b, (past, _) in enumerate(self.lens):
            nodes = min(int(self.nodes[b]), self.max_nodes)
            past = max(past, 0)
            n = min(past + nodes, self.max_kv)
            rows = slice(int(self.start[b]), int(self.start[b]) + nodes)
            live[rows] = True
            at = self.cache_rows(b, n)
            see = np.ones((nodes, n), bool)
            if n > past:
                j = np.arange(n - past)
                if self.mask is None:
                    see[:, past:] = j <= np.arange(nodes)[:, None]
                else:
                    w = self.mask[rows]
                    see[:, past:] = w[:, j // 32] >> (j % 32).astype(np.uint32) & 1
            see &= at >= 0
            at = np.maximum(at, 0)
            for h in range(self.heads):
                kk, vv, qq = k[at, h // group], v[at, h // group], q[rows, h]
                x = self.scale * (qq @ kk.T)
                d = (QN * self.hd + 8) * U * abs(self.scale) * (np.abs(qq) @ np.abs(kk).T)
                x = np.where(see, x, -np.inf)
                top = x.max(1, initial=-np.inf, keepdims=True)
                p = np.where(see, np.exp(x - np.where(np.isinf(top), 0, top)), 0)
                total = p.sum(1, keepdims=True)
                p = p / np.where(total == 0, 1, total)
                dm = np.where(see, d, 0).max(1, initial=0.0)[:, None]
                vf = np.where(np.isnan(vv), 0, vv)
                out[rows, h] = p @ vf
                tol[rows, h] = (2 * dm + (6 + PN * n) * U + cut) * (p @ np.abs(vf))
                tol[rows, h] += n * 2.0 ** -126 * (np.abs(vf).max(initial=0) + PN * float(MOST[self.f]))
        return out, tol + E.rounded(out, self.t), live

    def check(self, raw, what=""):
        want, tol, live = self.expected()
        got = E.decode(raw, self.t)[:, :self.heads * self.hd].reshape(want.shape)
        with np.errstate(invalid="ignore"):
            near = np.abs(got - want) <= tol
        if self.t == E.F16:
            # f16 ends at 65504: what rounds to 65520 or more is infinite.
            over = np.isinf(got) & (got * want > 0) & (np.abs(want) + tol >= 65520)
            near = over | (near & (np.abs(want) - tol <= 65520))
        bad = live[:, None, None] & ~near
        assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(),
                               float(np.nanmax(np.where(bad, np.abs(got - want) / tol, 0))))
        # rows of no sequence, and what lies behind the heads, as they were
        same = raw.view(np.uint8) == self.out0.view(np.uint8)
        assert same[~live].all() and same[:, self.heads * self.hd * E.SIZE[self.t]:].all(), what
