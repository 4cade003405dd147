"""Inputs, the 64-bit result and the error bound of tree attention calls, for
the operator's tests."""
from __future__ import annotations

import numpy as np

import elem_lib as E

U = E.U


class Tree:
    """One call: a ragged batch over a contiguous or paged cache.

    lens: [(committed positions, nodes)] of the sequences; mask "tree" (random
    ancestors), "chain" (no mask given) or an array [rows][words] of uint32."""

    def __init__(self, M, lens, heads, kvh, hd, t, page=0, mask="tree", seed=0, extra_rows=0,
                 max_nodes=None, max_kv=None, pad=0, scale=None):
        self.M, self.lens, self.heads, self.kvh, self.hd, self.t = M, lens, heads, kvh, hd, t
        rng = self.rng = np.random.default_rng(seed)
        n = len(lens)
        self.past = np.array([p for p, _ in lens], np.int32)
        self.nodes = np.array([k for _, k in lens], np.int32)
        self.start = np.concatenate([[0], np.cumsum(self.nodes)]).astype(np.int32)
        self.rows = int(self.start[-1]) + extra_rows
        self.max_nodes = max_nodes or max(1, int(self.nodes.max()))
        self.max_kv = max_kv or max(1, int((self.past + self.nodes).max()))
        self.words = -(-self.max_nodes // 32)
        self.page = page
        if page:
            self.max_pages = -(-self.max_kv // page)
            self.slots = n * self.max_pages * page
            self.pages = rng.permutation(n * self.max_pages).astype(np.int32)
            self.pages = self.pages.reshape(n, self.max_pages)
        else:
            self.slots, self.pages, self.max_pages = n * self.max_kv, None, 0
        self.ss = kvh * hd + pad                       # cache rows' stride
        self.qs = heads * hd + pad
        self.k = E.encode(rng.standard_normal((self.slots, self.ss)), t)
        self.v = E.encode(rng.standard_normal((self.slots, self.ss)), t)
        self.q = E.encode(1.5 * rng.standard_normal((self.rows, self.qs)), t)
        self.scale = hd ** -0.5 if scale is None else scale
        self.mask = None
        if not isinstance(mask, str):
            self.mask = mask
        elif mask == "tree":
            self.mask = np.zeros((self.rows, self.words), np.uint32)
            for b in range(n):
                for i in range(self.nodes[b]):
                    row = self.start[b] + i
                    parent = int(rng.integers(-1, i)) if i else -1
                    if parent >= 0:
                        self.mask[row] = self.mask[self.start[b] + parent]
                    if i < 32 * self.words:
                        self.mask[row, i // 32] |= np.uint32(1 << (i % 32))

    def args(self, **change):
        B = self.M.DeviceBuffer.from_array
        self.out0 = E.encode(np.full((self.rows, self.qs), 11.0), self.t)
        self.d = {"q": B(self.q), "k": B(self.k), "v": B(self.v), "out": B(self.out0),
                  "start": B(self.start), "past": B(self.past)}
        if self.pages is not None:
            self.d["pages"] = B(self.pages)
        if self.mask is not None:
            self.d["mask"] = B(self.mask)
        at = lambda k: self.d[k].ptr if k in self.d else None  # noqa: E731
        v = dict(type=self.t, n_seqs=len(self.lens), n_heads=self.heads, n_kv_heads=self.kvh,
                 head_dim=self.hd, q=at("q"), q_stride=self.qs, out=at("out"),
                 out_stride=self.qs, n_rows=self.rows, k_cache=at("k"), v_cache=at("v"),
                 slot_stride=self.ss, n_slots=self.slots,
                 seq_slots=0 if self.page else self.max_kv, pages=at("pages"),
                 page_size=self.page, max_pages=self.max_pages, seq_start=at("start"),
                 n_past=at("past"), mask=at("mask"), mask_words=self.words,
                 max_nodes=self.max_nodes, max_kv=self.max_kv, scale=self.scale)
        return self.M.TreeAttention(**{**v, **change})

    def call(self, stream=None, **change):
        a = self.args(**change)
        n = self.M.tree_attention_workspace(a)
        self.ws = self.M.DeviceBuffer.from_array(np.full(n, 0xFF, np.uint8))   # NaN, stale
        self.M.tree_attention_dev(a, self.ws.ptr, n, stream)
        self.M.check(self.M.lib.mynah_hip_sync(stream), "sync")
        return self.raw()

    def raw(self):
        return self.d["out"].download(E.NP[self.t], self.q.size).reshape(self.q.shape)

    def cache_rows(self, b, n):
        p = np.arange(n)
        if self.page:
            return self.pages[b, p // self.page].astype(np.int64) * self.page + p % self.page
        return b * self.max_kv + p

    def expected(self):
        """(out [rows][heads][hd], bound, which rows are written). Per output, with
        A = sum p |v|: a score is a sum of hd products in f32 and two roundings, off
        by at most d = (hd + 4) u scale |q| . |k| (its largest over the row), and
        exp follows it: 2 d A + 6 u A; the sums over n positions add n u A; of 16-bit
        types each probability is rounded to the type, a half step of A."""
        out = np.zeros((self.rows, self.heads, self.hd))
        tol = np.zeros_like(out)
        live = np.zeros(self.rows, bool)
        group = self.heads // self.kvh
        heads = lambda a, n: E.decode(a, self.t)[:, :n * self.hd].reshape(-1, n, self.hd)  # noqa
        q, k, v = heads(self.q, self.heads), heads(self.k, self.kvh), heads(self.v, self.kvh)
        for b, (past, _) in enumerate(self.lens):
            nodes = min(int(self.nodes[b]), self.max_nodes)
            past = max(past, 0)
            n = min(past + nodes, self.max_kv)
            rows = slice(int(self.start[b]), int(self.start[b]) + nodes)
            live[rows] = True
            at = self.cache_rows(b, n)
            there = (at >= 0) & (at < self.slots)
            if self.page:
                there &= self.pages[b, np.arange(n) // self.page] >= 0
            at = np.where(there, at, 0)
            see = np.ones((nodes, n), bool)
            for i in range(nodes):
                for j in range(max(n - past, 0)):
                    see[i, past + j] = j <= i if self.mask is None else \
                        bool(self.mask[rows.start + i, j // 32] >> np.uint32(j % 32) & 1)
            see &= there
            for h in range(self.heads):
                kk, vv, qq = k[at, h // group], v[at, h // group], q[rows, h]
                with np.errstate(invalid="ignore"):
                    x = self.scale * (qq @ kk.T)
                    d = (self.hd + 4) * U * abs(self.scale) * (np.abs(qq) @ np.abs(kk).T)
                x = np.where(see, x, -np.inf)
                top = x.max(1, initial=-np.inf, keepdims=True)
                p = np.where(see, np.exp(x - np.where(np.isinf(top), 0, top)), 0)
                total = p.sum(1, keepdims=True)
                p = p / np.where(total == 0, 1, total)
                for i in range(nodes):
                    s = see[i]
                    out[rows.start + i, h] = p[i, s] @ vv[s]
                    big = p[i, s] @ np.abs(vv[s])
                    dm = np.where(s, d[i], 0).max(initial=0.0)
                    tol[rows.start + i, h] = (2 * dm + (6 + n) * U +
                                              (0 if self.t == E.F32 else E.HALF[self.t])) * big
        return out, tol + E.rounded(out, self.t), live

    def check(self, raw, what=""):
        want, tol, live = self.expected()
        got = E.decode(raw, self.t)[:, :self.heads * self.hd].reshape(want.shape)
        with np.errstate(invalid="ignore"):
            bad = live[:, None, None] & ~(np.abs(got - want) <= tol)
            assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(),
                                   float(np.nanmax(np.where(bad, np.abs(got - want) / tol, 0))))
        # rows of no sequence, and what lies behind the heads, as they were
        same = raw.view(np.uint8) == self.out0.view(np.uint8)
        size = E.SIZE[self.t]
        assert same[~live].all() and same[:, self.heads * self.hd * size:].all(), what
