"""A page pool on the host and on the device, side by side: every call's definition
(include/mynah_cache.h) done one sequence and one position after the other."""
from __future__ import annotations

import ctypes as C

import numpy as np


class Pool:
    def __init__(self, M, n_pages, n_seqs, max_pages, page=16, parts=((64, 64),), seed=0):
        """parts: (bytes, stride) of a page's parts."""
        self.M, self.n_pages, self.n_seqs, self.max_pages, self.page = M, n_pages, n_seqs, max_pages, page
        rng = self.rng = np.random.default_rng(seed)
        self.sizes = parts
        self.parts = [rng.integers(0, 256, (n_pages, stride)).astype(np.uint8) for _, stride in parts]
        self.refs = np.zeros(n_pages, np.int32)
        self.pages = np.full((n_seqs, max_pages), -1, np.int32)
        self.n_past = np.zeros(n_seqs, np.int32)
        self.status = np.zeros(2, np.int32)
        self.d = None

    # ── the definition ───────────────────────────────────────────────────────

    def valid(self, p):
        return 0 <= p < self.n_pages

    def count(self):
        flat = self.pages[(self.pages >= 0) & (self.pages < self.n_pages)]
        self.refs = np.bincount(flat, minlength=self.n_pages).astype(np.int32)

    def move(self, pairs):
        old = [p.copy() for p in self.parts]
        for f, t in pairs:
            for (size, _), part, was in zip(self.sizes, self.parts, old):
                part[t, :size] = was[f, :size]

    def fork(self, source):
        table, past = self.pages.copy(), self.n_past.copy()
        for b, f in enumerate(source):
            some = 0 <= f < self.n_seqs
            self.pages[b] = table[f] if some else -1
            self.n_past[b] = past[f] if some else 0
        self.count()

    def reserve(self, n_new):
        spans, long_ = [], 0
        for b in range(self.n_seqs):
            past, n = max(int(self.n_past[b]), 0), max(int(n_new[b]), 0)
            to = -(-(past + n) // self.page)
            if n and to > self.max_pages:
                long_ += 1
            spans.append(range(past // self.page, min(to, self.max_pages)) if n else range(0))
        asks = {}
        for b, s in enumerate(spans):
            for j in s:
                asks.setdefault(int(self.pages[b, j]), []).append(b)
        get = []
        for b, s in enumerate(spans):
            for j in s:
                p = int(self.pages[b, j])
                if self.valid(p) and (self.refs[p] <= 1 or
                                      (len(asks[p]) == self.refs[p] and min(asks[p]) == b)):
                    continue
                get.append((b, j, p))
        free = np.flatnonzero(self.refs == 0)
        self.status[:] = max(0, len(get) - len(free)), long_
        if self.status.any():
            return
        pairs = []
        for (b, j, p), new in zip(get, free):
            self.pages[b, j] = new
            if self.valid(p) and j * self.page < self.n_past[b]:
                pairs.append((p, new))
        self.count()
        self.move(pairs)

    def release(self, keep):
        for b, k in enumerate(keep):
            if k >= 0:
                self.pages[b, -(-int(k) // self.page):] = -1
                self.n_past[b] = min(self.n_past[b], k)
        self.count()

    def compact(self):
        live = int((self.refs > 0).sum())
        to = [p for p in range(live) if self.refs[p] == 0]
        source = [p for p in range(live, self.n_pages) if self.refs[p] > 0]
        new = np.arange(self.n_pages)
        new[source] = to
        ok = (self.pages >= 0) & (self.pages < self.n_pages)
        self.pages[ok] = new[self.pages[ok]]
        self.count()
        self.move(list(zip(source, to)))
        self.status[:] = live, len(to)

    def copy(self, source, to):
        self.move([(f, t) for f, t in zip(source, to) if self.valid(f) and self.valid(t)])

    # ── the device ───────────────────────────────────────────────────────────

    def upload(self):
        B = self.M.DeviceBuffer.from_array
        self.d = {n: B(getattr(self, n)) for n in ("refs", "pages", "n_past", "status")}
        self.mem = [B(p) for p in self.parts]
        rows = np.array([[m.ptr, stride, size] for m, (size, stride) in zip(self.mem, self.sizes)],
                        np.uint64)
        self.d["parts"] = B(rows)
        self.args = self.M.PagePool(
            n_pages=self.n_pages, n_seqs=self.n_seqs, max_pages=self.max_pages, page_size=self.page,
            n_parts=len(self.parts), **{n: self.d[n].ptr for n in self.d})
        self.need = self.M.pages_workspace(self.args)
        self.ws = self.M.DeviceBuffer.from_array(np.full(self.need, 0x7F, np.uint8))
        self.ask = [self.M.DeviceBuffer(4 * max(self.n_seqs, self.n_pages)) for _ in range(2)]

    def call(self, op, *ints, stream=None):
        """One operator on the device; its definition on the host is the caller's."""
        M = self.M
        for buf, x in zip(self.ask, ints):
            buf.upload(np.ascontiguousarray(x, np.int32))
        a = self.ask[0].ptr
        if op == "fork":
            M.pages_fork_dev(self.args, a, self.ws.ptr, self.need, stream)
        elif op == "reserve":
            M.pages_reserve_dev(self.args, a, self.ws.ptr, self.need, stream)
        elif op == "release":
            M.pages_release_dev(self.args, a, stream)
        elif op == "compact":
            M.pages_compact_dev(self.args, self.ws.ptr, self.need, stream)
        else:
            M.pages_copy_dev(self.args, a, self.ask[1].ptr, len(ints[0]), stream)

    def both(self, op, *ints, what=""):
        if self.d is None:
            self.upload()
        self.call(op, *ints)
        getattr(self, op)(*ints)
        self.M.sync()
        self.check((what, op))

    def check(self, what=""):
        for n in ("pages", "refs", "n_past", "status"):
            want = getattr(self, n)
            got = self.d[n].download(np.int32, want.size).reshape(want.shape)
            if n == "status" and what and what[1] not in ("reserve", "compact"):
                self.status = got.copy()
                continue
            assert np.array_equal(got, want), (what, n, np.argwhere(got != want)[:4].tolist())
        for i, (m, p) in enumerate(zip(self.mem, self.parts)):
            got = m.download(np.uint8, p.size).reshape(p.shape)
            assert np.array_equal(got, p), (what, "part", i, np.argwhere(got != p)[:4].tolist())
