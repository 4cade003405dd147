"""Token rows that are not there in the 8-bit cache's store (mynah_hip_kv8_store_dev):
sequences that begin before row 0 or end behind n_rows, in batches whose blocks are
numbered by the longest sequence and by rows."""
from __future__ import annotations

import numpy as np
import pytest

import elem_lib as E
from kv8_lib import E4M3, I8, Kv8, codes_of, scale_of, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


class Rows(Kv8):
    """A batch whose sequences' rows lie `shift` from where they lay, `rows` of them there.
    A block that gets no row keeps its scale and codes."""

    def move(self, shift, rows=None):
        self.start = (self.start + shift).astype(np.int32)
        self.rows = max(1, int(self.start[-1]) if rows is None else rows)
        take = np.arange(self.rows) % len(self.kx)
        self.kx, self.vx, self.q = self.kx[take], self.vx[take], self.q[take]
        return self

    def expected_store(self):
        out = {n: getattr(self, n).copy() for n in ("k", "v", "ks", "vs")}
        heads, n = (-1, self.kvh, self.hd), self.kvh * self.hd
        for b, (past, _) in enumerate(self.lens):
            end = min(past + min(int(self.nodes[b]), self.max_nodes), self.max_kv)
            at = self.cache_rows(b, max(end, past))
            for first in range(past // self.block * self.block, end, self.block):
                p = np.arange(max(first, past), min(first + self.block, end))
                row = self.start[b] + p - past
                there = (row >= 0) & (row < self.rows)
                if end <= past or not there.any():
                    continue
                blk, kept = at[first] // self.block, at[first:past]
                for c, s, x in (("k", "ks", self.kx), ("v", "vs", self.vx)):
                    x = E.decode(x[row[there]], self.t).astype(np.float32)[:, :n].reshape(heads)
                    old = out[s][blk].copy()
                    old = np.where((old > 0) & np.isfinite(old), old, np.float32(0))
                    new = scale_of(np.abs(x).max((0, 2)), self.f)
                    if first < past:
                        new = np.maximum(new, old)
                        was = out[c][kept][:, :n].reshape(heads)
                        again = codes_of(values(was, self.f), (old / new)[:, None], self.f)
                        again = np.where((old == new)[:, None], was, again)
                        out[c][kept, :n] = again.reshape(-1, n)
                    out[s][blk] = new
                    put = codes_of(x, (np.float32(1) / new)[:, None], self.f)
                    out[c][at[p[there]], :n] = put.reshape(-1, n)
        return out


@pytest.mark.parametrize("f", [I8, E4M3])
@pytest.mark.parametrize("hd", [64, 256])
def test_blocks_that_get_no_row(M, f, hd):
    print("[case] kv8 rows", f, hd, flush=True)
    # Rows -50 .. 9 of positions 20 .. 79, 10 .. 12, and from 13 on more than there are.
    c = Rows(M, [(20, 60), (5, 3), (30, 40)], 2, 2, hd, E.F32, f, 16, page=32, seed=5).move(-50, 20)
    blocks = c.cache_rows(0, 80)[::16] // 16
    c.ks[blocks[1]], c.vs[blocks[2]], c.ks[blocks[0]] = np.nan, -1, 0
    c.check_store(c.store())


@pytest.mark.parametrize("f", [I8, E4M3])
@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("where", [0, 69])
@pytest.mark.parametrize("shift,cut", [(-2300, 0), (-2420, 0), (-20, 0), (37, 0), (0, 50), (-2300, 30)])
def test_ragged_batches_past_the_rows(M, f, page, where, shift, cut):
    """One long sequence among many, so that blocks are numbered by rows, some of which
    are before the first or behind the last one."""
    rng = np.random.default_rng(1)
    lens = [(int(a), int(b)) for a, b in zip(rng.integers(0, 20, 70), rng.integers(0, 4, 70))]
    lens[where] = (13, 2400)
    c = Rows(M, lens, 2, 1, 64, E.BF16, f, 16, page=page, seed=6)
    c.move(shift, max(1, int(c.start[-1]) + shift - cut))
    got = c.store()
    c.check_store(got, (shift, cut))
