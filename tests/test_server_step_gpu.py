"""A server's steps as a program would run them over a paged 8-bit cache: sequences fork
and get pages, q/k norms with rotation make the new rows, the store puts them into
the cache, the attention reads it, rules apply to logits made from its output; then
drafted tokens are cut off again, a sequence ends, and the pool is compacted. Each
stage is held to its definition on what the stage before left; the same run from a
captured graph gives the same bits."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import elem_lib as E
from kv8_lib import E4M3, I8, Kv8
from pages_lib import Pool
from test_logits_gpu import Case
from test_rope_gpu import close, turned
from test_tree_attention_gpu import Hip

pytestmark = pytest.mark.gpu
U = E.U


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


class Server:
    """One layer's cache of a pool of pages, four sequences at most."""
    heads, kvh, hd, block, page, max_pages, vocab = 6, 2, 64, 16, 32, 6, 384

    def __init__(self, M, t, f, max_new):
        self.M, self.t, self.f, self.n = M, t, f, 4
        self.max_new, row = max_new, self.kvh * self.hd
        self.n_pages = self.n * self.max_pages
        n_rows = self.n * max_new
        c = self.c = Kv8(M, [(0, max_new)] * self.n, self.heads, self.kvh, self.hd, t, f, self.block,
                         self.page, max_nodes=max_new, max_kv=self.max_pages * self.page, seed=3)
        assert c.max_pages == self.max_pages and c.rows == n_rows
        c.pages[:] = -1
        c.upload()
        self.pool = p = Pool(M, self.n_pages, self.n, self.max_pages, self.page,
                             ((self.page * row, self.page * row),) * 2 +
                             ((self.page // self.block * self.kvh * 4,) * 2,) * 2)
        for i, name in enumerate(("k", "v", "ks", "vs")):
            p.parts[i] = getattr(c, name).view(np.uint8).reshape(self.n_pages, -1).copy()
        p.upload()
        # the pool manages the cache's own memory, table and lengths
        rows = [[c.at(name), s, s] for name, (s, _) in zip(("k", "v", "ks", "vs"), p.sizes)]
        p.d["parts"].upload(np.array(rows, np.uint64))
        p.d["pages"], p.d["n_past"] = c.d["pages"], c.d["past"]
        c.d["past"].upload(p.n_past)
        p.args.pages, p.args.n_past = c.at("pages"), c.at("past")
        p.mem = [c.d[name] for name in ("k", "v", "ks", "vs")]
        # projections of the new tokens; norms, positions
        B = M.DeviceBuffer.from_array
        rng = self.rng = np.random.default_rng(5)
        self.width = (self.heads + 2 * self.kvh) * self.hd
        self.norm = (1 + 0.2 * rng.standard_normal((2, self.hd))).astype(np.float32)
        self.freqs, _ = M.rope_freqs(self.hd, 1e4)
        size = E.SIZE[t]
        self.d = {"x": M.DeviceBuffer(n_rows * self.width * size), "pos": M.DeviceBuffer(4 * n_rows),
                  "qn": B(self.norm[0]), "kn": B(self.norm[1]), "freqs": B(self.freqs),
                  "from": M.DeviceBuffer(16), "new": M.DeviceBuffer(16), "keep": M.DeviceBuffer(16)}
        at = lambda k: self.d[k].ptr  # noqa: E731
        self.qk = M.QkNormRope(
            type=t, out_type=t, layout=0, n_heads=self.heads, n_kv_heads=self.kvh, head_dim=self.hd,
            rot_dim=self.hd, tokens=n_rows, q=at("x"), k=at("x") + self.heads * self.hd * size,
            v=at("x") + (self.heads + self.kvh) * self.hd * size, q_stride=self.width,
            k_stride=self.width, v_stride=self.width, q_norm=at("qn"), k_norm=at("kn"), eps=1e-6,
            mscale=1.0, freqs=at("freqs"), pos=at("pos"), n_slots=n_rows, q_out=c.at("q"),
            q_out_stride=c.qs, k_cache=c.at("kx"), v_cache=c.at("vx"), slot_stride=c.xs)
        self.store, self.attn = c.store_args(), c.attn_args()
        self.need = M.kv8_attention_workspace(self.attn)
        self.ws = M.DeviceBuffer(self.need)
        # logits: the attention's rows, cut to the vocabulary
        self.rules = Case(M, n_rows, self.vocab, t, E.F32, hist=[9] * n_rows, bias=[3] * n_rows, masks=4,
                          seed=8)
        self.logits = self.rules.args()
        self.logits.x, self.logits.x_stride = c.at("out"), c.qs

    def launch(self, stream=None):
        M, p = self.M, self.pool
        M.pages_fork_dev(p.args, self.d["from"].ptr, p.ws.ptr, p.need, stream)
        M.pages_reserve_dev(p.args, self.d["new"].ptr, p.ws.ptr, p.need, stream)
        M.qk_norm_rope_dev(self.qk, stream)
        M.kv8_store_dev(self.store, stream)
        M.kv8_attention_dev(self.attn, self.ws.ptr, self.need, stream)
        M.logits_dev(self.logits, stream)

    def inputs(self, source, new):
        """Uploads a step's; the host's pool follows."""
        p, c = self.pool, self.c
        p.fork(source)
        p.reserve(new)
        assert not p.status.any()
        c.pages[:] = p.pages
        c.past[:] = p.n_past
        c.lens = [(int(a), int(b)) for a, b in zip(p.n_past, new)]
        c.nodes = np.array(new, np.int32)
        c.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.pos = np.zeros(c.rows, np.int32)
        for b, k in enumerate(new):
            self.pos[c.start[b]:c.start[b + 1]] = p.n_past[b] + np.arange(k)
        self.x = E.encode(self.rng.standard_normal((c.rows, self.width)) * 2, self.t)
        self.d["x"].upload(self.x)
        self.d["pos"].upload(self.pos)
        self.d["from"].upload(np.array(source, np.int32))
        self.d["new"].upload(np.array(new, np.int32))
        c.d["start"].upload(c.start)
        c.d["out"].upload(c.out0)

    def check(self, what):
        c, p, t = self.c, self.pool, self.t
        used = int(c.start[-1])
        # tables, and the content that moved (the store has written since: its rows below)
        for n in ("pages", "refs", "n_past", "status"):
            got = p.d[n].download(np.int32, getattr(p, n).size).reshape(getattr(p, n).shape)
            assert np.array_equal(got, getattr(p, n)), (what, n)
        # norms and rotation
        v = E.decode(self.x, t).reshape(c.rows, -1, self.hd)
        get = lambda n: c.d[n].download(E.NP[t], getattr(c, n).size).reshape(getattr(c, n).shape)  # noqa: E731
        c.q, c.kx, c.vx = get("q"), get("kx"), get("vx")
        for got, x, w in ((c.q, v[:, :self.heads], self.norm[0]),
                          (c.kx, v[:, self.heads:self.heads + self.kvh], self.norm[1])):
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w.astype(np.float64)
            want, size, far = turned(x, 0, self.hd, self.freqs, 1.0, self.pos)
            close(E.decode(got, t).reshape(want.shape), want, 18 * U * size + far + E.rounded(want, t),
                  what)
        assert np.array_equal(E.decode(c.vx, t).reshape(c.rows, -1, self.hd),
                              v[:, self.heads + self.kvh:])
        # the store, on the pages as the pool left them
        for i, n in enumerate(("k", "v", "ks", "vs")):
            a = getattr(c, n)
            setattr(c, n, p.parts[i].reshape(-1).view(a.dtype).reshape(a.shape).copy())
        got = c.stored()
        c.check_store(got, what)
        for i, n in enumerate(("k", "v", "ks", "vs")):
            setattr(c, n, got[n])
            p.parts[i] = got[n].view(np.uint8).reshape(self.n_pages, -1).copy()
        raw = c.raw()
        c.check(raw, what)
        # the rules, on the attention's own rows
        r = self.rules
        r.x = raw[:, :self.vocab]
        assert np.array_equal(r.get()[:used], r.expected()[:used]), what
        return raw[:used].copy(), r.get()[:used].copy()

    def step(self, source, new, what):
        self.inputs(source, new)
        self.launch()
        self.M.sync()
        out = self.check(what)
        self.advance(new)
        return out

    def advance(self, new):
        self.pool.n_past += np.array(new, np.int32)
        self.c.d["past"].upload(self.pool.n_past)

    def cut(self, keep):
        p = self.pool
        self.d["keep"].upload(np.array(keep, np.int32))
        self.M.pages_release_dev(p.args, self.d["keep"].ptr)
        p.release(keep)
        p.both("compact", what=keep)


@pytest.mark.parametrize("t", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("f", [I8, E4M3])
def test_steps(M, t, f):
    print("[case] server", t, f, flush=True)
    s = Server(M, t, f, 45)
    s.step([0, 1, -1, -1], [45, 33, 0, 0], "two prompts")
    s.step([0, 1, 0, 0], [1, 1, 1, 1], "samples of the first")
    s.step([0, 1, 2, 3], [4, 3, 0, 5], "drafts")
    s.cut([47, -1, 46, 0])                              # what was not taken; the last ends
    s.step([2, 1, 2, 0], [1, 20, 1, 1], "beams")
    s.step([3, 0, 1, 1], [1, 1, 1, 1], "beams in another order")


def test_captured_steps(M):
    """Steps of three shapes from one graph, each against the definition; then the same
    from the start by eager calls: the same bits."""
    plan = [([0, 1, -1, -1], [9, 12, 0, 0]), ([0, 0, 1, 1], [1, 1, 1, 1]), ([1, 3, 2, 0], [2, 1, 0, 5])]
    h, out = Hip(), []
    for captured in (True, False):
        s = Server(M, E.BF16, I8, 12)
        st = h.stream()
        if captured:
            g, e = h.capture(st, lambda: s.launch(st))
        got = []
        for source, new in plan:
            s.inputs(source, new)
            if captured:
                assert h.lib.hipGraphLaunch(e, C.c_void_p(st)) == 0
            else:
                s.launch(st)
            M.check(M.lib.mynah_hip_sync(st), "sync")
            got.append(s.check((captured, new)))
            s.advance(new)
        out.append(got)
        if captured:
            h.lib.hipGraphExecDestroy(e)
            h.lib.hipGraphDestroy(g)
        h.lib.hipStreamDestroy(C.c_void_p(st))
    for a, b in zip(*out):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))
