"""A layer's attention block as a serving program would run it: 8-bit products
around norms, rotation and cache store and the attention of drafted tokens over a
paged cache, launched one after the other on one stream. Each stage is held to its
formula in 64 bits on what the stage before left, with that operator's bound; the
same run is captured into a graph whose replays must give the same bits."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import elem_lib as E
from test_fp8_gpu import expected, operands, quantized, tolerance
from test_rope_gpu import close, turned
from test_tree_attention_gpu import Hip
from tree_lib import Tree

pytestmark = pytest.mark.gpu
U = E.U


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


class Block:
    def __init__(self, M, lens, t, d=1040, heads=6, kvh=2, hd=128):
        self.M, self.t, self.hd, self.heads, self.kvh, self.cols = M, t, hd, heads, kvh, d
        rng = self.rng = np.random.default_rng(len(lens))
        self.c = Tree(M, lens, heads, kvh, hd, t, page=16, seed=1)
        self.n = n = self.c.rows
        self.x = E.encode(rng.standard_normal((n, d)) * 2, t)
        self.row = (heads + 2 * kvh) * hd
        self.w = [operands(rng, self.row, d, 1)[:2], operands(rng, d, heads * hd, 1)[:2]]
        self.norms = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
        self.freqs, _ = M.rope_freqs(hd, 1e6)
        depth = [bin(int(v)).count("1") - 1 if self.c.words == 1 else 0
                 for v in self.c.mask[:, 0]]
        self.pos, self.slots = np.zeros(n, np.int32), np.zeros(n, np.int32)
        for b, (past, nodes) in enumerate(lens):
            at = slice(self.c.start[b], self.c.start[b] + nodes)
            self.pos[at] = past + np.array(depth[at], np.int32)
            self.slots[at] = self.c.cache_rows(b, past + nodes)[past:]
        self.args = self.c.args()
        B = M.DeviceBuffer.from_array
        self.d = {k: B(v) for k, v in dict(
            x=self.x, w0=self.w[0][0], s0=self.w[0][1], w1=self.w[1][0], s1=self.w[1][1],
            qn=self.norms[0], kn=self.norms[1], freqs=self.freqs, pos=self.pos,
            slots=self.slots).items()}
        nb = lambda k: -(-k // 128)  # noqa: E731
        size = E.SIZE[t]
        for k, bytes_ in dict(xq=n * d, xs=4 * n * nb(d), qkv=n * self.row * size,
                              aq=n * heads * hd, as_=4 * n * nb(heads * hd),
                              y=n * d * 4).items():
            self.d[k] = M.DeviceBuffer(bytes_)
        self.need = M.tree_attention_workspace(self.args)
        self.ws = M.DeviceBuffer(self.need)
        p, c = (lambda k: self.d[k].ptr), self.c
        self.qk = M.QkNormRope(
            type=t, out_type=t, layout=0, n_heads=heads, n_kv_heads=kvh, head_dim=hd, rot_dim=hd,
            tokens=n, q=p("qkv"), k=p("qkv") + heads * hd * size,
            v=p("qkv") + (heads + kvh) * hd * size, q_stride=self.row, k_stride=self.row,
            v_stride=self.row, q_norm=p("qn"), k_norm=p("kn"), eps=1e-6, mscale=1.0,
            freqs=p("freqs"), pos=p("pos"), slots=p("slots"), n_slots=c.slots,
            q_out=c.d["q"].ptr, q_out_stride=c.qs, k_cache=c.d["k"].ptr, v_cache=c.d["v"].ptr,
            slot_stride=c.ss)

    def run(self, stream=None):
        M, p, n, w = self.M, (lambda k: self.d[k].ptr), self.n, self.heads * self.hd
        M.fp8_quantize_dev(self.t, p("x"), self.cols, n, self.cols, p("xq"), p("xs"), stream)
        M.fp8_matmat_dev(p("w0"), p("s0"), self.row, self.cols, p("xq"), p("xs"), self.t,
                         p("qkv"), n, stream)
        M.qk_norm_rope_dev(self.qk, stream)
        M.tree_attention_dev(self.args, self.ws.ptr, self.need, stream)
        M.fp8_quantize_dev(self.t, self.c.d["out"].ptr, w, n, w, p("aq"), p("as_"), stream)
        M.fp8_matmat_dev(p("w1"), p("s1"), self.cols, w, p("aq"), p("as_"), E.F32, p("y"),
                         n, stream)

    def get(self, k, dtype, *shape):
        return self.d[k].download(dtype, int(np.prod(shape))).reshape(shape)

    def check(self):
        c, n, w, t = self.c, self.n, self.heads * self.hd, self.t
        nb = -(-self.cols // 128)
        codes, scales = quantized(E.decode(self.x, t).astype(np.float32))
        xq, xs = self.get("xq", np.uint8, n, self.cols), self.get("xs", np.float32, n, nb)
        assert np.array_equal(xs, scales) and np.array_equal(E.E4M3[xq], E.E4M3[codes])
        y, s, top = expected(*self.w[0], xq, xs)
        qkv = E.decode(self.get("qkv", E.NP[t], n, self.row), t)
        assert np.all(np.abs(qkv - y) <= tolerance(y, s, top, nb, t))
        v = qkv.reshape(n, -1, self.hd)
        old_k, old_v = c.k.copy(), c.v.copy()
        for key in ("q", "k", "v"):
            a = getattr(c, key)
            setattr(c, key, c.d[key].download(E.NP[t], a.size).reshape(a.shape))
        rows = np.setdiff1d(np.arange(c.slots), self.slots)
        assert np.array_equal(c.k[rows], old_k[rows]) and np.array_equal(c.v[rows], old_v[rows])
        for got, x, g in ((c.q, v[:, :self.heads], self.norms[0]),
                          (c.k[self.slots], v[:, self.heads:self.heads + self.kvh],
                           self.norms[1])):
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * g.astype(np.float64)
            want, size, far = turned(x, 0, self.hd, self.freqs, 1.0, self.pos)
            close(E.decode(got, t).reshape(want.shape), want,
                  18 * U * size + far + E.rounded(want, t), "qk")
        assert np.array_equal(E.decode(c.v[self.slots], t).reshape(n, -1, self.hd),
                              v[:, self.heads + self.kvh:])
        out = c.raw()
        c.check(out)
        codes, scales = quantized(E.decode(out, t).astype(np.float32))
        aq, as_ = self.get("aq", np.uint8, n, w), self.get("as_", np.float32, n, -(-w // 128))
        assert np.array_equal(as_, scales) and np.array_equal(E.E4M3[aq], E.E4M3[codes])
        y, s, top = expected(*self.w[1], aq, as_)
        assert np.all(np.abs(self.get("y", np.float32, n, self.cols) - y) <=
                      tolerance(y, s, top, -(-w // 128), E.F32))


@pytest.mark.parametrize("t", [E.F16, E.BF16])
@pytest.mark.parametrize("lens", [[(0, 1)], [(130, 1), (7, 1), (64, 1)],
                                  [(200, 24), (0, 3), (33, 16)], [(1500, 30), (20, 32), (3, 17)]],
                         ids=str)
def test_attention_block(M, t, lens):
    print("[case] block", t, lens, flush=True)
    b = Block(M, lens, t)
    b.run()
    M.sync()
    b.check()


def test_captured_block(M):
    b, hip = Block(M, [(90, 12), (5, 4)], E.BF16), Hip()
    st = hip.stream()
    g, e = hip.capture(st, lambda: b.run(st))
    for turn in range(3):
        x = E.encode(b.rng.standard_normal(b.x.shape) * (turn + 1), b.t)
        b.d["x"].upload(x)
        assert hip.lib.hipGraphLaunch(e, C.c_void_p(st)) == 0
        M.check(M.lib.mynah_hip_sync(st), "sync")
        replay = b.get("y", np.uint32, b.n, b.cols)
        assert np.isfinite(replay.view(np.float32)).all()
        b.d["y"].upload(np.zeros((b.n, b.cols), np.float32))
        b.run()                                         # the library's own stream
        M.sync()
        assert np.array_equal(replay, b.get("y", np.uint32, b.n, b.cols))
    hip.lib.hipGraphExecDestroy(e)
    hip.lib.hipGraphDestroy(g)
    hip.lib.hipStreamDestroy(C.c_void_p(st))
