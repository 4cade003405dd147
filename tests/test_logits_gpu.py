"""Rules on a batch's logits (mynah_hip_logits_dev) against their definition in 32
bits, bit for bit: penalties, biases, grammars and all of them together, over types,
odd vocabularies and strides, in place, captured; penalties for each occurrence
against the device sampler's."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import elem_lib as E
from test_tree_attention_gpu import Hip

pytestmark = pytest.mark.gpu

F = np.float32


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


class Case:
    def __init__(self, M, rows, vocab, t=E.F32, o=E.F32, hist=(), bias=(), masks=0, pad=0, seed=0,
                 each=0, off=0):
        """hist, bias: each row's number of entries; off: elements by which x and y start late."""
        self.M, self.n, self.vocab, self.t, self.o, self.each, self.off = M, rows, vocab, t, o, each, off
        rng = self.rng = np.random.default_rng(seed)
        self.stride = vocab + pad
        self.x = E.encode(4 * rng.standard_normal((rows, self.stride)), t)
        self.y0 = E.encode(np.full((rows, self.stride), 7.0), o)
        self.a = {}
        if len(hist):
            # few tokens, often; the first and the last among them; some that are none
            ids = np.concatenate([rng.integers(0, vocab, 3 + sum(hist) // 8),
                                  [0, vocab - 1, vocab, -1, 2 ** 31 - 1, -2 ** 31]])
            self.a["hist"] = rng.choice(ids, sum(hist)).astype(np.int32)
            self.a["hist_start"] = np.concatenate([[0], np.cumsum(hist)]).astype(np.int64)
            self.a["repeat"] = rng.uniform(0.8, 1.5, rows).astype(F)
            self.a["freq"], self.a["presence"] = rng.uniform(-0.2, 0.6, (2, rows)).astype(F)
        if len(bias):
            ids = np.concatenate([rng.integers(0, vocab, 1 + sum(bias) // 2), [0, vocab - 1, vocab, -1]])
            self.a["bias_id"] = rng.choice(ids, sum(bias)).astype(np.int32)
            self.a["bias"] = rng.normal(0, 5, sum(bias)).astype(F)
            self.a["bias_start"] = np.concatenate([[0], np.cumsum(bias)]).astype(np.int64)
        self.masks, self.words = masks, -(-vocab // 32)
        if masks:
            self.a["allowed"] = rng.integers(0, 1 << 32, (masks, self.words)).astype(np.uint32)
            self.a["mask_row"] = rng.integers(-1, masks + 1, rows).astype(np.int32)

    def args(self, in_place=False, **change):
        B = self.M.DeviceBuffer.from_array
        flat = lambda z: np.concatenate([np.zeros(self.off, z.dtype), z.ravel()])  # noqa: E731
        self.d = {k: B(v) if v.size else self.M.DeviceBuffer(16) for k, v in self.a.items()}
        self.d["x"], self.d["y"] = B(flat(self.x)), B(flat(self.y0))
        p = {k: v.ptr for k, v in self.d.items()}
        p["x"] += self.off * E.SIZE[self.t]
        p["y"] += self.off * E.SIZE[self.o]
        if in_place:
            p["y"] = p["x"]
        return self.M.Logits(**{**p, **dict(
            type=self.t, out_type=self.o, n_rows=self.n, vocab=self.vocab, x_stride=self.stride,
            y_stride=self.stride, penalty=self.each, mask_words=self.words, n_masks=self.masks),
            **change})

    def get(self, name="y"):
        dtype = E.NP[self.o if name == "y" else self.t]
        return self.d[name].download(dtype, self.off + self.n * self.stride)[self.off:].reshape(
            self.n, self.stride)

    def expected(self):
        want = E.decode(self.x, self.t).astype(F)[:, :self.vocab].copy()
        with np.errstate(all="ignore"):
            for r in range(self.n):
                if "hist" in self.a:
                    s = self.a["hist_start"]
                    h = self.a["hist"][s[r]:s[r + 1]]
                    rep, freq, pres = (self.a[k][r] if k in self.a else F(d) for k, d in
                                       (("repeat", 1), ("freq", 0), ("presence", 0)))
                    for t, c in zip(*np.unique(h[(h >= 0) & (h < self.vocab)], return_counts=True)):
                        l = want[r, t]
                        for _ in range(c if self.each else 1):
                            l = l / rep if l > 0 else l * rep
                            l = l - F(freq * F(c))
                            l = l - pres
                        want[r, t] = l
                if "bias" in self.a:
                    s = self.a["bias_start"]
                    last = {int(i): b for i, b in zip(self.a["bias_id"][s[r]:s[r + 1]],
                                                      self.a["bias"][s[r]:s[r + 1]])}
                    for i, b in last.items():
                        if 0 <= i < self.vocab:
                            want[r, i] = want[r, i] + b
                m = int(self.a["mask_row"][r]) if "mask_row" in self.a else r
                if self.masks and 0 <= m < self.masks:
                    bits = np.unpackbits(self.a["allowed"][m].view(np.uint8), bitorder="little")
                    want[r, bits[:self.vocab] == 0] = -np.inf
        return E.encode(want, self.o)

    def check(self, got, what=""):
        want = self.expected()
        assert np.array_equal(E.decode(got[:, :self.vocab], self.o), E.decode(want, self.o),
                              equal_nan=True), what
        return got

    def call(self, **change):
        self.M.logits_dev(self.args(**change))
        self.M.sync()
        got = self.get()
        assert np.array_equal(got[:, self.vocab:], self.y0[:, self.vocab:])
        return self.check(got)


VOCABS = [1, 3, 31, 32, 33, 4099, 8192, 8193, 20_000, 151_936]


@pytest.mark.parametrize("each", [0, 1])
@pytest.mark.parametrize("vocab", VOCABS)
def test_everything_at_once(M, vocab, each):
    print("[case] logits", vocab, each, flush=True)
    c = Case(M, 5, vocab, hist=[0, 1, 40, 700, 3000], bias=[9, 0, 1, 70, 3], masks=3, seed=vocab,
             each=each)
    c.call()


@pytest.mark.parametrize("t", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("o", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("pad,off", [(0, 0), (3, 0), (4, 0), (0, 1)])
def test_types_and_strides(M, t, o, pad, off):
    c = Case(M, 3, 9000, t, o, hist=[50, 500, 7], bias=[4, 4, 4], masks=2, pad=pad, off=off, seed=pad)
    c.call()


@pytest.mark.parametrize("kw", [dict(), dict(hist=[30, 0, 5, 9]), dict(bias=[5, 0, 20, 1]),
                                dict(masks=4), dict(hist=[30, 0, 5, 9], masks=2),
                                dict(bias=[600, 0, 20, 1], hist=[1, 1, 1, 1])], ids=str)
def test_one_rule_or_none(M, kw):
    Case(M, 4, 5001, E.BF16, E.F32, seed=1, **kw).call()


def test_penalties_left_out(M):
    c = Case(M, 4, 3000, hist=[100] * 4, seed=2)
    full = dict(c.a)
    for keep in (("repeat",), ("freq",), ("presence",), ()):
        c.a = {k: v for k, v in full.items() if k.startswith("hist") or k in keep}
        c.call()
    c.a = dict(full)
    c.a["repeat"], c.a["freq"] = np.ones(4, F), np.zeros(4, F)
    c.a["presence"] = np.array([0, 1, 0, 0], F)
    c.call()


def test_masks_of_their_own_rows(M):
    c = Case(M, 4, 700, masks=4, seed=3)
    del c.a["mask_row"]
    c.a["allowed"][1] = 0                               # nothing is allowed
    c.a["allowed"][2] = 0xFFFFFFFF
    got = c.call()
    assert np.isneginf(got[1]).all()


def test_not_finite(M):
    """NaN and infinities go the way of the arithmetic, and are -inf where masked."""
    c = Case(M, 3, 400, hist=[200, 200, 200], bias=[5, 5, 5], masks=2, seed=4)
    c.x[:, ::7], c.x[:, 1::7], c.x[:, 2::7] = np.nan, np.inf, -np.inf
    c.a["mask_row"][:] = [0, -1, 1]
    c.call()
    # a row of -inf, and one of f32's lowest value
    c = Case(M, 2, 400, hist=[200, 200], bias=[5, 5], masks=2, seed=4)
    c.x[0], c.x[1] = -np.inf, np.finfo(F).min
    c.call()


def test_a_token_many_times(M):
    for each in (0, 1):
        c = Case(M, 2, 64, hist=[70_000, 66_000], seed=5, each=each)
        c.a["hist"][:] = 5
        c.a["freq"][:] = [1e-3, 0]
        c.call()


@pytest.mark.parametrize("t", [E.F32, E.BF16])
def test_in_place(M, t):
    c = Case(M, 6, 33_000, t, t, hist=[64] * 6, bias=[3] * 6, masks=2, pad=8, seed=6)
    M.logits_dev(c.args(in_place=True))
    M.sync()
    got = c.get("x")
    c.check(got)
    assert np.array_equal(got[:, c.vocab:], c.x[:, c.vocab:])


def test_many_rows(M):
    c = Case(M, 700, 96, E.F16, E.F16, hist=[20] * 700, bias=[2] * 700, masks=9, seed=7)
    c.call()


@pytest.mark.parametrize("kw", [
    dict(repeat_penalty=1.3, penalty_window=16), dict(repeat_penalty=0.9, penalty_window=64),
    dict(freq_penalty=0.2, presence_penalty=0.1, penalty_window=8),
    dict(repeat_penalty=1.1, freq_penalty=0.05, presence_penalty=0.2, penalty_window=4096)], ids=str)
def test_each_is_the_samplers(M, kw):
    vocab, n = 9000, 30
    rng = np.random.default_rng(n)
    s = M.DeviceSampler(vocab, temp=0.0, **kw)
    recent = []
    for _ in range(n):
        x = (3 * rng.standard_normal(vocab)).astype(F)
        window = recent[-kw["penalty_window"]:]
        c = Case(M, 1, vocab, hist=[max(1, len(window))], each=1)
        c.x[0], c.a["hist"] = x, np.array(window or [-1], np.int32)
        for k, name in (("repeat", "repeat_penalty"), ("freq", "freq_penalty"),
                        ("presence", "presence_penalty")):
            c.a[k] = np.array([kw.get(name, 1.0 if k == "repeat" else 0.0)], F)
        got = c.call()[0]
        s.sample(x)                                     # penalises x in place
        assert np.array_equal(got.view(np.uint32), x.view(np.uint32))
        t = int(rng.integers(0, 12))
        s.accept(t)
        recent.append(t)


def test_captured_call_follows_its_inputs(M):
    h = Hip()
    c = Case(M, 4, 20_001, E.BF16, E.F32, hist=[300, 20, 5, 0], bias=[5, 1, 0, 9], masks=3, seed=8)
    a, s = c.args(), h.stream()
    g, e = h.capture(s, lambda: M.logits_dev(a, s))
    for turn in range(4):
        c.x = E.encode(4 * c.rng.standard_normal(c.x.shape), c.t)
        c.a["hist"] = c.rng.integers(0, 50, 325).astype(np.int32)
        c.a["hist_start"] = np.sort(c.rng.integers(0, 326, 5)).astype(np.int64)
        c.a["mask_row"] = c.rng.integers(-1, 3, 4).astype(np.int32)
        for k in ("hist", "hist_start", "mask_row"):
            c.d[k].upload(c.a[k])
        c.d["x"].upload(c.x)
        assert h.lib.hipGraphLaunch(e, C.c_void_p(s)) == 0
        M.check(M.lib.mynah_hip_sync(s), "sync")
        c.check(c.get(), turn)
    h.lib.hipGraphExecDestroy(e)
    h.lib.hipGraphDestroy(g)
    h.lib.hipStreamDestroy(C.c_void_p(s))


def test_offsets_past_32_bits(M):
    """Rows behind 2^32 elements of f16 and masks behind 2^32 bytes."""
    vocab, rows = 151_936, 28_600
    x = M.DeviceBuffer(rows * vocab * 2)
    c = Case(M, 1, vocab, E.F16, E.F16, hist=[40], bias=[6], masks=1, seed=9)
    x.upload(c.x, (rows - 1) * vocab * 2)
    start = lambda s: np.concatenate([np.zeros(rows - 1, np.int64), s])  # noqa: E731
    of, words = np.full(rows, -1, np.int32), -(-vocab // 32)
    many = (1 << 32) // (4 * words) + 5
    masks = M.DeviceBuffer(many * words * 4)
    masks.upload(c.a["allowed"], (many - 1) * words * 4)
    of[-1] = many - 1
    for k in ("hist_start", "bias_start"):
        c.a[k] = start(c.a[k])
    per_row = {k: np.concatenate([np.ones(rows - 1, F), c.a[k]]) for k in ("repeat", "freq", "presence")}
    one = {k: c.a[k] for k in per_row}
    c.a.update(per_row, mask_row=of)
    a = c.args(n_rows=rows, n_masks=many)
    a.x = a.y = x.ptr
    a.allowed = masks.ptr
    M.logits_dev(a)
    M.sync()
    got = x.download(np.float16, vocab, (rows - 1) * vocab * 2).reshape(1, -1)
    c.a.update(one, hist_start=np.array([0, 40]), bias_start=np.array([0, 6]),
               mask_row=np.zeros(1, np.int32))
    c.check(got)
