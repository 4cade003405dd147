"""Verification of drafted tokens by the decoder (mynah_hip_qwen3_verify, _accept,
_drop) against its own single steps.

A verified node's logits differ from a step's by f32 rounding in the attention
and the rotation alone; the products and norms run in the step's order. How far that
may go, u = 2^-24: a score is 128 products of heads whose norms make |q| |k| <= 128
(weights about 1), times 128^-0.5, so each side's is off by up to 132 u 128^0.5 =
1493 u, a probability by twice that (the sum's share), and the attention's output, and
with it what the layer adds, by 4 * 1493 u = 3.6e-4 of itself between the two sides. Norms
keep a relative error, so three layers add up to 1.1e-3 of x. A random matrix with r
rows over 512 columns makes of that at most (r^0.5 + 512^0.5) / r^0.5 times as much of
its product's norm: 1.4 for the 4096 logits, 2.4 for a row of 256 keys or values.
So per row |got - want| <= 3e-3 |want| in the 2-norm. (A bound of 1e-4 a logit,
which the split attention's tests hold over random cached rows, holds no such proof:
with the nodes' few own keys alone 1.2e-4 was seen, 11 u of x.) A wrong position, parent
or row is off by a good part of |want|."""
from __future__ import annotations

import numpy as np
import pytest

import configs as CF
import elem_lib as E
import oracle_lib as O

pytestmark = pytest.mark.gpu
TOL = 3e-3
SHAPE = CF.QWEN3_TINY


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    mynah_amd.check(mynah_amd.lib.mynah_hip_set_gemv_order(0), "order")
    return mynah_amd


@pytest.fixture(scope="module")
def model(M):
    return M.SynthQwen3(SHAPE, 0)


def decoder(M, model, past, n_ctx, shape=SHAPE):
    print(f"[case] draft past={past} n_ctx={n_ctx}", flush=True)
    dec = M.Qwen3Decoder(model, n_ctx)
    if past:
        k, v = O.kv_prefill(O.substream, shape, 0, past)
        dec.set_kv(k, v, past)
    return dec


def off(got, want):
    """The largest 2-norm of a row's difference, relative to the row's."""
    d = np.linalg.norm(got.astype(np.float64) - want, axis=-1)
    return float(np.max(d / np.linalg.norm(want.astype(np.float64), axis=-1)))


def rewind(dec, past):
    dec.drop(past, dec.n_past - past)


def path_logits(dec, tokens):
    """Logits of single steps along `tokens`; the position is taken back."""
    past = dec.n_past
    out = [dec.forward(int(t)) for t in tokens]
    rewind(dec, past)
    return out


@pytest.mark.parametrize("past", [0, 1, 16, 700])
@pytest.mark.parametrize("n", [1, 2, 33])
def test_chain(M, model, past, n):
    dec = decoder(M, model, past, past + n + 2)
    tokens = np.random.default_rng(n).integers(0, SHAPE.vocab, n)
    want = path_logits(dec, tokens)
    ids, got = dec.verify(tokens, want_logits=True)
    assert dec.n_past == past
    for i in range(n):
        assert off(got[i], want[i]) <= TOL, i
        assert int(ids[i]) == int(np.argmax(got[i]))
    dec.accept(np.arange(n))
    assert dec.n_past == past + n
    k, v = dec.get_kv(past + n)
    one = decoder(M, model, past, past + n + 2)
    for t in tokens:
        one.forward(int(t), want_logits=False)
    kk, vv = one.get_kv(past + n)
    assert np.array_equal(k[:, :past], kk[:, :past]) and np.array_equal(v[:, :past], vv[:, :past])
    assert off(k, kk) <= TOL and off(v, vv) <= TOL
    assert off(dec.forward(3), one.forward(3)) <= TOL


def random_tree(rng, n):
    return np.array([-1 if i == 0 else int(rng.integers(-1, i)) for i in range(n)], np.int32)


def path_to(parents, node):
    p = []
    while node >= 0:
        p.append(int(node))
        node = parents[node]
    return p[::-1]


@pytest.mark.parametrize("past,n", [(0, 7), (40, 24), (700, 70), (5, 256)])
def test_tree(M, model, past, n):
    rng = np.random.default_rng(past + n)
    dec = decoder(M, model, past, past + n + 1)
    tokens, parents = rng.integers(0, SHAPE.vocab, n), random_tree(rng, n)
    _, got = dec.verify(tokens, parents, want_logits=True)
    # A path that is no prefix of the rows, the longest one and two others.
    paths = sorted((path_to(parents, i) for i in range(n)), key=len)
    paths = [paths[-1], paths[len(paths) // 2], path_to(parents, n - 1)]
    for p in paths:
        for node, want in zip(p, path_logits(dec, tokens[p])):
            assert off(got[node], want) <= TOL, (p, node)
    for p in paths:
        # the steps above wrote the rows behind the position: the nodes are gone
        with pytest.raises(M.HipError):
            dec.accept(p)
        ids = dec.verify(tokens, parents)
        assert np.array_equal(ids, np.argmax(got, 1))
        dec.accept(p)
        assert dec.n_past == past + len(p)
        k, v = dec.get_kv(dec.n_past)
        rewind(dec, past)
        for t in tokens[p]:
            dec.forward(int(t), want_logits=False)
        kk, vv = dec.get_kv(dec.n_past)
        assert off(k, kk) <= TOL and off(v, vv) <= TOL
        rewind(dec, past)


def test_committed_rows_and_later_steps_keep_their_bits(M, model):
    past = 50
    a, b = decoder(M, model, past, 90), decoder(M, model, past, 90)
    before = a.get_kv(past)
    a.verify(np.arange(9), [-1, 0, 0, 1, 1, 2, -1, 6, 6])
    assert all(np.array_equal(x, y) for x, y in zip(before, a.get_kv(past)))
    a.verify([5, 6, 7])                                 # the same rows again
    a.accept([])                                        # nothing of it
    assert a.n_past == past
    for t in (4, 9, 2):
        assert np.array_equal(a.forward(t).view(np.uint32), b.forward(t).view(np.uint32))


def test_drafted_decoding_gives_the_greedy_tokens(M, model):
    """Draft trees whose first branch is right for a while and then wrong: the
    accepted tokens are those of the greedy loop."""
    past, steps, first = 16, 40, 3
    dec = decoder(M, model, past, past + steps + 20)
    want, _ = dec.generate(first, steps)
    rewind(dec, past)
    logits = path_logits(dec, [first] + want[:-1])
    # up to the first choice that hangs on a rounding: 8 times what a chain of the
    # same tokens differs by
    _, chain = dec.verify([first] + want[:-1], want_logits=True)
    err = max(float(np.abs(a - b).max()) for a, b in zip(chain, logits))
    margin = [float(np.diff(np.sort(x)[-2:])[0]) for x in logits]
    sure = next((i for i, m in enumerate(margin) if m <= 8 * err), steps)
    print(f"largest difference {err:.2e}, {sure} sure choices", flush=True)
    rng, got, last, calls = np.random.default_rng(1), [], first, 0
    while len(got) < steps:
        good = int(rng.integers(0, 5))
        guess = (want[len(got):len(got) + good] + [1, 2])[:6]
        wrong = [(g + 1) % SHAPE.vocab for g in guess]
        tokens = [last] + wrong[:2] + guess             # a wrong branch first
        parents = [-1, 0, 1] + [0] + list(range(3, 2 + len(guess)))
        tokens, parents = tokens[:3 + len(guess)], parents[:3 + len(guess)]
        ids = dec.verify(tokens, parents)
        calls += 1
        path = [0]
        while True:
            nxt = [i for i in range(len(tokens))
                   if parents[i] == path[-1] and tokens[i] == ids[path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        dec.accept(path)
        got += [int(tokens[i]) for i in path[1:]] + [int(ids[path[-1]])]
        last = got[-1]
    assert got[:sure] == want[:sure] and calls < steps


def test_drop_moves_and_turns_back(M, model):
    """Values keep their bits; a key row is itself turned back by n positions,
    within f32 rounding of the rotation (6 u of the pair) and of the result."""
    past, first, n = 61, 7, 13
    dec = decoder(M, model, past, 80)
    k, v = dec.get_kv(past)
    dec.drop(first, n)
    assert dec.n_past == past - n
    kk, vv = dec.get_kv(past - n)
    rest = list(range(first)) + list(range(first + n, past))
    assert np.array_equal(vv, v[:, rest]) and np.array_equal(kk[:, :first], k[:, :first])
    hd = SHAPE.head_dim
    freqs, _ = M.rope_freqs(hd, SHAPE.rope_theta)
    x = k[:, first + n:].reshape(SHAPE.n_layers, -1, SHAPE.n_kv_heads, 2, hd // 2).astype(np.float64)
    c, s = np.cos(-n * freqs), np.sin(-n * freqs)
    want = np.stack([x[..., 0, :] * c - x[..., 1, :] * s, x[..., 0, :] * s + x[..., 1, :] * c], -2)
    size = np.abs(x).sum(-2, keepdims=True)
    got = kk[:, first:].reshape(want.shape)
    assert np.all(np.abs(got - want) <= 6 * E.U * size + E.U * np.abs(want))


@pytest.mark.parametrize("n", [1, 40])
def test_drop_from_the_front_is_a_shorter_prompt(M, model, n):
    """The first layer's keys and values depend on token and position alone: with
    the front dropped they are those of the rest at its own start."""
    tokens = np.random.default_rng(n).integers(0, SHAPE.vocab, 75)
    a, b = M.Qwen3Decoder(model, 80), M.Qwen3Decoder(model, 80)
    a.prefill(tokens)
    a.drop(0, n)
    b.prefill(tokens[n:])
    (ka, va), (kb, vb) = a.get_kv(75 - n), b.get_kv(75 - n)
    assert np.array_equal(va[0], vb[0])
    # three rotations' roundings (there, back, and the other's)
    assert np.all(np.abs(ka[0] - kb[0]) <= 3 * 8 * E.U * 2 * np.abs(kb).max())
    a.forward(5), b.forward(5)


def test_drop_at_the_end_is_an_undo(M, model):
    dec = decoder(M, model, 20, 40)
    a = dec.forward(7)
    dec.forward(8, want_logits=False)
    dec.drop(20, 2)
    assert np.array_equal(a.view(np.uint32), dec.forward(7).view(np.uint32))
    dec.drop(0, 21)
    assert dec.n_past == 0
    dec.drop(0, 0)


@pytest.mark.parametrize("mode", ["ATTN_EXACT", "ATTN_SPLIT"])
@pytest.mark.parametrize("late,early", [(100, 50), (600, 3)])
def test_steps_captured_late_run_early(M, model, mode, late, early):
    # A step's graph that was captured further on runs again after a drop.
    a, b = decoder(M, model, late, late + 20), decoder(M, model, early, late + 20)
    for dec in (a, b):
        dec.set_attention(getattr(M, mode))
    a.generate(3, 9)
    a.verify([1, 2, 3])
    a.drop(early, a.n_past - early)
    k, v = O.kv_prefill(O.substream, SHAPE, 0, early)
    a.set_kv(k, v, early)
    for t in (5, 6):
        assert np.array_equal(a.forward(t).view(np.uint32), b.forward(t).view(np.uint32))


def test_drop_of_more_rows_than_move_at_a_time(M, model):
    past, n = 9001, 2
    dec = decoder(M, model, past, 9010)
    _, v = dec.get_kv(past)
    dec.drop(1, n)
    k2, v2 = dec.get_kv(past - n)
    assert np.array_equal(v2, np.delete(v, [1, 2], 1)) and np.isfinite(k2).all()


def test_refusals(M, model):
    dec = decoder(M, model, 10, 14)
    v = SHAPE.vocab
    for tokens, parents in (([], None), ([1] * 257, None), ([1] * 5, None), ([v], None),
                            ([1, 2], [-1, 1]), ([1, 2], [0, 0]), ([1, 2], [-1, -2])):
        with pytest.raises(M.HipError):
            dec.verify(tokens, parents)
    with pytest.raises(ValueError):
        dec.verify([1, 2], [-1])
    with pytest.raises(M.HipError):
        dec.accept([0])                                 # nothing waits
    dec.verify([1, 2, 3], [-1, 0, 0])
    for path in ([1], [0, 0], [0, 1, 2], [0, 3], [0, 2, 1]):
        with pytest.raises(M.HipError):
            dec.accept(path)
    assert dec.n_past == 10
    dec.accept([0, 2])                                  # a refused path changed nothing
    assert dec.n_past == 12
    with pytest.raises(M.HipError):
        dec.accept([0])                                 # they are kept already
    for write in (lambda: dec.forward(1), lambda: dec.prefill([1]), lambda: dec.drop(0, 0),
                  dec.reset):
        dec.verify([1])
        write()
        with pytest.raises(M.HipError):
            dec.accept([0])
        dec.reset()
    dec.prefill([1, 2, 3])
    for first, n in ((0, 4), (4, 0), (3, 1), (2, 2), (1, (1 << 32) - 1)):
        with pytest.raises(M.HipError):
            dec.drop(first, n)
    assert dec.n_past == 3


def test_two_decoders(M, model):
    a, b = decoder(M, model, 30, 60), decoder(M, model, 8, 60)
    want = a.verify([1, 2, 3]).tolist(), b.verify([4, 5]).tolist()
    b.accept([0])
    a.accept([0, 1])
    rewind(a, 30), rewind(b, 8)
    assert (a.verify([1, 2, 3]).tolist(), b.verify([4, 5]).tolist()) == want
