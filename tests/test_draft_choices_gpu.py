"""The greedy choices of verified nodes (mynah_hip_qwen3_verify), where no rounding
can turn them: a row of logits is within TOL of the step's in the 2-norm (the bound
of test_draft_gpu.py, which does not look at what verify gives), so a choice is sure
where the step's own two largest logits are more than 2 TOL of that norm apart."""
from __future__ import annotations

import numpy as np
import pytest

from test_draft_gpu import (SHAPE, TOL, M, decoder, model, path_logits, path_to,  # noqa: F401
                            random_tree, rewind)

pytestmark = pytest.mark.gpu


def sure(logits):
    x = np.asarray(logits, np.float64)
    top = np.sort(x, -1)[..., -2:]
    return top[..., 1] - top[..., 0] > 2 * TOL * np.linalg.norm(x, axis=-1)


@pytest.mark.parametrize("past,least", [(16, 20), (300, 15)])
def test_choices_of_a_chain_and_a_tree(M, model, past, least):  # noqa: F811
    rng = np.random.default_rng(past)
    tokens = rng.integers(0, SHAPE.vocab, 40)
    dec = decoder(M, model, past, past + 60)
    steps = path_logits(dec, tokens)
    at = sure(steps)
    print(f"{int(at.sum())} sure choices", flush=True)
    assert at.sum() >= least and len({int(np.argmax(x)) for x, s in zip(steps, at) if s}) > 1
    ids = dec.verify(tokens)
    assert np.array_equal(ids[at], np.argmax(steps, 1)[at])
    parents = random_tree(rng, 40)
    ids, seen = dec.verify(tokens, parents), 0
    for node in range(0, 40, 3):
        path = path_to(parents, node)
        last = path_logits(dec, tokens[path])[-1]
        if sure(last):
            seen += 1
            assert int(ids[node]) == int(np.argmax(last)), path
    assert seen >= 3


def test_drafted_decoding_where_every_choice_is_sure(M, model):  # noqa: F811
    past, steps, first = 16, 40, 205
    dec = decoder(M, model, past, past + steps + 20)
    want, _ = dec.generate(first, steps)
    rewind(dec, past)
    assert sure(path_logits(dec, [first] + want[:-1])).all()
    rng, got, last, calls = np.random.default_rng(2), [], first, 0
    while len(got) < steps:
        guess = (want[len(got):len(got) + int(rng.integers(0, 5))] + [1, 2])[:6]
        wrong = [(g + 1) % SHAPE.vocab for g in guess[:2]]
        tokens = [last] + wrong + guess                 # a wrong branch first
        parents = ([-1] + list(range(len(wrong))) + [0] +
                   list(range(len(wrong) + 1, len(tokens) - 1)))
        ids, path = dec.verify(tokens, parents), [0]
        while True:
            nxt = [i for i in range(len(tokens))
                   if parents[i] == path[-1] and tokens[i] == ids[path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        dec.accept(path)
        got += [int(tokens[i]) for i in path[1:]] + [int(ids[path[-1]])]
        last, calls = got[-1], calls + 1
    assert got[:steps] == want and calls < steps
