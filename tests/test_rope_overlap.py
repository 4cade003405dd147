"""Rotary calls whose output rows would overlap are refused, others not, before any
device work: every call here has positions off their alignment, which is looked at
after the strides, so none goes further."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import mynah_amd as M
from test_attention_ops import P, QK, ROPE, error


def meets(tokens, token, heads, head, n):
    at = (np.arange(tokens)[:, None] * token + np.arange(heads) * head).ravel()
    at.sort()
    return len(at) > 1 and int(np.diff(at).min()) < n


def rope(**change):
    # pos off its alignment: refused in any case, after the strides
    v = {**ROPE, "pos": P + 2, **change}
    assert M.lib.mynah_hip_rope_dev(*v.values(), None) == -1
    return "overlap" in error()


@pytest.mark.parametrize("tokens,token,heads,head", [
    (3, 1024, 8, 128), (3, 1023, 8, 128), (3, 128, 8, 384), (3, 128, 8, 383), (1, 0, 8, 128),
    (1, 0, 8, 127), (5, 128, 1, 0), (5, 127, 1, 0), (2, 128, 2, 128), (2, 0, 2, 128),
    (2, 384, 2, 256), (3, 256, 2, 384), (4, 256, 2, 384), (3, 300, 3, 500), (3, 300, 3, 450),
    (1, 0, 1, 0), (7, 130, 5, 1100), (9, 130, 9, 1100)])
def test_rope_rows(tokens, token, heads, head):
    got = rope(tokens=tokens, y_token=token, heads=heads, y_head=head)
    assert got == meets(tokens, token, heads, head, 128)


def test_rope_rows_at_random():
    rng = np.random.default_rng(0)
    seen = set()
    for _ in range(4000):
        tokens, heads = (int(v) for v in rng.integers(1, 12, 2))
        token, head = (int(v) for v in rng.choice([0, 60, 64, 65, 128, 190, 192, 200, 384, 700], 2))
        want = meets(tokens, token, heads, head, 64)
        seen.add(want)
        assert rope(tokens=tokens, y_token=token, heads=heads, y_head=head, head_dim=64,
                    rot_dim=64) == want, (tokens, token, heads, head)
    assert len(seen) == 2


def test_inputs_may_share_rows():
    assert not rope(x_token=0)
    assert not rope(x_head=0, x_token=8)


@pytest.mark.parametrize("change,want", [
    ({}, False), ({"q_out_stride": 1023}, True), ({"q_out_stride": 1023, "tokens": 1}, False),
    ({"slot_stride": 255}, True), ({"slot_stride": 0}, True),
    ({"slot_stride": 0, "n_slots": 1}, False), ({"slot_stride": 255, "n_kv_heads": 0}, False),
    ({"q_out_stride": 0, "n_heads": 0}, False), ({"q_stride": 0, "k_stride": 8}, False),
    ({"q_out_stride": 4096, "slot_stride": 512}, False)])
def test_qk_norm_rope_rows(change, want):
    a = M.QkNormRope(**{**QK, "pos": P + 2, **change})
    assert M.lib.mynah_hip_qk_norm_rope_dev(C.byref(a), None) == -1
    assert ("overlap" in error()) == want
