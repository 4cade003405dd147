"""What the 8-bit cache's store refuses beside its arguments one by one: sequences
whose rows would meet. On the CPU, ahead of any device work."""
from __future__ import annotations

import ctypes as C

import pytest

import mynah_amd as M
from test_attention_ops import error
from test_cache_ops import ATTN, CACHE, STORE, refused_store


@pytest.mark.parametrize("seq_slots,max_kv", [(0, 1), (0, 128), (64, 65), (96, 128)])
def test_sequences_that_would_meet(seq_slots, max_kv):
    """Without pages a sequence may not grow into the next one's rows."""
    cache = {"pages": None, "seq_slots": seq_slots}
    assert "seq_slots" in refused_store(cache, max_kv=max_kv)


@pytest.mark.parametrize("cache,change", [
    ({"pages": None, "seq_slots": 64}, {"max_kv": 64}),
    ({"pages": None, "seq_slots": 0}, {"n_seqs": 1}), ({"seq_slots": 0}, {})])
def test_sequences_that_do_not(cache, change):
    a = M.Kv8Store(cache=M.Kv8Cache(**{**CACHE, **cache}), **{**STORE, **change, "k_stride": 255})
    assert M.lib.mynah_hip_kv8_store_dev(C.byref(a), None) == -1
    assert "stride" in error()                          # what is looked at next


def test_attention_shares_rows():
    cache = M.Kv8Cache(**{**CACHE, "pages": None, "seq_slots": 0})
    a = M.Kv8Attention(cache=cache, **{**ATTN, "q_stride": 1000})
    assert M.lib.mynah_hip_kv8_attention_dev(C.byref(a), None, 0, None) == -1
    assert "stride" in error()
