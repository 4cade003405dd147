"""Calls with more workgroups than one launch counts threads for (2^32 along a
dimension) are refused on the host, before any device work."""
from __future__ import annotations

import ctypes as C

import pytest

import mynah_amd as M
from test_attention_ops import P, QK, ROPE, TREE, error

MOST = (1 << 31) - 1


def far(change):
    v = {**ROPE, "x_token": 128, "y_token": 128, "heads": 1, **change}
    assert M.lib.mynah_hip_rope_dev(*v.values(), None) == -1
    return "too many rows" in error()


def test_rope():
    # 16 heads of 128 a workgroup of 256 threads, 8 of 256
    assert far({"tokens": MOST})
    assert far({"tokens": 1 << 28})
    assert far({"tokens": 1 << 27, "head_dim": 256, "x_token": 256, "y_token": 256})


def test_qk_norm_rope():
    a = M.QkNormRope(**{**QK, "tokens": MOST, "n_heads": 1, "n_kv_heads": 0, "q_stride": 128,
                        "q_out_stride": 128})
    assert M.lib.mynah_hip_qk_norm_rope_dev(C.byref(a), None) == -1
    assert "too many rows" in error()


@pytest.mark.parametrize("change", [
    {"n_kv_heads": 512}, {"n_kv_heads": 256, "type": 0}, {"n_kv_heads": 8, "max_nodes": 65535,
                                                         "mask": None}])
def test_tree_attention(change):
    v = {**TREE, "n_seqs": 65536, "pages": None, "n_rows": 65536, **change}
    kvh = v["n_kv_heads"]
    v.update(n_heads=kvh, slot_stride=128 * kvh, q_stride=128 * kvh, out_stride=128 * kvh)
    a = M.TreeAttention(**v)
    assert M.lib.mynah_hip_tree_attention_dev(C.byref(a), P, 1 << 30, None) == -1
    assert "too many workgroups" in error()
    assert M.lib.mynah_hip_tree_attention_workspace(C.byref(a)) == 0


def test_fp8():
    assert M.lib.mynah_hip_fp8_quantize_dev(0, P, 2048, MOST, 2048, P, P, None) == -1
    assert "too many values" in error()
    assert M.lib.mynah_hip_fp8_matmat_dev(P, P, 1 << 28, 128, P, P, 0, P, 1, None) == -1
    assert "row count" in error()
