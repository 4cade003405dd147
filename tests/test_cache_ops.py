"""The 8-bit cache's operators on the CPU: every refusal, which comes before any
device work."""
from __future__ import annotations

import ctypes as C
import math
import os
import re

import pytest

import mynah_amd as M
from test_attention_ops import P, error
from test_code_object import ROOT

CACHE = dict(format=0, n_kv_heads=2, head_dim=128, block=32, k=P, v=P, slot_stride=256, n_slots=128,
             k_scale=P, v_scale=P, seq_slots=0, pages=P, page_size=64, max_pages=2)
STORE = dict(type=30, n_seqs=2, k=P, v=P, k_stride=256, v_stride=256, n_rows=6, seq_start=P,
             n_past=P, max_nodes=3, max_kv=128)
ATTN = dict(type=30, n_seqs=2, n_heads=8, q=P, q_stride=1024, out=P, out_stride=1024, n_rows=6,
            seq_start=P, n_past=P, mask=P, mask_words=1, max_nodes=3, max_kv=128, scale=0.1)

BAD_CACHE = [
    {"format": 2}, {"format": -1}, {"n_kv_heads": 0}, {"head_dim": 96}, {"head_dim": 0}, {"block": 0},
    {"block": 8}, {"block": 48}, {"block": 512}, {"k": None}, {"v": None}, {"k_scale": None},
    {"v_scale": None}, {"slot_stride": 240}, {"slot_stride": 264}, {"slot_stride": 1 << 24},
    {"n_slots": 0}, {"n_slots": 100}, {"n_slots": (1 << 40) + 32}, {"pages": None, "seq_slots": 40},
    {"pages": None, "seq_slots": 1 << 40}, {"page_size": 16}, {"page_size": 0}, {"page_size": 96},
    {"max_pages": 1}, {"k": P + 8}, {"v": P + 4}, {"k_scale": P + 2}, {"pages": P + 2}]


def refused_store(cache={}, **change):
    a = M.Kv8Store(cache=M.Kv8Cache(**{**CACHE, **cache}), **{**STORE, **change})
    assert M.lib.mynah_hip_kv8_store_dev(C.byref(a), None) == -1
    return error()


def refused_attn(cache={}, **change):
    a = M.Kv8Attention(cache=M.Kv8Cache(**{**CACHE, **cache}), **{**ATTN, **change})
    assert M.lib.mynah_hip_kv8_attention_dev(C.byref(a), P, 1 << 30, None) == -1
    why = error()
    assert M.lib.mynah_hip_kv8_attention_workspace(C.byref(a)) == 0
    return why


@pytest.mark.parametrize("change", BAD_CACHE)
def test_cache_refused(change):
    assert refused_store(change) and refused_attn(change)


@pytest.mark.parametrize("change", [
    {"type": 8}, {"k": None}, {"v": None}, {"seq_start": None}, {"n_past": None}, {"n_seqs": 0},
    {"n_seqs": 65537}, {"n_rows": 0}, {"n_rows": 1 << 31}, {"max_nodes": 0},
    {"max_nodes": (1 << 24) + 1}, {"max_kv": 0}, {"max_kv": (1 << 26) + 1}, {"max_kv": 129},
    {"k_stride": 255}, {"v_stride": 128}, {"k_stride": 260}, {"k_stride": 1 << 62}, {"k": P + 8},
    {"v": P + 2}, {"n_past": P + 2}, {"seq_start": P + 1}])
def test_store_refused(change):
    assert refused_store(**change)
    assert M.lib.mynah_hip_kv8_store_dev(None, None) == -1


@pytest.mark.parametrize("change", [
    {"type": 8}, {"q": None}, {"out": None}, {"seq_start": None}, {"n_past": None}, {"n_heads": 0},
    {"n_heads": 7}, {"n_heads": 130}, {"n_seqs": 0}, {"n_rows": 0}, {"n_rows": 1 << 31},
    {"max_nodes": 0}, {"max_nodes": 65536, "mask": None}, {"max_kv": 0}, {"max_kv": (1 << 26) + 1},
    {"max_kv": 129}, {"mask_words": 0}, {"max_nodes": 33}, {"q_stride": 1000}, {"out_stride": 512},
    {"q": P + 8}, {"out": P + 2}, {"q_stride": 1028}, {"mask": P + 2}, {"scale": math.nan},
    {"scale": math.inf}, {"q_stride": 1 << 61}, {"n_rows": 1 << 30, "mask_words": 8,
                                                 "q_stride": 1024}])
def test_attention_refused(change):
    assert refused_attn(**change)


def test_attention_workspace_refused():
    a = M.Kv8Attention(cache=M.Kv8Cache(**CACHE), **ATTN)
    assert M.lib.mynah_hip_kv8_attention_dev(C.byref(a), None, 1 << 30, None) == -1
    assert M.lib.mynah_hip_kv8_attention_dev(C.byref(a), P + 16, 1 << 30, None) == -1
    assert "workspace" in error()
    assert M.lib.mynah_hip_kv8_attention_dev(None, P, 1 << 30, None) == -1
    assert M.lib.mynah_hip_kv8_attention_workspace(None) == 0


def test_launches_too_large():
    assert "too many blocks" in refused_store(
        {"pages": None, "seq_slots": 128, "n_kv_heads": 512, "slot_stride": 65536}, n_seqs=65536,
        k_stride=65536, v_stride=65536)
    assert "too many workgroups" in refused_attn(
        {"pages": None, "seq_slots": 128, "n_kv_heads": 512, "slot_stride": 65536}, n_seqs=65536,
        n_heads=512, q_stride=65536, out_stride=65536)


# ── pages ────────────────────────────────────────────────────────────────────

POOL = dict(n_pages=8, n_seqs=3, max_pages=4, page_size=16, n_parts=2, parts=P, refs=P, pages=P,
            n_past=P, status=P)
BIG = 1 << 30


@pytest.mark.parametrize("change", [
    {"n_pages": 0}, {"n_pages": 1 << 28}, {"n_seqs": 0}, {"n_seqs": 65537}, {"max_pages": 0},
    {"max_pages": 1 << 27}, {"page_size": 0}, {"page_size": 24}, {"n_parts": 0}, {"n_parts": 65535},
    {"parts": None}, {"refs": None}, {"pages": None}, {"n_past": None}, {"status": None},
    {"parts": P + 4}, {"refs": P + 2}, {"status": P + 1}])
def test_pool_refused(change):
    a = C.byref(M.PagePool(**{**POOL, **change}))
    lib = M.lib
    assert lib.mynah_hip_pages_workspace(a) == 0 and error()
    assert lib.mynah_hip_pages_fork_dev(a, P, P, BIG, None) == -1
    assert lib.mynah_hip_pages_reserve_dev(a, P, P, BIG, None) == -1
    assert lib.mynah_hip_pages_release_dev(a, P, None) == -1
    assert lib.mynah_hip_pages_compact_dev(a, P, BIG, None) == -1
    assert lib.mynah_hip_pages_copy_dev(a, P, P, 1, None) == -1


def test_pool_arguments_refused():
    a, lib = C.byref(M.PagePool(**POOL)), M.lib
    need = lib.mynah_hip_pages_workspace(a)
    assert need >= 4 * (3 * 5 + 6 * 8 + 1)
    for x in (None, P + 2):
        assert lib.mynah_hip_pages_fork_dev(a, x, P, BIG, None) == -1
        assert lib.mynah_hip_pages_reserve_dev(a, x, P, BIG, None) == -1
        assert lib.mynah_hip_pages_release_dev(a, x, None) == -1
        assert lib.mynah_hip_pages_copy_dev(a, x, P, 1, None) == -1
        assert lib.mynah_hip_pages_copy_dev(a, P, x, 1, None) == -1
    assert lib.mynah_hip_pages_copy_dev(a, P, P, 0, None) == -1
    for ws, n in ((None, need), (P + 16, need), (P, need - 1)):
        assert lib.mynah_hip_pages_fork_dev(a, P, ws, n, None) == -1 and "workspace" in error()
        assert lib.mynah_hip_pages_reserve_dev(a, P, ws, n, None) == -1
        assert lib.mynah_hip_pages_compact_dev(a, ws, n, None) == -1
    assert lib.mynah_hip_pages_workspace(None) == 0


# ── sizes that a kernel and its host code both state ─────────────────────────

@pytest.mark.parametrize("host,host_name,source,kernel", [
    ("kv8.c", r"#define KV8_WAVES (\d+)u", "kv8.hip", r"struct Kv8Shape \{.*?int W = (\d+);"),
    ("kv8.c", r"#define KV8_WIDE_WAVES (\d+)u", "kv8.hip", r"struct Kv8Wide \{.*?int W = (\d+);"),
    ("pages.c", r"#define PAGES_FORK (\d+)u", "pages.hip", r"#define PG_FORK (\d+)u")])
def test_sizes_stated_twice_agree(host, host_name, source, kernel):
    def value(path, pattern):
        with open(os.path.join(ROOT, "mynah-slm_amd", "csrc", path)) as f:
            return re.search(pattern, f.read(), re.S).group(1)
    assert value(host, host_name) == value(source, kernel)
