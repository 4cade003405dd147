"""The attention's operators (include/mynah_attention.h) and the 8-bit floating
point product on the CPU: the rotary frequency table against the formulas, and
every refusal, which comes before any device work."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

import elem_lib as E
import mynah_amd as M

BUF = np.zeros(4096, np.uint64)          # never read: every call here is refused
P = (M.ptr(BUF) + 255) & ~255


def error():
    return M.lib.mynah_hip_last_error().decode()


# ── frequencies ──────────────────────────────────────────────────────────────

def formula(rot, theta, scaling, factor, trained, high, low):
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == M.ROPE_LINEAR:
        return [x / factor for x in f]
    if scaling == M.ROPE_YARN:
        def pair(turns):
            return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))
        a, b = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rot - 1)
        g = [min(max((i - a) / max(b - a, 0.001), 0.0), 1.0) for i in range(rot // 2)]
        return [x / factor * y + x * (1 - y) for x, y in zip(f, g)]
    if scaling == M.ROPE_BANDS:
        g = [min(max((trained * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
        return [x / factor * (1 - y) + x * y for x, y in zip(f, g)]
    return f


@pytest.mark.parametrize("rot,theta", [(128, 1e6), (64, 1e4), (8, 5e5), (2, 1e4), (512, 1e7)])
@pytest.mark.parametrize("scaling,high,low", [(0, 0, 0), (1, 0, 0), (2, 32.0, 1.0), (3, 4.0, 1.0),
                                              (2, 8.0, 0.5)])
def test_frequencies(rot, theta, scaling, high, low):
    got, m = M.rope_freqs(rot, theta, scaling, 4.0, 32768.0, high, low)
    want = formula(rot, theta, scaling, 4.0, 32768.0, high, low)
    # a few roundings of 2^-53, pow's and the ramp's included
    np.testing.assert_allclose(got, want, rtol=1e-14)
    assert m == np.float32(0.1 * math.log(4.0) + 1.0 if scaling == M.ROPE_YARN else 1.0)


def test_mscale():
    assert M.rope_freqs(64, 1e4, mscale=0.5)[1] == 0.5
    assert M.rope_freqs(64, 1e4, M.ROPE_YARN, 8.0, 4096.0, 32.0, 1.0, mscale=1.25)[1] == 1.25
    assert M.rope_freqs(64, 1e4, M.ROPE_YARN, 0.5, 4096.0, 32.0, 1.0)[1] == 1.0


@pytest.mark.parametrize("change", [
    {"rot_dim": 0}, {"rot_dim": 7}, {"theta": 1.0}, {"theta": math.nan}, {"theta": math.inf},
    {"scaling": 4}, {"scaling": -1}, {"factor": 0.0}, {"factor": math.nan}, {"trained": 0.0},
    {"low": 0.0}, {"high": 1.0}, {"high": math.inf}, {"mscale": -1.0}, {"mscale": math.nan}])
def test_frequencies_refused(change):
    v = {"rot_dim": 64, "scaling": M.ROPE_YARN, "theta": 1e4, "factor": 4.0, "trained": 4096.0,
         "high": 32.0, "low": 1.0, "mscale": 0.0, **change}
    p, out, m = M.RopeParams(**v), (C.c_double * 64)(), C.c_float()
    assert M.lib.mynah_hip_rope_freqs(C.byref(p), out, C.byref(m)) == -1
    assert "rope" in error()


def test_frequencies_null():
    p, out, m = M.RopeParams(64, 0, 1e4), (C.c_double * 64)(), C.c_float()
    assert M.lib.mynah_hip_rope_freqs(None, out, C.byref(m)) == -1
    assert M.lib.mynah_hip_rope_freqs(C.byref(p), None, C.byref(m)) == -1
    assert M.lib.mynah_hip_rope_freqs(C.byref(p), out, None) == -1


# ── refusals ─────────────────────────────────────────────────────────────────

ROPE = dict(type=0, layout=0, x=P, x_token=1024, x_head=128, y=P, y_token=1024, y_head=128,
            tokens=3, heads=8, head_dim=128, rot_dim=128, freqs=P, mscale=1.0, pos=P)


@pytest.mark.parametrize("change", [
    {"type": 2}, {"type": -1}, {"layout": 2}, {"layout": -1}, {"x": None}, {"y": None},
    {"freqs": None}, {"tokens": 0}, {"heads": 0}, {"heads": 65537}, {"tokens": 1 << 31},
    {"head_dim": 0}, {"head_dim": 12}, {"head_dim": 520}, {"rot_dim": 0}, {"rot_dim": 4},
    {"rot_dim": 136}, {"x": P + 2}, {"type": 1, "y": P + 1}, {"freqs": P + 4}, {"pos": P + 2},
    {"x_token": 1 << 62}, {"y_head": 1 << 61}])
def test_rope_refused(change):
    v = {**ROPE, **change}
    assert M.lib.mynah_hip_rope_dev(*v.values(), None) == -1
    assert error()


QK = dict(type=0, out_type=30, layout=0, n_heads=8, n_kv_heads=2, head_dim=128, rot_dim=64,
          tokens=5, q=P, k=P, v=P, q_stride=1536, k_stride=1536, v_stride=1536, q_norm=P, k_norm=P,
          eps=1e-6, mscale=1.0, freqs=P, pos=P, slots=P, n_slots=16, q_out=P, q_out_stride=1024,
          k_cache=P, v_cache=P, slot_stride=256)


@pytest.mark.parametrize("change", [
    {"type": 3}, {"out_type": 8}, {"layout": 5}, {"n_heads": 0, "n_kv_heads": 0}, {"head_dim": 100},
    {"rot_dim": 200}, {"tokens": 0}, {"q": None}, {"q_out": None}, {"k": None}, {"k_cache": None},
    {"v_cache": None}, {"freqs": None}, {"n_slots": 0}, {"n_slots": 1 << 31}, {"eps": -1.0},
    {"eps": math.nan}, {"q": P + 2}, {"q_out": P + 1}, {"k_cache": P + 1}, {"v": P + 1},
    {"q_norm": P + 2}, {"slots": P + 1}, {"pos": P + 2}, {"slot_stride": 1 << 61},
    {"q_stride": 1 << 62}])
def test_qk_norm_rope_refused(change):
    a = M.QkNormRope(**{**QK, **change})
    assert M.lib.mynah_hip_qk_norm_rope_dev(C.byref(a), None) == -1
    assert error()
    assert M.lib.mynah_hip_qk_norm_rope_dev(None, None) == -1


TREE = dict(type=30, n_seqs=2, n_heads=8, n_kv_heads=2, head_dim=128, q=P, q_stride=1024, out=P,
            out_stride=1024, n_rows=6, k_cache=P, v_cache=P, slot_stride=256, n_slots=64,
            seq_slots=0, pages=P, page_size=16, max_pages=2, seq_start=P, n_past=P, mask=P,
            mask_words=1, max_nodes=3, max_kv=32, scale=0.1)


@pytest.mark.parametrize("change", [
    {"type": 8}, {"q": None}, {"out": None}, {"k_cache": None}, {"v_cache": None},
    {"seq_start": None}, {"n_past": None}, {"head_dim": 96}, {"head_dim": 0}, {"n_heads": 0},
    {"n_kv_heads": 0}, {"n_heads": 7}, {"n_heads": 130}, {"n_seqs": 0}, {"n_rows": 0},
    {"n_rows": 1 << 31, "mask_words": 2}, {"max_nodes": 0}, {"max_nodes": 65536, "mask": None}, {"max_kv": 0}, {"max_kv": (1 << 26) + 1},
    {"n_slots": 0}, {"mask_words": 0}, {"max_nodes": 33}, {"page_size": 8}, {"page_size": 24},
    {"page_size": 0}, {"max_kv": 33}, {"pages": None, "seq_slots": 1 << 40}, {"q_stride": 1000},
    {"out_stride": 512}, {"slot_stride": 128}, {"slot_stride": (1 << 24) + 8}, {"q": P + 8},
    {"k_cache": P + 8}, {"q_stride": 1028}, {"slot_stride": 260}, {"mask": P + 2},
    {"scale": math.nan}, {"scale": math.inf}, {"q_stride": 1 << 61}])
def test_tree_attention_refused(change):
    a = M.TreeAttention(**{**TREE, **change})
    assert M.lib.mynah_hip_tree_attention_dev(C.byref(a), P, 1 << 30, None) == -1
    assert error()
    assert M.lib.mynah_hip_tree_attention_workspace(C.byref(a)) == 0


def test_tree_attention_workspace_refused():
    a = M.TreeAttention(**TREE)
    assert M.lib.mynah_hip_tree_attention_dev(C.byref(a), None, 1 << 30, None) == -1
    assert M.lib.mynah_hip_tree_attention_dev(C.byref(a), P + 16, 1 << 30, None) == -1
    assert "workspace" in error()
    assert M.lib.mynah_hip_tree_attention_dev(None, P, 1 << 30, None) == -1
    assert M.lib.mynah_hip_tree_attention_workspace(None) == 0


@pytest.mark.parametrize("change", [
    {"type": 12}, {"x": None}, {"xq": None}, {"xs": None}, {"tokens": 0}, {"cols": 0},
    {"cols": 24}, {"x_stride": 240}, {"x": P + 8}, {"xq": P + 8}, {"xs": P + 2},
    {"x_stride": 258}, {"tokens": 1 << 31}])
def test_fp8_quantize_refused(change):
    v = dict(type=0, x=P, x_stride=256, tokens=3, cols=256, xq=P, xs=P)
    assert M.lib.mynah_hip_fp8_quantize_dev(*{**v, **change}.values(), None) == -1
    assert error()


@pytest.mark.parametrize("change", [
    {"w": None}, {"ws": None}, {"xq": None}, {"xs": None}, {"y": None}, {"rows": 0}, {"cols": 0},
    {"cols": 100}, {"tokens": 0}, {"type": 3}, {"w": P + 8}, {"xq": P + 4}, {"ws": P + 2},
    {"xs": P + 1}, {"y": P + 2}, {"rows": 1 << 31}, {"cols": 1 << 31}, {"tokens": 1 << 31}])
def test_fp8_matmat_refused(change):
    v = dict(w=P, ws=P, rows=100, cols=256, xq=P, xs=P, type=0, y=P, tokens=3)
    assert M.lib.mynah_hip_fp8_matmat_dev(*{**v, **change}.values(), None) == -1
    assert error()


def test_element_types():
    # The tests' own encodings: every code back from its value, ties to even.
    c = np.array([k for k in range(256) if k & 127 != 127], np.uint8)
    assert np.array_equal(E.to_e4m3(E.E4M3[c]), c)
    assert list(E.to_e4m3(np.array([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 455.0]))) == \
        list(E.to_e4m3(np.array([16.0, 20.0, 0.0, 2.0 ** -8, 448.0])))
    x = np.array([1.0, -2.5, 1.00390625, 1.01171875, np.inf], np.float32)
    assert list(E.decode(E.encode(x, E.BF16), E.BF16)) == [1.0, -2.5, 1.0, 1.015625, np.inf]


# ── the decoder's paths ──────────────────────────────────────────────────────

def test_decoder_without_a_state():
    t = np.zeros(4, np.uint32)
    assert M.lib.mynah_hip_qwen3_verify(None, M.ptr(t), None, 4, M.ptr(t), None) == -1
    assert "verify" in error()
    assert M.lib.mynah_hip_qwen3_accept(None, M.ptr(t), 4) == -1 and "accept" in error()
    assert M.lib.mynah_hip_qwen3_drop(None, 0, 0) == -1 and "drop" in error()
