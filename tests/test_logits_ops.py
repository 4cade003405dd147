"""The rules on logits on the CPU: every refusal, which comes before any device work;
and the size that a kernel and its host code both state."""
from __future__ import annotations

import ctypes as C
import os
import re

import pytest

import mynah_amd as M
from test_attention_ops import P, error
from test_code_object import ROOT

GOOD = dict(type=30, out_type=0, n_rows=3, vocab=1000, x=P, x_stride=1000, y=P + 4096, y_stride=1000,
            hist=P, hist_start=P, repeat=P, freq=P, presence=P, penalty=0, bias_id=P, bias=P,
            bias_start=P, allowed=P, mask_row=P, mask_words=32, n_masks=2)


@pytest.mark.parametrize("change", [
    {"type": 8}, {"out_type": -1}, {"n_rows": 0}, {"vocab": 0}, {"vocab": 1 << 31}, {"x": None},
    {"y": None}, {"x_stride": 999}, {"y_stride": 999}, {"x_stride": 1 << 62}, {"y": P}, {"penalty": 2},
    {"penalty": -1}, {"type": 0, "y": P, "y_stride": 1004}, {"hist_start": None}, {"bias": None},
    {"bias_start": None}, {"mask_words": 31}, {"mask_words": 0}, {"x": P + 1}, {"y": P + 2},
    {"hist": P + 2}, {"hist_start": P + 4}, {"repeat": P + 1}, {"freq": P + 2}, {"presence": P + 3},
    {"bias_id": P + 2}, {"bias": P + 1}, {"bias_start": P + 4}, {"allowed": P + 2},
    {"mask_row": P + 2}])
def test_refused(change):
    a = M.Logits(**{**GOOD, **change})
    assert M.lib.mynah_hip_logits_dev(C.byref(a), None) == -1
    assert error()
    assert M.lib.mynah_hip_logits_dev(None, None) == -1


def test_too_many_rows():
    a = M.Logits(**{**GOOD, "n_rows": 1 << 23, "vocab": 8193, "x_stride": 8193, "y_stride": 8193,
                    "mask_words": 257})
    assert M.lib.mynah_hip_logits_dev(C.byref(a), None) == -1
    assert "too many rows" in error()


def test_size_stated_twice():
    def value(path, name):
        with open(os.path.join(ROOT, "mynah-slm_amd", "csrc", path)) as f:
            return re.search(rf"#define {name} (\d+)u", f.read()).group(1)
    assert value("runtime_internal.h", "MYNAH_LOGITS_CH") == value("logits.hip", "LG_CH")
