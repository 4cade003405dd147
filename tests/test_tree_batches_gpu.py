"""Tree attention (mynah_hip_tree_attention_dev) up to 64 heads to a key head, and
over more sequences than are cut into pieces."""
from __future__ import annotations

import numpy as np
import pytest

import elem_lib as E
from tree_lib import Tree

pytestmark = pytest.mark.gpu
TYPES = [E.F32, E.F16, E.BF16]


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("group", [9, 16, 33, 64])
def test_many_heads_to_a_key_head(M, t, hd, group):
    print("[case] group", t, hd, group, flush=True)
    c = Tree(M, [(77, 5), (0, 1)], group, 1, hd, t, seed=group)
    c.check(c.call())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lens", [[(3000, 1)] + [(37 * i % 500, 1) for i in range(39)],
                                  [(i % 7, 1) for i in range(300)],
                                  [(900, 1)] + [(11 * i, 1) for i in range(32)]],
                         ids=lambda v: str(len(v)))
def test_batches_of_single_tokens(M, t, lens):
    # More sequences than there are slots to cut them into: whole ones.
    print("[case] single tokens", t, len(lens), flush=True)
    c = Tree(M, lens, 16, 8, 128, t, page=16, seed=len(lens))
    c.check(c.call())
