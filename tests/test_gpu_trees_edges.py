"""Calls on drafted trees at the ends of what their documentation allows, each against its formula in 64 bits. Tolerances of attention are those of test_gpu_trees.py."""
import numpy as np
import pytest

import _inputs as I
import _oracle as O
from _bounded import Cache
from test_gpu_trees import Call

pytestmark = pytest.mark.gpu

KVS = {"f16": O.KV_F16, "q8_0": O.KV_Q8_0, "q4_0": O.KV_Q4_0}


@pytest.mark.parametrize("Hq", [1, 12])                         # (20 columns: waves with keys of their own; 240: waves that share them)
@pytest.mark.parametrize("kv", list(KVS))
def test_masks_that_name_slots_past_the_cache(p1a, kv, Hq):
    """trees that reach past n_ctx, which ends inside a tile of keys: slots behind it are nobody's, whatever the masks say"""
    g = I.rng(91)
    some = [g.random((20, 20)) < 0.4 for _ in range(2)]
    some[0][0] = False
    some[0][0, [3, 12]] = True                                  # position 93 and, of a cache of 100, none
    every = [np.ones((20, 20), bool)] * 2
    for D, out_bf16 in ((64, False), (128, True), (256, False)):
        flat = Cache(p1a, KVS[kv], 1, D, 0, [100], 92, paged=False)
        paged = Cache(p1a, KVS[kv], 1, D, 4, [48, 48], 93, max_pages=3)
        assert flat.kv.n_ctx == 100 and paged.kv.n_ctx == 48
        for window, n_sink in ((0, 0), (30, 3)):
            for see in (some, every):
                Call(p1a, flat, Hq, [20], [90], window, n_sink, see=see[:1]).check(p1a, out_bf16, lse=not out_bf16)
                Call(p1a, paged, Hq, [20, 20], [40, 47], window, n_sink, see=see, junk=True, words=2).check(p1a, out_bf16, lse=not out_bf16)
