"""Calls on drafted trees whose sizes leave what a launch can hold are refused before anything is launched; steps without rows are not (no GPU)."""
import ctypes
import importlib

from test_bounded import SHAPE, cache, rows
from test_trees import tree, tree_rows, verify

p1a = importlib.import_module("p100e-engine_amd")


def test_verifications_that_a_launch_does_not_hold():
    """2^24 workgroups of 256 threads and more: stretches of 4096 logits of all rows; of all sequences, four times where a node's children are looked at in rounds"""
    V = 1 << 20                                                 # 256 stretches
    for bad in (dict(r=rows(T=1 << 16, n_seq=1 << 13, max_rows=8), V=V), dict(r=rows(T=(1 << 20) - 1, n_seq=60000, max_rows=100), V=17 * 4096),
                dict(r=rows(T=16, n_seq=1 << 14, max_rows=8), V=V, draft=4096, kids=3), dict(r=rows(T=16, n_seq=1 << 14, max_rows=8), V=V, draft=4096, kids=2, flags=1),
                dict(r=rows(T=32, n_seq=65535, max_rows=8), V=V, draft=4096, kids=2, flags=3)):
        assert verify(**bad) == SHAPE and b"workgroups" in p1a.lib().p1a_last_error(), bad


def test_attention_that_a_launch_does_not_hold():
    assert tree(kv=cache(n_ctx=256, Hkv=512, pstride=512 * 512 << 8), r=rows(T=1000, n_seq=8192, max_rows=1000), words=32, Hq=32768) == SHAPE
    assert b"workgroups" in p1a.lib().p1a_last_error()


def test_a_step_without_rows():
    """... whose tensors have no memory"""
    r = rows(T=0)
    assert tree(r=r, q=None, out=None, mask=None) == 0 and tree_rows(r=r, parent=None, mask=None, pos=None, slot=None) == 0
