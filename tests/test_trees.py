"""Calls on drafted trees that are refused before anything is launched (no GPU), their scratch, and the kernels' register budget."""
import ctypes
import importlib
import re

import numpy as np
import pytest

import _trees as R
from test_bounded import ARG, CACHES, ROWS, SHAPE, cache, rows
from test_kernel_resources import VGPR_FORM, resource_report

p1a = importlib.import_module("p100e-engine_amd")
b = importlib.import_module("p100e-engine_amd.binding")


def tree(kv=None, r=None, q=4096, out=4096, gate=None, lse=None, mask=4096, words=1, qt=0, ot=0, Hq=24):
    kv, r = kv or cache(), r or rows()
    return p1a.lib().p1a_attn_tree(q, qt, ctypes.byref(kv), out, ot, gate, lse, ctypes.byref(r), mask, words, Hq, 0.1, None, 0, None)


def tree_rows(r=None, parent=4096, mask=4096, words=1, pos=4096, slot=4096):
    return p1a.lib().p1a_tree_rows(parent, ctypes.byref(r or rows()), mask, words, pos, slot, None)


def verify(r=None, target=4096, tt=0, ld=0, draft=None, dt=0, dld=0, V=100, token=4096, parent=4096, temp=4096, u=4096, un=4096, n=4096, path=4096, width=4, nxt=4096, kids=2, flags=0):
    return p1a.lib().p1a_tree_verify(target, tt, ld, draft, dt, dld, V, token, parent, temp, u, un, n, path, width, nxt, ctypes.byref(r or rows()), kids, flags, None, 0, None)


def commit(layers=None, n_layers=None, r=None, n=4096, path=4096, width=4):
    layers = [cache()] * 2 if layers is None else layers
    a = (b.p1a_kv * max(len(layers), 1))(*layers)
    return p1a.lib().p1a_tree_commit(a, len(layers) if n_layers is None else n_layers, ctypes.byref(r or rows()), n, path, width, None)


def test_no_rows_are_no_work():
    for r in (rows(T=0), rows(n_seq=0), rows(n_seq=0, T=0, row0=None)):
        assert tree(r=r) == 0 and tree_rows(r=r) == 0 and commit(r=r) == 0
        assert p1a.lib().p1a_attn_tree_scratch_bytes(ctypes.byref(cache()), ctypes.byref(r), 24, 1) == 0
    assert verify(r=rows(n_seq=0)) == 0 and commit(n_layers=0) == 0


@pytest.mark.parametrize("change, rc", ROWS)
def test_rows_refused(change, rc):
    assert tree(r=rows(**change)) == rc and p1a.lib().p1a_last_error()
    if not set(change) & {"max_n", "window", "n_sink"}:        # (what calls without a cache do not look at)
        assert tree_rows(r=rows(**change)) == rc and commit(r=rows(**change)) == rc
        if "pos0" not in change:
            assert verify(r=rows(**change)) == rc


@pytest.mark.parametrize("change, rc", CACHES)
def test_caches_refused(change, rc):
    assert tree(kv=cache(**change)) == rc and p1a.lib().p1a_last_error()


def test_arguments_refused():
    for bad, rc in ((dict(q=None), ARG), (dict(out=None), ARG), (dict(mask=None), ARG), (dict(words=-1), ARG), (dict(qt=2), ARG), (dict(ot=-1), ARG), (dict(words=0), SHAPE), (dict(words=33), SHAPE),
                    (dict(r=rows(T=64, max_rows=33)), SHAPE), (dict(r=rows(T=2000, max_rows=1025), words=32), SHAPE), (dict(q=4100), SHAPE), (dict(out=4104), SHAPE), (dict(gate=4100), SHAPE),
                    (dict(lse=4098), SHAPE), (dict(mask=4098), SHAPE), (dict(Hq=2), SHAPE), (dict(Hq=26), SHAPE), (dict(Hq=4 * 65), SHAPE)):
        assert tree(**bad) == rc, bad
    for bad, rc in ((dict(parent=None), ARG), (dict(mask=None), ARG), (dict(words=-1), ARG), (dict(words=0), SHAPE), (dict(r=rows(T=64, max_rows=33)), SHAPE), (dict(parent=4097), SHAPE),
                    (dict(pos=4098), SHAPE), (dict(slot=4099), SHAPE), (dict(r=rows(T=2000, max_rows=1025), words=33), SHAPE)):
        assert tree_rows(**bad) == rc, bad
    for bad, rc in ((dict(target=None), ARG), (dict(token=None), ARG), (dict(u=None), ARG), (dict(un=None), ARG), (dict(n=None), ARG), (dict(path=None), ARG), (dict(nxt=None), ARG), (dict(width=0), ARG),
                    (dict(V=0), ARG), (dict(flags=4), ARG), (dict(draft=4096, kids=0), ARG), (dict(tt=2), ARG), (dict(draft=4096, dt=5), ARG), (dict(V=(1 << 20) + 1), SHAPE), (dict(ld=99), SHAPE),
                    (dict(draft=4096, dld=99), SHAPE), (dict(ld=(1 << 40) + 1), SHAPE), (dict(target=4098), SHAPE), (dict(target=4097, tt=1), SHAPE), (dict(draft=4098), SHAPE), (dict(token=4098), SHAPE),
                    (dict(r=rows(T=2000, max_rows=1025)), SHAPE), (dict(r=rows(T=(1 << 20) + 1, max_rows=8)), SHAPE)):
        assert verify(**bad) == rc, bad
    other = dict(type=p1a.KV_Q8_0, n_ctx=100, Hkv=2, D=128, pt=8192, rtab=8192, psh=4, pstride=1 << 22)
    for bad, rc in ((dict(n=None), ARG), (dict(path=None), ARG), (dict(width=0), ARG), (dict(n_layers=-1), ARG), (dict(layers=[cache()] * 129), SHAPE), (dict(n=4098), SHAPE), (dict(path=4097), SHAPE),
                    (dict(layers=[cache(k=4097)]), SHAPE), (dict(layers=[cache(pstride=(4 * 512 << 8) + 1)]), SHAPE), (dict(layers=[cache(type=9)]), ARG), (dict(layers=[cache(pt=None)]), ARG),
                    (dict(layers=[cache(rtab=None)]), ARG), (dict(layers=[cache(n_ctx=-1)]), ARG)):
        assert commit(**bad) == rc, bad
    for k, v in other.items():
        assert commit(layers=[cache(), cache(**{k: v})]) == ARG, k
    L = p1a.lib()
    assert L.p1a_attn_tree(4096, 0, None, 4096, 0, None, None, ctypes.byref(rows()), 4096, 1, 24, 0.1, None, 0, None) == ARG
    assert L.p1a_attn_tree(4096, 0, ctypes.byref(cache()), 4096, 0, None, None, None, 4096, 1, 24, 0.1, None, 0, None) == ARG
    assert L.p1a_tree_commit(None, 1, ctypes.byref(rows()), 4096, 4096, 4, None) == ARG


def test_sizes_past_the_limits():
    """steps that would leave 32 bits"""
    assert tree(kv=cache(n_ctx=1 << 30, Hkv=1, pstride=1 << 24), r=rows(T=60000, n_seq=60000, max_rows=1), Hq=8) == SHAPE
    assert tree(kv=cache(n_ctx=(1 << 30) + 1)) == SHAPE


def test_binding_refuses():
    torch = pytest.importorskip("torch")
    i, f = torch.zeros(8, dtype=torch.int32), torch.zeros(8)
    r = p1a.Rows(8)
    x = torch.zeros(8, 10)
    ok = dict(target=x, token=i, rows=r, u=f, u_next=f, n_accept=i, path=i.view(1, 8), next=i)
    for bad in (dict(target=x.half()), dict(target=x[:4]), dict(target=x.t()), dict(target=x.expand(8, 10)[:, ::2]), dict(draft=x[:, :9]), dict(token=i.long()), dict(token=i[:7]), dict(u=f[:7]), dict(u=f.double()),
                dict(parent=i[:7]), dict(temp=f[:0]), dict(n_accept=i[:0]), dict(next=f), dict(path=i.view(1, 8).long())):
        with pytest.raises(p1a.P1AError):
            p1a.tree_verify(**{**ok, **bad})
    for bad in ((i[:7], r, i.view(8, 1)), (i, r, i[:4].view(4, 1)), (i.long(), r, i.view(8, 1))):
        with pytest.raises(p1a.P1AError):
            p1a.tree_rows(*bad)
    with pytest.raises(p1a.P1AError):
        p1a.tree_commit([b.KVDesc(cache())], p1a.Rows(8, n_seq=1), i.long(), i.view(1, 8))
    q = torch.zeros(8, 4, 256, dtype=torch.float16)
    with pytest.raises(p1a.P1AError, match="float32 or bfloat16"):
        p1a.attn_tree(q, b.KVDesc(cache()), q, r, i.view(8, 1), 4, 0.1)
    with pytest.raises(p1a.P1AError, match="on end"):
        p1a.attn_tree(q.float()[:7], b.KVDesc(cache()), q.float(), r, i.view(8, 1), 4, 0.1)


def test_native_calls_hand_over_what_they_are_given(monkeypatch):
    """the calls that come through the native module: every argument at its place in the C call, tensors looked at first; and after the module was loaded anew"""
    torch = pytest.importorskip("torch")
    b = importlib.import_module("p100e-engine_amd.binding")
    got = []

    def stand_in(*types):
        return ctypes.CFUNCTYPE(ctypes.c_int, *types)(lambda *a: got.append(tuple(bytes(x.contents) if isinstance(x, R) else x for x in a)) or -7)
    VP, I = ctypes.c_void_p, ctypes.c_int
    R = ctypes.POINTER(b.p1a_rows)
    kept = [stand_in(VP, R, VP, I, VP, VP, VP), stand_in(VP, I, R, VP, VP, I, VP)]
    for again in range(2):
        got.clear()
        if again:
            b._call = None
        m = b._trees()
        m.bind(*(ctypes.cast(getattr(b.lib(), n), VP).value for n in ("p1a_attn_prep", "p1a_attn_decode_a16", "p1a_attn_prefill", "p1a_kv_append")), b.KVCache, lambda: 0x7770,
               ctypes.c_int, ctypes.c_uint32, ctypes.c_size_t, ctypes.c_float, VP, b.p1a_kv)
        m.bind_trees(*(ctypes.cast(f, VP).value for f in kept), b._of, torch.int32)
        try:
            r = b.Rows(6, n_seq=2, p0=3)
            parent, mask, pos, slot = (torch.zeros(n, dtype=torch.int32) for n in (6, 12, 6, 6))
            mask = mask.view(6, 2)
            layers = b.Layers([b.KVCache(1, 64, 1, 64, 0x1000, 0x2000)] * 3)
            path = torch.zeros(2, 5, dtype=torch.int32)
            for f in (lambda: b.tree_rows(parent, r, mask, pos, slot), lambda: b.tree_rows(parent, r, mask), lambda: b.tree_commit(layers, r, pos, path)):
                with pytest.raises(b.P1AError, match="-7"):
                    f()
            at = bytes(r._st)
            assert got == [(parent.data_ptr(), at, mask.data_ptr(), 2, pos.data_ptr(), slot.data_ptr(), 0x7770), (parent.data_ptr(), at, mask.data_ptr(), 2, None, None, 0x7770),
                           (layers._at, 3, at, pos.data_ptr(), path.data_ptr(), 5, 0x7770)]
            for f in (lambda: b.tree_rows(parent[:5], r, mask), lambda: b.tree_rows(parent.long(), r, mask), lambda: b.tree_rows(parent, r, mask[:, :1]), lambda: b.tree_rows(parent, r, mask, pos[::2]),
                      lambda: b.tree_commit(layers, r, pos[:1], path), lambda: b.tree_commit(layers, r, pos, path.float()), lambda: b.tree_commit(layers, r, pos, path[:, :3])):
                with pytest.raises(b.P1AError, match="on end"):
                    f()
            for f in (lambda: b.tree_rows(parent, None, mask), lambda: b.tree_rows(parent, r, None), lambda: b.tree_rows(3, r, mask), lambda: m.tree_rows(parent, r, mask, pos)):
                with pytest.raises((AttributeError, TypeError)):
                    f()
            assert len(got) == 3
        finally:
            b._call = b._tree = None                           # (the library's own entry points again)
    with pytest.raises(RuntimeError, match="bind"):
        b._calls().tree_rows(parent, r, mask, None, None)
    b._trees()


def test_scratch():
    L = p1a.lib()
    one = L.p1a_attn_tree_scratch_bytes(ctypes.byref(cache(n_ctx=32768)), ctypes.byref(rows(T=16, n_seq=1, max_rows=16)), 24, 1)
    assert 0 < one <= (128 << 20) + 4096
    many = L.p1a_attn_tree_scratch_bytes(ctypes.byref(cache(n_ctx=32768)), ctypes.byref(rows(T=40000, n_seq=2500, max_rows=16)), 24, 0)
    assert many == 0
    r = rows(T=100, n_seq=20, max_rows=5)
    assert L.p1a_tree_verify_scratch_bytes(ctypes.byref(r), 151936, 0) > L.p1a_tree_verify_scratch_bytes(ctypes.byref(r), 151936, 1) > 0
    assert L.p1a_tree_verify_scratch_bytes(ctypes.byref(r), (1 << 20) + 1, 0) == 0


def test_kernels_fit_their_budget(tmp_path):
    """nothing in memory; two workgroups to a compute unit where heads have 128 dims and fewer"""
    ks = {k: v for k, v in resource_report(tmp_path, "p1a_tree.hip", VGPR_FORM).items() if re.search("few_kI|team_kI", k)}
    assert len(ks) >= 54, sorted(ks)
    for name, r in ks.items():
        D = int(re.search(r"ILj\d+ELi(\d+)E", name).group(1))
        assert r.get("ScratchSize", 0) == 0, (name, r)
        assert r["Occupancy"] >= (2 if D <= 128 else 1), (name, r)


def test_the_oracle_keeps_the_target_s_distribution():
    """what the walk's definition promises, on the CPU: the first token behind node 0 has the target's distribution, whatever was drafted"""
    g = np.random.default_rng(5)
    V, N = 6, 20000
    p, q = R.softmax(g.normal(size=V) * 1.5), R.softmax(g.normal(size=V) * 1.5)
    target = np.log(np.stack([p] * 4)).astype(np.float32)
    for how in ("none", "iid", "distinct"):
        seen = np.zeros(V)
        for _ in range(N):
            if how == "iid":
                kids = g.choice(V, 3, p=q)
            elif how == "distinct":
                kids = g.choice(V, 3, p=q, replace=False)
            else:
                kids = np.argsort(-q)[:3]
            path, nxt = R.verify(target, [0, *kids], [-1, 0, 0, 0], g.random(4), g.random(), None if how == "none" else np.stack([q] * 4), distinct=how == "distinct")
            seen[kids[path[0] - 1] if path else nxt] += 1
        # (each count is binomial: five standard deviations)
        assert (np.abs(seen / N - p) <= 5 * np.sqrt(p * (1 - p) / N)).all(), (how, seen / N, p)


def test_no_load_to_lds_right_behind_the_write_of_its_address(tmp_path):
    """a load whose data go to LDS at M0 needs an instruction between it and the scalar one that writes M0"""
    import os
    import shutil
    import subprocess

    from test_kernel_resources import ROOT, SRC
    from test_kernel_waits import instructions
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc here")
    out = str(tmp_path / "tree.s")
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-I" + os.path.join(ROOT, "include"), "-I" + SRC, "-Xclang", "-target-feature", "-Xclang",
                        "-packed-fp32-ops", "-Wno-unused-command-line-argument", "-Wno-inline-asm", "--cuda-device-only", "-S", *VGPR_FORM, os.path.join(SRC, "p1a_tree.hip"), "-o", out],
                       capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    before, loads, bare = "", 0, 0
    for line in instructions(out):
        if re.match(r"(global|buffer)_load_lds_", line):
            loads += 1
            bare += bool(re.match(r"s_\w+ m0\b", before))
        before = line
    assert loads and not bare, (loads, bare)
