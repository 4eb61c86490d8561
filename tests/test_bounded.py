"""Calls over bounded caches that are refused before anything is launched (no GPU), the kernels' register budget, and the pool's side of an eviction."""
import ctypes
import importlib
import re

import pytest

from test_kernel_resources import VGPR_FORM, resource_report

p1a = importlib.import_module("p100e-engine_amd")
b = importlib.import_module("p100e-engine_amd.binding")
ARG, SHAPE = -2, -1


def cache(**change):
    kv = b.p1a_kv(p1a.KV_F16, 4096, 4, 256, 4096, 8192, 4096, 4096, 8, 4 * 256 * 2 << 8)
    for k, v in change.items():
        setattr(kv, k, v)
    return kv


def rows(**change):
    r = b.p1a_rows(32, 4, 8, 0, 4096, 4096, 0, 0, 0)
    for k, v in change.items():
        setattr(r, k, v)
    return r


ROWS = [(dict(T=-1), ARG), (dict(n_seq=-1), ARG), (dict(max_rows=-1), ARG), (dict(max_n=-1), ARG), (dict(window=-1), ARG), (dict(n_sink=-1), ARG), (dict(pos0=None), ARG),
        (dict(row0=None, T=33), ARG), (dict(n_seq=65536), SHAPE), (dict(T=1 << 29), SHAPE)]
CACHES = [(dict(type=5), ARG), (dict(k=None), ARG), (dict(pt=None), ARG), (dict(rtab=None), ARG), (dict(n_ctx=-1), ARG), (dict(psh=25), ARG), (dict(pstride=0), ARG), (dict(D=96), SHAPE),
          (dict(D=512), SHAPE), (dict(Hkv=5), SHAPE), (dict(k=4104), SHAPE), (dict(v=4098), SHAPE), (dict(pstride=4 * 512 * 256 + 8), SHAPE),
          (dict(type=p1a.KV_Q8_0, k=4098), SHAPE), (dict(type=p1a.KV_Q4_0, v=4097), SHAPE)]


def chunk(kv=None, r=None, q=4096, out=4096, gate=None, lse=None, qt=0, ot=0, Hq=24):
    kv, r = kv or cache(), r or rows()
    return p1a.lib().p1a_attn_chunk(q, qt, ctypes.byref(kv), out, ot, gate, lse, ctypes.byref(r), Hq, 0.1, None, 0, None)


def mass(kv=None, r=None, q=4096, lse=4096, m=4096, ld=64, qt=0, Hq=24):
    kv, r = kv or cache(), r or rows()
    return p1a.lib().p1a_attn_mass(q, qt, ctypes.byref(kv), lse, m, ld, ctypes.byref(r), Hq, 0.1, None, 0, None)


def test_no_rows_are_no_work():
    for r in (rows(T=0), rows(n_seq=0), rows(n_seq=0, T=0, row0=None)):
        assert chunk(r=r) == 0 and mass(r=r) == 0
        assert p1a.lib().p1a_attn_chunk_scratch_bytes(ctypes.byref(cache()), ctypes.byref(r), 24) == 0
    assert mass(ld=0) == 0


@pytest.mark.parametrize("change, rc", ROWS)
def test_rows_refused(change, rc):
    assert chunk(r=rows(**change)) == rc and mass(r=rows(**change)) == rc and p1a.lib().p1a_last_error()


@pytest.mark.parametrize("change, rc", CACHES)
def test_caches_refused(change, rc):
    assert chunk(kv=cache(**change)) == rc and mass(kv=cache(**change)) == rc and p1a.lib().p1a_last_error()


def test_arguments_refused():
    L = p1a.lib()
    for bad, rc in ((dict(q=None), ARG), (dict(out=None), ARG), (dict(qt=2), ARG), (dict(ot=-1), ARG), (dict(q=4100), SHAPE), (dict(out=4104), SHAPE), (dict(gate=4100), SHAPE),
                    (dict(lse=4098), SHAPE), (dict(Hq=2), SHAPE), (dict(Hq=26), SHAPE), (dict(Hq=4 * 65), SHAPE)):
        assert chunk(**bad) == rc, bad
    for bad, rc in ((dict(q=None), ARG), (dict(lse=None), ARG), (dict(m=None), ARG), (dict(ld=-1), ARG), (dict(qt=7), ARG), (dict(q=4104), SHAPE), (dict(lse=4097), SHAPE), (dict(m=4098), SHAPE)):
        assert mass(**bad) == rc, bad
    assert L.p1a_attn_chunk(4096, 0, None, 4096, 0, None, None, ctypes.byref(rows()), 24, 0.1, None, 0, None) == ARG
    assert L.p1a_attn_chunk(4096, 0, ctypes.byref(cache()), 4096, 0, None, None, None, 24, 0.1, None, 0, None) == ARG

    def select(m=4096, ld=64, n_seq=2, Hkv=4, n_dev=4096, n=0, budget=32, n_sink=4, n_recent=8, keep=4096):
        return L.p1a_evict_select(m, ld, n_seq, Hkv, n_dev, n, budget, n_sink, n_recent, keep, None)
    for bad, rc in ((dict(m=None), ARG), (dict(keep=None), ARG), (dict(ld=-1), ARG), (dict(n_seq=-1), ARG), (dict(Hkv=0), ARG), (dict(n_sink=-1), ARG), (dict(n_recent=-1), ARG),
                    (dict(n_dev=None, n=-1), ARG), (dict(budget=11), SHAPE), (dict(budget=(1 << 20) + 1), SHAPE), (dict(budget=-1, n_sink=0, n_recent=0), SHAPE),
                    (dict(n_sink=2147483647, n_recent=2147483647), SHAPE), (dict(n_seq=65536), SHAPE), (dict(m=4098), SHAPE), (dict(keep=4097), SHAPE)):
        assert select(**bad) == rc, bad
    assert select(n_seq=0) == 0 and select(budget=0, n_sink=0, n_recent=0) == 0

    def compact(kv=None, keep=4096, n_seq=2, budget=8, m=None, out=None, ld=0):
        return L.p1a_kv_compact(ctypes.byref(kv or cache()), keep, n_seq, budget, m, out, ld, None)
    for bad, rc in ((dict(keep=None), ARG), (dict(n_seq=-1), ARG), (dict(budget=-1), ARG), (dict(m=4096), ARG), (dict(out=4096), ARG), (dict(m=4096, out=8192, ld=-1), ARG),
                    (dict(m=4096, out=4100, ld=64), ARG), (dict(kv=cache(pt=None)), ARG), (dict(kv=cache(rtab=None)), ARG), (dict(kv=cache(n_ctx=-1)), ARG), (dict(budget=(1 << 20) + 1), SHAPE),
                    (dict(kv=cache(k=4097)), SHAPE), (dict(kv=cache(pstride=8193)), SHAPE), (dict(keep=4098), SHAPE), (dict(kv=cache(type=9)), ARG)):
        assert compact(**bad) == rc, bad
    assert compact(n_seq=0) == 0 and compact(budget=0) == 0


def test_sizes_past_the_limits():
    """positions, totals and grids whose arithmetic would leave 32 bits"""
    L = p1a.lib()
    for change in (dict(n_ctx=(1 << 30) + 1), dict(Hkv=4097)):
        assert chunk(kv=cache(**change), Hq=4097 if "Hkv" in change else 24) == SHAPE and mass(kv=cache(**change), Hq=4097 if "Hkv" in change else 24) == SHAPE, change
    wide = dict(kv=cache(Hkv=128, pstride=1 << 24), r=rows(T=65535, n_seq=65535, max_rows=1), Hq=128)
    assert chunk(**wide) == SHAPE and mass(**wide) == SHAPE
    assert mass(ld=(1 << 30) + 1) == SHAPE and L.p1a_attn_mass_scratch_bytes(ctypes.byref(cache()), (1 << 30) + 1, ctypes.byref(rows()), 24) == 0
    assert L.p1a_evict_select(4096, (1 << 30) + 1, 2, 4, None, 64, 32, 4, 8, 4096, None) == SHAPE
    assert L.p1a_evict_select(4096, 64, 2, 4097, None, 64, 32, 4, 8, 4096, None) == SHAPE
    assert L.p1a_kv_compact(ctypes.byref(cache()), 4096, 65535, 8, None, None, 0, None) == SHAPE
    assert L.p1a_kv_compact(ctypes.byref(cache()), 4096, 2, 8, 4096, 4096, (1 << 30) + 1, None) == SHAPE


def test_binding_refuses_other_types():
    torch = pytest.importorskip("torch")
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    with pytest.raises(p1a.P1AError, match="float32 or bfloat16"):
        p1a.attn_chunk(q, None, q, p1a.Rows(1), 4, 0.1)


def test_scratch_follows_the_split():
    """the bytes asked for are those of the partials, and none where the device is full without a split"""
    L = p1a.lib()
    one = L.p1a_attn_chunk_scratch_bytes(ctypes.byref(cache(n_ctx=32768)), ctypes.byref(rows(T=1, n_seq=1, max_rows=1)), 24)
    assert one > 0
    full = L.p1a_attn_chunk_scratch_bytes(ctypes.byref(cache(n_ctx=32768)), ctypes.byref(rows(T=20000, n_seq=4, max_rows=8000)), 24)
    assert full == 0


def test_an_evicted_sequence_gives_pages_back():
    pool = p1a.Pool(p1a.KV_Q8_0, 2, 2, 64, 4, 256, 2, 512, host_memory=True)
    i = pool.seq_create()
    pool.seq_advance(i, list(range(100)))
    free = pool.free_pages
    for bad in (101, -1):
        with pytest.raises(p1a.P1AError):
            pool.seq_evict(i, bad)
    pool.seq_evict(i, 40)
    assert pool.seq_len(i) == 40 and pool.free_pages == free + 7 - 3 and pool.seq_tokens(i) == [-1] * 40
    assert pool.seq_advance(i, [7]) == 41 and pool.seq_tokens(i)[40:] == [7]
    pool.seq_evict(i, 41)                                      # (moved within what it holds: no page, but no token has its place)
    assert pool.seq_tokens(i) == [-1] * 41
    with pytest.raises(p1a.P1AError):
        pool.seq_evict(1, 0)


@pytest.mark.parametrize("source, kernel, builds", [("p1a_chunk.hip", "chunk_k", 18), ("p1a_step.hip", "step_k", 36), ("p1a_mass.hip", "mass_k", 9), ("p1a_mass.hip", "mass_step_k", 18)])
def test_kernels_fit_their_budget(tmp_path, source, kernel, builds):
    """nothing in memory; two workgroups to a compute unit where heads have 128 dims and fewer"""
    ks = {k: v for k, v in resource_report(tmp_path, source, VGPR_FORM).items() if kernel in k}
    assert len(ks) >= builds, sorted(ks)
    for name, r in ks.items():
        D = int(re.search(r"ILj\d+ELi(\d+)E", name).group(1))
        assert r.get("VGPRs Spill", 0) == 0 and r.get("ScratchSize", 0) == 0, (name, r)
        assert r["Occupancy"] >= (2 if D <= 128 else 1), (name, r)
