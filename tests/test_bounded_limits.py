"""Arithmetic of the calls over bounded caches at the ends of what they take (no GPU): the kernels' own lines, compiled for the host."""
import ctypes
import importlib
import os
import shutil
import subprocess

import pytest

from test_kernel_resources import ROOT, SRC

SHIM = '''
#include "p1a_tiles.hpp"
extern "C" void through(int first, int rows, int steps, int * o) {
    typedef p1a::step_runs<4>::of_lane lane;
    const lane x{first, 0, 0, lane::both(steps, rows)};
    o[0] = x.first;
    o[1] = x.rows();
    o[2] = x.steps();
}
'''


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc here")
    d = tmp_path_factory.mktemp("limits")
    (d / "shim.hip").write_text(SHIM)
    subprocess.run([hipcc, "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wno-inline-asm", "-Wno-unused-command-line-argument",
                    "-I" + os.path.join(ROOT, "include"), "-I" + SRC, str(d / "shim.hip"), "-o", str(d / "shim.so")], check=True, capture_output=True, timeout=300)
    return ctypes.CDLL(str(d / "shim.so"))


@pytest.mark.parametrize("first", [0, 2 ** 21, 2 ** 25 - 1, 2 ** 25, 2 ** 26 + 3, 2 ** 30 - 1])
@pytest.mark.parametrize("steps", [0, 1, 2 ** 23 + 1])
@pytest.mark.parametrize("rows", [0, 1, 32])
def test_a_sequences_rows_and_steps_fit_what_holds_them(host, first, steps, rows):
    """calls of few rows: whatever its first row's number, a sequence is found again as it was"""
    o = (ctypes.c_int * 3)()
    host.through(first, rows, steps, o)
    assert list(o) == [first, rows, steps]


@pytest.mark.parametrize("max_rows", [1, 64])
@pytest.mark.parametrize("kv_type", ["KV_F16", "KV_Q8_0", "KV_Q4_0"])
def test_caches_of_no_positions_need_no_scratch(kv_type, max_rows):
    """a descriptor with room for nothing: no row sees anything, and the work can be dealt out all the same"""
    p1a, b = importlib.import_module("p100e-engine_amd"), importlib.import_module("p100e-engine_amd.binding")
    kv = b.p1a_kv(getattr(p1a, kv_type), 0, 4, 256, 4096, 8192, 4096, 4096, 8, 4 * 256 * 2 << 8)
    for window in (0, 100):
        rows = b.p1a_rows(64, 1, max_rows, 0, 4096, 4096, 0, window, 0)
        assert p1a.lib().p1a_attn_chunk_scratch_bytes(ctypes.byref(kv), ctypes.byref(rows), 24) == 0
        assert p1a.lib().p1a_attn_mass_scratch_bytes(ctypes.byref(kv), 64, ctypes.byref(rows), 24) >= 0


def test_partial_sums_of_weights_go_by_what_rows_see():
    """... and not by the length of the totals' rows, nor without bound"""
    p1a, b = importlib.import_module("p100e-engine_amd"), importlib.import_module("p100e-engine_amd.binding")
    kv = b.p1a_kv(p1a.KV_F16, 1 << 20, 4, 256, 4096, 8192, 4096, 4096, 8, 4 * 256 * 2 << 8)
    for n_seq in (1, 4):
        rows = b.p1a_rows(4096, n_seq, 4096, 0, 4096, 4096, 0, 512, 4)
        need = p1a.lib().p1a_attn_mass_scratch_bytes(ctypes.byref(kv), 1 << 20, ctypes.byref(rows), 24)
        assert 0 < need <= 32 * n_seq * 4 * 4 * (512 + 4096 + 4 + 96)              # (32 splits at most)
    for max_n in (0, 3000):                                    # (understated, maybe: totals have to fit all the same)
        rows = b.p1a_rows(4096, 1, 4096, max_n, 4096, 4096, 0, 0, 0)
        assert p1a.lib().p1a_attn_mass_scratch_bytes(ctypes.byref(kv), 1 << 20, ctypes.byref(rows), 24) <= 256 << 20


def chunk_bytes(T, n_seq, max_rows, n_ctx, Hq, Hkv, D):
    p1a, b = importlib.import_module("p100e-engine_amd"), importlib.import_module("p100e-engine_amd.binding")
    kv = b.p1a_kv(p1a.KV_F16, n_ctx, Hkv, D, 4096, 8192, 4096, 4096, 8, Hkv * D * 2 << 8)
    rows = b.p1a_rows(T, n_seq, max_rows, 0, 4096, 4096, 0, 0, 0)
    return p1a.lib().p1a_attn_chunk_scratch_bytes(ctypes.byref(kv), ctypes.byref(rows), Hq)


@pytest.mark.parametrize("n_seq", [1, 64, 256, 1024, 4096, 16384, 65535])
def test_partials_of_few_rows_are_bounded(n_seq):
    """single tokens: partials of at most 64 MB and the words beside them, whatever the number of sequences"""
    assert chunk_bytes(n_seq, n_seq, 1, 32768, 32, 8, 128) <= (64 << 20) + 4 * n_seq + 1024
    assert chunk_bytes(1 << 25, n_seq, 1, 32768, 32, 8, 128) == 0                  # (many rows of no sequence)


@pytest.mark.parametrize("T, n_seq, max_rows, n_ctx, Hq, Hkv, D", [(91206, 64, 2145, 973763, 128, 8, 128), (2110, 1, 512, 1 << 18, 24, 4, 256), (1 << 20, 24, 100, 8192, 32, 8, 128),
                                                                   (45012, 16, 4802, 6588, 16, 1, 128)])
def test_partials_of_blocks_are_bounded(T, n_seq, max_rows, n_ctx, Hq, Hkv, D):
    assert chunk_bytes(T, n_seq, max_rows, n_ctx, Hq, Hkv, D) <= (256 << 20) + 1024


def test_the_binding_refuses_tensors_that_would_be_misread():
    """numbers of another size, too few of them, or not on end: a position in 64 bits would be read as two"""
    torch = pytest.importorskip("torch")
    p1a = importlib.import_module("p100e-engine_amd")
    i32 = dict(dtype=torch.int32)
    for bad in (dict(row0=torch.zeros(4, dtype=torch.int64)), dict(pos0=torch.zeros(3, dtype=torch.int64)), dict(pos0=torch.zeros(3)), dict(row0=torch.zeros(3, **i32)),
                dict(pos0=torch.zeros(2, **i32)), dict(pos0=torch.zeros(6, **i32)[::2])):
        with pytest.raises(p1a.P1AError, match=next(iter(bad))):
            p1a.Rows(9, n_seq=3, **bad)
    rows = p1a.Rows(9, n_seq=3, row0=torch.zeros(4, **i32), pos0=torch.zeros(3, **i32))
    cache = p1a.KVCache(p1a.KV_F16, 64, 1, 64, 4096, 8192)
    q, lse, mass, keep = torch.zeros(9, 2, 64), torch.zeros(9, 2), torch.zeros(3, 1, 64), torch.zeros(3, 1, 8, **i32)
    for x in (lse.bfloat16(), lse[:8], torch.zeros(2, 9).t()):
        with pytest.raises(p1a.P1AError, match="lse"):
            p1a.attn_chunk(q, cache, q, rows, 2, 0.1, lse=x)
        with pytest.raises(p1a.P1AError, match="lse"):
            p1a.attn_mass(q, cache, x, mass, rows, 2, 0.1)
    with pytest.raises(p1a.P1AError, match="gate"):
        p1a.attn_chunk(q, cache, q, rows, 2, 0.1, gate=torch.zeros(9, 128, dtype=torch.bfloat16))
    for x in (mass.double(), mass[:2], torch.zeros(3, 1, 128)[..., ::2]):
        with pytest.raises(p1a.P1AError, match="mass"):
            p1a.attn_mass(q, cache, lse, x, rows, 2, 0.1)
    for call, what in ((lambda: p1a.evict_select(mass.double(), 9, keep), "mass"), (lambda: p1a.evict_select(mass, torch.zeros(3, dtype=torch.int64), keep), "n"),
                       (lambda: p1a.evict_select(mass, 9, keep.long()), "keep"), (lambda: p1a.evict_select(mass, 9, keep[:2]), "keep"), (lambda: p1a.kv_compact(cache, keep.long()), "keep"),
                       (lambda: p1a.kv_compact(cache, torch.zeros(3, 2, 8, **i32)), "keep"), (lambda: p1a.kv_compact(cache, keep, mass=mass, mass_out=mass[:2]), "mass_out")):
        with pytest.raises(p1a.P1AError, match=what):
            call()
