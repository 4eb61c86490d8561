"""The C++ face of the pool (include/p100e_kv_pool.hpp) where it has no counterpart in the reference: its call reaches the library with its arguments (no GPU:
the program brings the library's functions that would need one)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r'''
#include "p100e_kv_pool.hpp"
#include <cstdio>
static int pool, calls, last_id, last_n;
extern "C" p1a_pool * p1a_pool_create(const p1a_pool_cfg *, void *) { return (p1a_pool *) &pool; }
extern "C" void p1a_pool_destroy(p1a_pool *) {}
extern "C" int p1a_seq_evict(p1a_pool * p, int id, int n) {
    if ((void *) p != &pool) return P1A_E_ARG;
    ++calls; last_id = id; last_n = n;
    return n > 100 ? P1A_E_ARG : P1A_OK;
}
int main() {
    p100e::kv_pool p(P1A_KV_F16, 1, 1, 64, 4, 256, 2, nullptr);
    int thrown = 0;
    try { p.seq_evict(0, 1); } catch (const std::runtime_error &) { ++thrown; }
    if (thrown != 1 || calls) { puts("a pool that is not there"); return 1; }
    p.alloc_pool(256);
    p.seq_evict(3, 40);
    if (calls != 1 || last_id != 3 || last_n != 40) { puts("arguments"); return 1; }
    try { p.seq_evict(3, 101); } catch (const std::runtime_error &) { ++thrown; }
    if (thrown != 2) { puts("a refusal"); return 1; }
    puts("fine");
    return 0;
}
'''


def test_eviction_reaches_the_pool(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc here")
    lib = os.path.join(ROOT, "p100e-engine_amd")
    (tmp_path / "evict.cpp").write_text(PROGRAM)
    r = subprocess.run([hipcc, "-std=c++17", "-O1", "-I" + os.path.join(ROOT, "include"), str(tmp_path / "evict.cpp"), "-o", str(tmp_path / "evict"), "-L" + lib, "-lp1a_attn",
                        "-Wl,-rpath," + lib], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(tmp_path / "evict")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
