"""Arithmetic of the calls over bounded caches at the ends of what they take (no GPU): the kernels' own lines, compiled for the host."""
import ctypes
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
