"""What the compiler does not look after in inline assembly, read from its assembly listing (no GPU needed: hipcc cross-compiles)."""
import os
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_kernel_resources import ROOT, SRC, VGPR_FORM

SOURCES = {"p1a_decode.hip": (), "p1a_prefill.hip": VGPR_FORM, "p1a_chunk.hip": VGPR_FORM, "p1a_step.hip": VGPR_FORM, "p1a_mass.hip": VGPR_FORM}


def instructions(path):
    with open(path) as f:
        for line in f:
            line = line.split(";")[0].strip()
            if line and not line.startswith((".", "#")) and not line.endswith(":"):
                yield line


def test_no_load_to_lds_right_behind_the_write_of_its_address(tmp_path):
    """a load whose data go to LDS at M0 needs an instruction between it and the scalar one that writes M0"""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc here")

    def listing(source):
        out = str(tmp_path / (source + ".s"))
        r = subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-I" + os.path.join(ROOT, "include"), "-I" + SRC, "-Xclang", "-target-feature", "-Xclang",
                            "-packed-fp32-ops", "-Wno-unused-command-line-argument", "-Wno-inline-asm", "--cuda-device-only", "-S", *SOURCES[source], os.path.join(SRC, source), "-o", out],
                           capture_output=True, text=True, timeout=900)
        assert r.returncode == 0, r.stderr[-2000:]
        return out
    with ThreadPoolExecutor(4) as pool:
        listings = dict(zip(SOURCES, pool.map(listing, SOURCES)))
    for source, path in listings.items():
        before, loads, bare = "", 0, 0
        for line in instructions(path):
            if re.match(r"(global|buffer)_load_lds_", line):
                loads += 1
                bare += bool(re.match(r"s_\w+ m0\b", before))
            before = line
        assert loads and not bare, (source, loads, bare)
