"""What a wave keeps for all its lanes is saved with all lanes active, read from the machine code of the built library (no GPU needed).

Where lanes part, the compiler jumps past what none of them does and brings the mask of active lanes back behind it. Where registers are short it has put copies of values into other
registers between the two: whoever came with an empty mask saved nothing, and the addresses made from such a value later were anywhere."""
import glob
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def lost_copies(lines):
    """(kernel, instruction) of vector registers written where an empty mask arrives, ahead of the mask's return. lines: a listing with labels, L: or <L>:"""
    lines = [x.split("//")[0].split(";")[0].strip() for x in lines]
    empty = {m.group(1) for x in lines if (m := re.match(r"s_cbranch_execz\s+<?([.\w]+)>?", x))}
    kernel, at, written = "", False, []
    for x in lines:
        if not x:
            continue
        m = re.match(r"(?:[0-9a-f]+ )?<?([.\w$]+)>?:$", x)
        if m:
            name = m.group(1)
            if name.startswith("_Z"):
                kernel = name
            at, written = name in empty, []
        elif re.match(r"s_cbranch_execnz\b", x):               # (a loop's end: behind it nobody is active)
            at, written = True, []
        elif not at:
            continue
        elif "saveexec" in x or re.match(r"s_\w+ exec,", x):
            if x.startswith(("s_or_b64 exec, exec", "s_mov_b64 exec", "s_andn2_saveexec", "s_or_saveexec")):
                yield from ((kernel, w) for w in written)
            at = False
        elif x.startswith(("s_cbranch", "s_branch", "s_endpgm", "s_setpc")):
            at = False                                         # (the mask does not change here: it was never empty)
        elif re.match(r"(v_|ds_read|ds_bpermute|(global|buffer|flat|scratch)_load)", x) and not re.match(r"v_readlane|v_readfirstlane|v_writelane", x):
            written.append(x)


def test_values_are_not_saved_where_no_lane_is_active(p1a, tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump here")
    lib = shutil.copy(p1a.lib_path(), tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True, timeout=120)
    parts = [f for f in glob.glob(str(tmp_path / "*gfx950*")) if os.path.getsize(f)]
    kernels, joins, bad = 0, 0, []
    for f in parts:
        text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", "--no-show-raw-insn", f], check=True, capture_output=True, text=True, timeout=300).stdout.split("\n")
        kernels += sum(re.match(r"[0-9a-f]+ <_Z", x) is not None for x in text)
        joins += sum("s_cbranch_execz" in x for x in text)
        bad += lost_copies(text)
    assert kernels > 300 and joins > 1000, (kernels, joins)
    assert not bad, (len(bad), bad[:8])


def test_the_check_finds_them():
    """a copy behind the jump of an empty mask, one behind a loop, and what is right: work ahead of a jump, copies behind the mask's return"""
    head = ["_Zk:", "s_and_saveexec_b64 s[2:3], vcc", "s_cbranch_execz .L1", "v_add_u32_e32 v1, 1, v1", ".L0:", "v_add_u32_e32 v2, 1, v1", "s_andn2_b64 exec, exec, s[6:7]", "s_cbranch_execnz .L0"]
    right = [*head, "s_or_b64 exec, exec, s[6:7]", ".L1:", "s_or_b64 exec, exec, s[2:3]", "v_accvgpr_write_b32 a1, v3", "s_endpgm"]
    assert list(lost_copies(right)) == []
    assert list(lost_copies([*head, "s_or_b64 exec, exec, s[6:7]", ".L1:", "v_accvgpr_write_b32 a1, v3", "s_or_b64 exec, exec, s[2:3]", "s_endpgm"])) == [("_Zk", "v_accvgpr_write_b32 a1, v3")]
    assert list(lost_copies([*head, "v_mov_b32_e32 v9, v3", "s_or_b64 exec, exec, s[6:7]", ".L1:", "s_or_b64 exec, exec, s[2:3]", "s_endpgm"])) == [("_Zk", "v_mov_b32_e32 v9, v3")]
