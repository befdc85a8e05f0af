"""gfx950's conversions of 32 values at a time write their results in several passes: in the objects built here none shares a result register with an
operand, and none is read by the instruction behind it."""
import glob
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJECTS = sorted(glob.glob(os.path.join(ROOT, "saragossa_amd", "csrc", "kernels*.o")))
LLVM = "/opt/rocm/llvm/bin/"


def registers(text):
    """Numbers of the vector registers of an operand, or of several."""
    found = set()
    for lo, hi, one in re.findall(r"\bv(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        found |= set(range(int(lo), int(hi) + 1)) if lo else {int(one)}
    return found


def test_registers():
    assert registers("v[82:87]") == set(range(82, 88)) and registers("v66") == {66} and registers(" v[2:3], v7") == {2, 3, 7} and not registers("s[0:3], vcc")


@pytest.mark.skipif(not OBJECTS or not shutil.which(LLVM + "llvm-objdump"), reason="no objects built here, or no llvm-objdump")
def test_results_are_apart_from_operands(tmp_path):
    seen = 0
    for path in OBJECTS:
        fat, code = tmp_path / "fat", tmp_path / "code"
        subprocess.run([LLVM + "llvm-objcopy", f"--dump-section=.hip_fatbin={fat}", path, str(tmp_path / "copy")], check=True)
        subprocess.run([LLVM + "clang-offload-bundler", "--type=o", "--unbundle", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                        f"--input={fat}", f"--output={code}"], check=True, capture_output=True)
        text = subprocess.run([LLVM + "llvm-objdump", "-d", "--no-show-raw-insn", str(code)], check=True, capture_output=True, text=True).stdout
        lines = [line.split("//")[0].strip() for line in text.splitlines()]
        for line, behind in zip(lines, lines[1:]):
            if re.match(r"v_cvt_scalef32_(2xpk16|pk32)_", line):
                result, operands = line.split(None, 1)[1].split(",", 1)
                assert not registers(result) & registers(operands), (path, line)
                assert not registers(result) & registers(behind), (path, line, behind)
                seen += 1
    assert seen > 100
