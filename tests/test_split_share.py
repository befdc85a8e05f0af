"""How many splits share a launch's pages, on the host: a g++ build of saragossa_amd/csrc/split_share.h with tests/native/split_share.cpp."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_shares_of_any_context_have_32_bits(tmp_path):
    exe = tmp_path / "split_share"
    build = subprocess.run(["g++", "-std=c++17", "-O2", "-I" + os.path.join(ROOT, "saragossa_amd", "csrc"),
                            os.path.join(ROOT, "tests", "native", "split_share.cpp"), "-o", str(exe)], capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stderr[-2000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout
