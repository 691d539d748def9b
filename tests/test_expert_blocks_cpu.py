"""The rule that shapes blocks of products grouped by expert, built with g++."""
import os
import subprocess

from conftest import PKG_NAME, ROOT


def test_blocks_take_what_was_measured_quicker(tmp_path):
    exe = str(tmp_path / "expert_blocks")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", os.path.join(ROOT, "tests", "integration", "expert_blocks.cpp"), "-I", os.path.join(ROOT, PKG_NAME, "csrc"),
                           "-I", "/usr/local/cuda/include", "-o", exe])
    done = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
