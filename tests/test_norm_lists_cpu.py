"""Rules of the launches of many tensors, at the ends of their lists."""
import os
import subprocess

from conftest import PKG_NAME, ROOT


def test_rules_without_members(tmp_path):
    """Lists whose last launch was full ask for none: an answer, and no division by it."""
    exe = str(tmp_path / "norm_no_members")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", os.path.join(ROOT, "tests", "integration", "norm_no_members.cpp"), "-I", os.path.join(ROOT, PKG_NAME, "csrc"), "-o", exe])
    done = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, (done.returncode, done.stdout[:2000])
