"""Masks of the tile transforms, built with g++ and the address sanitizer."""
import os
import subprocess

from conftest import PKG_NAME, ROOT


def test_shapes_past_the_slots_are_refused(tmp_path):
    exe = str(tmp_path / "masks")
    hellm = os.path.join(ROOT, PKG_NAME, "csrc", "hellm")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=address", "-I", hellm, "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "integration", "masks.cpp"),
                           "-Wl,--unresolved-symbols=ignore-all", "-o", exe])
    done = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr[-2000:]
