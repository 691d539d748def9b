"""Products grouped by expert from a program on the C++ headers, built with g++ against the two shared libraries."""
import subprocess

import pytest

from test_gpu_boundary import _compiled


@pytest.mark.gpu
def test_grouped_products_of_a_separately_compiled_program(tmp_path):
    r = subprocess.run([str(_compiled("grouped_calls", tmp_path))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_the_program_compiles(tmp_path):
    _compiled("grouped_calls", tmp_path)
