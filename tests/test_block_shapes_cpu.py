"""The cases of the GPU tests of block shapes reach every block that the rules of dispatch can choose; the rules are built with g++."""
import os
import subprocess

import pytest

from conftest import PKG_NAME, ROOT
from test_gpu_block_shapes import EXPERTS, PAIRS, RINGS


@pytest.fixture(scope="module")
def blocks(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("blocks") / "block_cases")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", os.path.join(ROOT, "tests", "integration", "block_cases.cpp"), "-I", os.path.join(ROOT, PKG_NAME, "csrc"), "-o", exe])

    def run(lines):
        done = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=120)
        assert done.returncode == 0, done.stderr
        return [[int(v) for v in line.split()] for line in done.stdout.splitlines()]

    return run


def _expert_blocks(blocks):
    """(M, T, sizes, tiles, most products of a sum) of every case"""
    lines = [" ".join(map(str, ["experts", (1 << RINGS[ring]["log_n"]) // 128 * (level + 1), tiles, *sizes])) for ring, level, _, _, _, sizes, tiles, _ in EXPERTS]
    return [(m, t, case[5], case[6], case[2] * case[4] if case[7] else 0) for (m, t), case in zip(blocks(lines), EXPERTS)]


def test_every_block_of_experts(blocks):
    flat = blocks(["kernels"])[0]
    kernels = set(zip(flat[::2], flat[1::2]))
    assert len(kernels) == 15
    reached = {}
    for m, t, sizes, tiles, _ in _expert_blocks(blocks):
        places = reached.setdefault((m, t), (set(), set()))
        places[0].update(n for size in sizes for n in ([m] if size >= m else []) + ([size % m] if size % m else []))
        places[1].add(tiles % t)
    assert set(reached) == kernels
    for (m, t), (positions, rests) in reached.items():
        assert positions == set(range(1, m + 1)), (m, t, positions)   # blocks that are full, and with every number of positions less
    assert {k for k, (_, rests) in reached.items() if rests - {0}} >= {(1, 2), (1, 3), (1, 4), (1, 6), (1, 8), (2, 6), (3, 4)}   # a last block with fewer tiles


def test_sums_of_experts_past_every_reduction(blocks):
    for m in (2, 3):
        products = {n for mm, _, _, _, n in _expert_blocks(blocks) if mm == m and n}
        assert {127, 128, 129} <= products


def test_every_run_of_ranges(blocks):
    lines = [" ".join(map(str, ["pairs", 1 << RINGS[ring]["log_n"], level + 1, heads, nq, nk])) for ring, level, _, heads, nq, nk, _ in PAIRS]
    reached = {tuple(b) for b in blocks(lines)}
    assert reached == {(block, run) for block in range(6) for run in (1, 2, 4, 8, 16)}
    several = [case for case, (_, run) in zip(PAIRS, blocks(lines)) if run >= 4]
    assert {1, 2, 3, 5} <= {case[2] for case in several}   # one group: every copy begins a range; and numbers that are no multiple of the ring's four stages
    assert any(case[6] for case in several)
