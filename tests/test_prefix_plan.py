"""Which kernel prefix attention takes (pz_prefixplan.h): the GPU cases run the ones that
they are made for, so that none of them passes by another's work."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "native", "prefix_plan_check.cpp")
INC = os.path.join(ROOT, "project-zero_amd", "csrc")
FEW, SOME, WIDE = range(3)


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "prefix_plan_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", INC, SRC, "-o", str(exe)],
                   check=True)

    def run(*args):
        out = subprocess.run([str(exe)] + [str(v) for v in args], capture_output=True, text=True,
                             check=True, timeout=60)
        return int(out.stdout)

    return run


@pytest.fixture(scope="module")
def kernel(program):
    def call(P, B, T, heads, kv, positions, D, ld=4096, shift=4):
        k = min(P, B)
        rows = (B * T * (heads // kv) + k - 1) // k
        return program(rows, k * kv, positions // 32 + 1, B * kv, D, ld, shift)

    return call


def test_forms_of_the_gpu_cases(kernel):
    # many rows of many heads: 35, 70 and 300 sequences of each of four prefixes, 64 key heads
    for each in (35, 70, 300):
        assert kernel(4, 4 * each, 1, 64, 64, 224, 128) == WIDE
    # many rows of a long prefix
    assert kernel(1, 90, 1, 32, 16, 8544, 128, shift=3) == WIDE
    # far pages
    assert kernel(2, 4, 1, 8, 2, 224, 64) == FEW
    assert kernel(2, 20, 1, 8, 2, 224, 64) == SOME
    assert kernel(2, 140, 1, 64, 64, 224, 64) == WIDE
    # one infinite value
    assert kernel(1, 40, 1, 32, 16, 6128, 64) == SOME
    assert kernel(1, 40, 1, 32, 16, 8208, 64) == WIDE
    # long prefixes of few heads
    assert kernel(1, 2, 1, 8, 2, 3008, 128) == FEW
    assert kernel(1, 6, 1, 8, 2, 3008, 128) == SOME
    assert kernel(1, 96, 1, 16, 2, 3008, 128) == SOME


def test_the_ends_of_the_rule(kernel):
    assert kernel(1, 16, 1, 1, 1, 64, 64) == FEW
    assert kernel(1, 17, 1, 1, 1, 64, 64) == SOME
    assert kernel(64, 64 * 16, 1, 1, 1, 64, 64) == FEW
    assert kernel(60, 60 * 17, 1, 1, 1, 64, 64) == SOME   # 1020 of its own
    assert kernel(61, 61 * 17, 1, 1, 1, 64, 64) == WIDE   # 1037
    assert kernel(61, 61 * 17, 1, 1, 1, 64, 256) == SOME
    assert kernel(1, 65, 1, 1, 1, 32 * 4094, 64) == SOME
    assert kernel(1, 65, 1, 1, 1, 32 * 4095, 64) == WIDE
    assert kernel(1, 64, 1, 1, 1, 32 * 4095, 64) == SOME
    assert kernel(1, 257, 1, 1, 1, 32 * 2046, 64) == SOME  # two blocks of rows
    assert kernel(1, 257, 1, 1, 1, 32 * 2047, 64) == WIDE
    # more prefixes than sequences: a sequence's rows are the least
    assert kernel(100, 2, 40, 8, 2, 64, 64) == SOME
    # strides and pages whose offsets pass 32 bits
    assert kernel(61, 61 * 17, 1, 1, 1, 64, 64, ld=1 << 26) == SOME
    assert kernel(61, 61 * 17, 1, 1, 1, 64, 64, ld=1 << 24, shift=6) == WIDE
    assert kernel(61, 61 * 17, 1, 1, 1, 64, 64, ld=1 << 24, shift=7) == SOME


def test_splits(program):
    """In range, one where there is no room for more, and no CU left over where the work is
    a whole number of rounds."""
    for wgs in (1, 8, 32, 100, 256, 5000):
        for tiles in (1, 8, 129, 1025, 1 << 22):
            most = min(64, tiles // 8)
            S = program("splits", wgs, tiles, 0, most)
            assert 1 <= S <= max(most, 1)
    assert program("splits", 64, 1025, 0, 0) == 1
    assert program("splits", 64, 1025, 0, -3) == 1
    assert program("splits", 256, 1 << 20, 0, 64) in range(1, 65)
    assert program("splits", 32, 1025, 4608, 64) == 7
    assert program("splits", 128, 513, 576, 64) == 2
