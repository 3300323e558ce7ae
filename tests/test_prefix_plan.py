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
def kernel(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "prefix_plan_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", INC, SRC, "-o", str(exe)],
                   check=True)

    def call(P, B, T, heads, kv, positions, D, ld=4096, shift=4):
        k = min(P, B)
        rows = (B * T * (heads // kv) + k - 1) // k
        args = (rows, k * kv, positions // 32 + 1, D, ld, shift)
        out = subprocess.run([str(exe)] + [str(v) for v in args], capture_output=True, text=True,
                             check=True, timeout=60)
        return int(out.stdout)

    return call


def test_forms_of_the_gpu_cases(kernel):
    # many rows of many heads: 35, 70 and 300 sequences of each of four prefixes, 64 key heads
    assert kernel(4, 140, 1, 64, 64, 224, 128) == SOME
    assert kernel(4, 280, 1, 64, 64, 224, 64) == WIDE
    assert kernel(4, 1200, 1, 64, 64, 80, 128) == WIDE
    # many rows of a long prefix
    assert kernel(1, 90, 1, 32, 16, 8544, 128, shift=3) == WIDE
    assert kernel(1, 80, 1, 32, 16, 6136, 64) == SOME
    assert kernel(1, 80, 1, 32, 16, 8208, 64) == WIDE
    # long prefixes of few heads
    assert kernel(1, 2, 1, 8, 2, 3008, 128) == FEW
    assert kernel(1, 6, 1, 8, 2, 3008, 128) == SOME
    assert kernel(1, 96, 1, 16, 2, 3008, 128) == SOME


def test_the_ends_of_the_rule(kernel):
    assert kernel(1, 16, 1, 1, 1, 64, 64) == FEW
    assert kernel(1, 17, 1, 1, 1, 64, 64) == SOME
    assert kernel(256, 256 * 64, 1, 1, 1, 64, 64) == SOME
    assert kernel(256, 256 * 65, 1, 1, 1, 64, 64) == WIDE
    assert kernel(256, 256 * 65, 1, 1, 1, 64, 256) == SOME
    assert kernel(1, 65, 1, 1, 1, 32 * 4094, 64) == SOME
    assert kernel(1, 65, 1, 1, 1, 32 * 4095, 64) == WIDE
    # more prefixes than sequences: a sequence's rows are the least
    assert kernel(100, 2, 40, 8, 2, 64, 64) == SOME
    # strides and pages whose offsets pass 32 bits
    assert kernel(256, 256 * 65, 1, 1, 1, 64, 64, ld=1 << 26) == SOME
    assert kernel(256, 256 * 65, 1, 1, 1, 64, 64, ld=1 << 24, shift=6) == WIDE
    assert kernel(256, 256 * 65, 1, 1, 1, 64, 64, ld=1 << 24, shift=7) == SOME
