"""Which kernel tree attention takes (pz_treeplan.h): the GPU cases run the ones that
they are made for, so that none of them passes by another's work."""
import os
import subprocess

import pytest
from test_gpu_tree_far import FAR, POSITIONS, table_of
from test_gpu_tree_range import FORMS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "native", "tree_plan_check.cpp")
INC = os.path.join(ROOT, "project-zero_amd", "csrc")
FEW_SHORT, FEW, SOME, WIDE16, WIDE32 = range(5)


@pytest.fixture(scope="module")
def kernel(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "tree_plan_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", INC, SRC, "-o", str(exe)],
                   check=True)

    def call(B, T, heads, kv, positions, D, ld=4096, ld_n=4096):
        tiles = positions // 32 + 1 + (T + 31) // 32
        args = (T * (heads // kv), B * kv, tiles, D, ld, ld_n)
        out = subprocess.run([str(exe)] + [str(v) for v in args], capture_output=True, text=True,
                             check=True, timeout=60)
        return int(out.stdout)

    return call


def test_forms_of_the_range_tests(kernel):
    got = {}
    for name, (B, T, heads, kv, ctx) in FORMS.items():
        per = (ctx + T + 15) // 16 + 2  # (the tables that the cases make)
        got[name] = kernel(B, T, heads, kv, per * 16, 64)
    assert got == {"one tile": FEW_SHORT, "two row tiles": SOME, "splits": FEW,
                   "many splits of more rows": SOME, "many rows": WIDE16,
                   "many rows, two tiles a wave": WIDE32, "many rows in splits": WIDE16,
                   "many rows in splits, two tiles a wave": WIDE32}


def test_far_strides(kernel):
    """The wide kernels up to the strides whose offsets fit, the others past them."""
    for name, (T, heads, kv, ld, ld_n, wide) in FAR.items():
        got = kernel(1, T, heads, kv, table_of(kv) * 8, 64, ld, ld_n)
        want = (WIDE16 if T * heads // kv <= 64 else WIDE32) if wide else SOME
        assert got == want, name
    assert POSITIONS < table_of(2) * 8


def test_the_ends_of_the_rule(kernel):
    assert kernel(1, 1, 1, 1, 640, 128) == FEW_SHORT
    assert kernel(1, 1, 1, 1, 1024, 128) == FEW
    assert kernel(1, 1, 1, 1, 640, 256) == FEW
    assert kernel(512, 1, 1, 1, 64, 64) == FEW
    assert kernel(1, 17, 1, 1, 64, 64) == SOME
    assert kernel(256, 32, 1, 1, 64, 64) == SOME
    assert kernel(256, 33, 1, 1, 64, 64) == WIDE16
    assert kernel(256, 64, 2, 1, 64, 64) == WIDE32
    assert kernel(256, 64, 2, 1, 64, 256) == SOME
    assert kernel(1, 64, 1, 1, 130000, 64) == SOME
    assert kernel(1, 64, 1, 1, 131072, 64) == WIDE16
