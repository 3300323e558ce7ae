"""The 8-bit LM head's tile rule (pz_lmtile.h): the cases of
test_gpu_lmhead_i8.py launch every shape, and a shape serves the batch it is
taken for."""
import os
import subprocess

from test_gpu_lmhead_i8 import I8_TILE_BATCHES, I8_TILE_VOCABS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "native", "i8_tile_check.cpp")
INC = os.path.join(ROOT, "project-zero_amd", "csrc")


def tiles(tmp_path, cases, *how):
    exe = tmp_path / "i8_tile_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", INC, SRC, "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe), *how] + [str(v) for c in cases for v in c], capture_output=True,
                         text=True, timeout=60, check=True)
    count, *got = [int(v) for v in out.stdout.split()]
    return count, got


def test_the_gpu_cases_reach_every_shape(tmp_path):
    count, got = tiles(tmp_path, [(B, V) for B in I8_TILE_BATCHES for V in I8_TILE_VOCABS])
    assert set(got) == set(range(count))


def test_the_gpu_cases_reach_every_shape_of_odd_rows(tmp_path):
    count, got = tiles(tmp_path, [(B, V) for B in I8_TILE_BATCHES for V in I8_TILE_VOCABS], "odd")
    assert set(got) == set(range(count))


def test_the_ends_of_the_rule_of_odd_rows(tmp_path):
    _, got = tiles(tmp_path, [(1, 1), (16, 2 ** 31 - 1), (17, 1), (64, 2 ** 31 - 1), (65, 1),
                              (100000, 2 ** 31 - 1)], "odd")
    assert got == [0, 1, 2, 4, 5, 7]


def test_the_ends_of_the_rule(tmp_path):
    _, got = tiles(tmp_path, [(1, 1), (1, 2 ** 31 - 1), (16, 2 ** 31 - 1), (17, 1), (256, 1),
                              (257, 1), (100000, 1), (100000, 2 ** 31 - 1)])
    # (100000 rows: 391 blocks of one row of W each, 1.5 rows per CU)
    assert got == [0, 1, 2, 3, 15, 15, 15, 19]
