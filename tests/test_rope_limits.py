"""The rotation's largest calls, without a device (pz_refuse.h)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_threads_of_the_largest_calls_fit_32_bits(tmp_path):
    exe = tmp_path / "rope_limits_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I",
                    os.path.join(ROOT, "project-zero_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "rope_limits_check.cpp"), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout


def test_the_choice_of_kernel_asks():
    text = open(os.path.join(ROOT, "project-zero_amd", "csrc", "pz_rope.hip")).read()
    assert "pz_rope_in_fours(A.n, A.heads[0] + A.heads[1])" in text
