"""The exponential of beam selection (pz_beamexp.h) over its whole range, without a device."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = tmp_path_factory.mktemp("exp") / "beam_exp_check"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I",
                    os.path.join(ROOT, "project-zero_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "beam_exp_check.cpp"), "-o", str(exe)],
                   check=True)

    def run(*args):
        out = subprocess.run([str(exe)] + [str(a) for a in args], capture_output=True, text=True,
                             timeout=100)
        assert out.returncode == 0, out.stdout
        return float(out.stdout.split()[0])

    return run


def test_off_by_at_most_2_43(program):
    """Every table entry is 2^(i / 32) as the definition has it, and no result is off by more
    than the stated 2^-43 of itself (the long double reference by 2^-62 of that)."""
    assert program() <= 1.0


@pytest.mark.parametrize("entry", [0, 1, 17, 31])
def test_a_wrong_entry_is_seen(program, entry):
    """One that is off by 2^-43 of itself or more."""
    assert program(entry) > 1.0
