"""The walk over a page's 16-byte pieces that copies make (pz_pages.h), without a device."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_piece_once_and_an_end(tmp_path):
    exe = tmp_path / "pieces_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I",
                    os.path.join(ROOT, "project-zero_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "pieces_check.cpp"), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout + out.stderr


def test_copies_of_pages_take_it():
    """Both copies of a reordering: no piece's own number is kept in 32 bits."""
    text = open(os.path.join(ROOT, "project-zero_amd", "csrc", "pz_beam.hip")).read()
    assert text.count("for (PzPieces i(") == 2
