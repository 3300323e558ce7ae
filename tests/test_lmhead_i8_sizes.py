"""The sizes of the 8-bit LM head: what it refuses (on the host) and the largest
vocabularies that it takes."""
import os
import subprocess

import pytest

import pzsample as pz

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "native", "i8_launch_check.cpp")
INC = os.path.join(ROOT, "project-zero_amd", "csrc")


def test_sizes_and_launches(tmp_path):
    exe = tmp_path / "i8_launch_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", INC, SRC, "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    print(out.stdout)
    assert out.returncode == 0, out.stdout


@pytest.mark.gpu
def test_a_launch_that_does_not_fit_is_refused(torch_cuda):
    """Refused on the host, before the buffers (too small for it) are read."""
    torch = torch_cuda
    w = torch.zeros(64, dtype=torch.int8, device="cuda")
    f = torch.zeros(64, device="cuda")
    ids = torch.full((4,), 7, dtype=torch.int32, device="cuda")
    with pz.Sampler(4, 16) as s:
        for V, B in ((1 << 30, 1), ((1 << 30) + 1, 1), (2 ** 31 - 1, 4)):
            with pytest.raises(pz.PzError) as e:
                s.lm_head_argmax_i8(w, f, V, 1, w, f, B, 1, ids)
            assert e.value.code == pz.PZ_ERANGE, V
            with pytest.raises(pz.PzError) as e:
                s.lm_head_i8(w, f, V, 1, w, f, B, 1, f, V)
            assert e.value.code == pz.PZ_ERANGE, V
        s.sync()
    assert (ids == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [16, 7])
def test_many_ids(torch_cuda, n):
    """2^25 + 3 ids: the greedy one is the last, then one in the middle."""
    torch = torch_cuda
    V = (1 << 25) + 3
    w = torch.ones((V, n), dtype=torch.int8, device="cuda")
    sw = torch.ones(V, device="cuda")
    x = torch.ones((2, n), dtype=torch.int8, device="cuda")
    x[1] = -1
    sx = torch.ones(2, device="cuda")
    ids = torch.empty(2, dtype=torch.int32, device="cuda")
    w[V - 1] = 3
    w[V // 2] = -2
    y = torch.empty((2, V), device="cuda")
    with pz.Sampler(2, 16) as s:
        s.lm_head_argmax_i8(w, sw, V, n, x, sx, 2, n, ids)
        s.lm_head_i8(w, sw, V, n, x, sx, 2, n, y, V)
        s.sync()
    assert ids.tolist() == [V - 1, V // 2]
    exp = w.sum(1, dtype=torch.float32)
    assert torch.equal(y, torch.stack([exp, -exp]))
