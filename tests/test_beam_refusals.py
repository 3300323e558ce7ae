"""Which calls of prefix attention, the rotation and the beam search are refused
(pz_refuse.h, host only), that their entry points take no null sampler, and the layout of
their structs."""
import ctypes
import os
import subprocess

import pzsample as pz

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INC = os.path.join(ROOT, "project-zero_amd", "csrc")


def test_each_wrong_argument_is_refused(tmp_path):
    exe = tmp_path / "beam_refuse_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", INC,
                    os.path.join(ROOT, "tests", "native", "beam_refuse_check.cpp"), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout


def test_null_sampler():
    lib = pz.load()
    cache, prefix, rope = pz.kv_cache(type=pz.PZ_BF16), pz.kv_prefix(), pz.qk_rope()
    assert lib.pz_prefix_attention(None, ctypes.byref(cache), ctypes.byref(prefix), 16, 16, 64, 1,
                                   1, None, None, 1, 1.0, 16, 64, 16, 64) == pz.PZ_EINVAL
    assert lib.pz_qk_norm_rope(None, ctypes.byref(rope), 16, 64, 16, 64, 16, 64, 16, 64, 1,
                               16) == pz.PZ_EINVAL
    assert lib.pz_beam_select(None, 16, 8, 1, 1, 8, 16, None, 0, 1, 16, 16, 16,
                              None) == pz.PZ_EINVAL
    assert lib.pz_beam_reorder(None, (pz.KvCache * 1)(cache), 1, 1, 1, 16, 16, 1, 1, 32, 32,
                               None) == pz.PZ_EINVAL


def test_struct_layouts_match_the_header(tmp_path):
    src = tmp_path / "layout.c"
    structs = (("pz_kv_prefix", pz.KvPrefix), ("pz_qk_rope", pz.QkRope))
    src.write_text('#include <stdio.h>\n#include "pz_sampler.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu\\n", offsetof({c}, {n}));\n'
                             for c, s in structs for n, _ in s._fields_)
                   + "".join(f'  printf("%zu\\n", sizeof({c}));\n' for c, _ in structs)
                   + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    want = [getattr(s, n).offset for _, s in structs for n, _ in s._fields_]
    assert got == want + [ctypes.sizeof(s) for _, s in structs]


def test_constants_match_the_header():
    text = open(os.path.join(ROOT, "include", "pz_sampler.h")).read()
    for name in ("PZ_ROPE_HALVES", "PZ_ROPE_PAIRS", "PZ_BEAM_MAX_WIDTH", "PZ_BEAM_MAX_SELECT",
                 "PZ_BEAM_WORKSPACE", "PZ_BEAM_MAX_POOL", "PZ_BEAM_MAX_BEAMS"):
        line = next(li for li in text.splitlines() if li.startswith(f"#define {name} "))
        assert eval(line.split(None, 2)[2]) == getattr(pz, name), name
