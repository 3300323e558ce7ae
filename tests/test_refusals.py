"""Which calls of the logit rules, the 8-bit LM head, the tree attention and the
cache append are refused (pz_refuse.h, host only), where positions of a paged
cache lie (pz_pages.h), and that their entry points
take no null sampler."""
import ctypes
import os
import subprocess

import pzsample as pz

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "native", "refuse_check.cpp")
INC = os.path.join(ROOT, "project-zero_amd", "csrc")


def test_each_wrong_argument_is_refused(tmp_path):
    exe = tmp_path / "refuse_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", INC, SRC, "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    print(out.stdout)
    assert out.returncode == 0, out.stdout


def test_positions_of_bad_pages_and_lengths(tmp_path):
    exe = tmp_path / "pages_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", INC,
                    os.path.join(ROOT, "tests", "native", "pages_check.cpp"), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout


def test_null_sampler():
    lib = pz.load()
    rules, cache = pz.logit_rules(), pz.kv_cache(type=pz.PZ_BF16)
    assert lib.pz_rules_batch(None, 16, 8, 16, 8, 1, 8, ctypes.byref(rules)) == pz.PZ_EINVAL
    assert lib.pz_quant_rows_i8(None, 16, pz.PZ_F32, 8, 1, 8, 16, 8, 16) == pz.PZ_EINVAL
    assert lib.pz_lm_head_i8(None, 16, 16, 8, 8, 16, 16, 1, 8, 16, 8) == pz.PZ_EINVAL
    assert lib.pz_lm_head_argmax_i8(None, 16, 16, 8, 8, 16, 16, 1, 8, 16) == pz.PZ_EINVAL
    assert lib.pz_tree_attention(None, ctypes.byref(cache), 16, 16, 64, 1, 1, None, None, 1, 1.0,
                                 16, 64, 16, 64) == pz.PZ_EINVAL
    assert lib.pz_cache_append(None, ctypes.byref(cache), 16, 16, 64, 1, 1, None,
                               None) == pz.PZ_EINVAL


def test_struct_layouts_match_the_header(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "pz_sampler.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu\\n", offsetof({c}, {n}));\n'
                             for c, s in (("pz_logit_rules", pz.LogitRules),
                                          ("pz_kv_cache", pz.KvCache)) for n, _ in s._fields_)
                   + '  printf("%zu\\n%zu\\n", sizeof(pz_logit_rules), sizeof(pz_kv_cache));\n'
                   "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    want = [getattr(s, n).offset for s in (pz.LogitRules, pz.KvCache) for n, _ in s._fields_]
    assert got == want + [ctypes.sizeof(pz.LogitRules), ctypes.sizeof(pz.KvCache)]
