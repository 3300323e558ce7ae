"""The cache append and what reads the cache after it, ordered by the sampler's
stream (pz_cache_append, pz_tree_attention): the caller keeps the call's
buffers, and the lengths it changes, until the sampler is synchronized."""
import ctypes

import numpy as np
import pytest

import pzsample as pz
from test_gpu_tree import Case

pytestmark = pytest.mark.gpu


def test_a_token_as_a_node_and_then_as_part_of_the_cache(torch_cuda):
    """The second token of a chain: as a node beside the first, and after the
    first one's append, both against the reference."""
    torch = torch_cuda
    c = Case(torch, "bf16", [37, 64], 2, 4, 2, 64, 16, 95)
    exp, tol = c.want()
    with pz.Sampler(1, 16) as s:
        chain = c.run(s, "chain of two")
        d = c.device()
        count = torch.ones(2, dtype=torch.int32, device="cuda")
        s.cache_append(c.cache(d), d["kn"], d["vn"], 128, 2, 2, d_count=count)
        s.sync()  # (the append reads d["lens"])
        d["lens"] += 1
        kn, vn, q = (d[n][:, 1:].contiguous() for n in ("kn", "vn", "q"))
        out = torch.zeros_like(q)
        s.tree_attention(c.cache(d), kn, vn, 128, 2, 1, 4, c.scale, q, 256, out, 256)
        s.sync()
    for got in (out[:, 0], chain[:, 1]):
        got = got.double().cpu().numpy().reshape(2, 4, 64)
        assert (np.abs(got - exp[:, 1]) <= tol[:, 1]).all()


def test_appends_and_attention_without_a_wait_between(torch_cuda):
    """Appends of single tokens and attention over them, one call after the other
    on the sampler's stream, each with lengths of its own: the cache at the end
    and every result as with a wait after each call."""
    torch = torch_cuda
    steps = 6
    c = Case(torch, "fp16", [5, 40, 0], steps, 4, 2, 64, 8, 96)

    def loop(s, wait):
        d = c.device()
        lens = [(d["lens"] + i).contiguous() for i in range(steps + 1)]
        parts = [[d[n][:, i:i + 1].contiguous() for n in ("kn", "vn", "q")] for i in range(steps)]
        outs = [torch.zeros_like(q) for _, _, q in parts]
        caches = [c.cache(dict(d, lens=n)) for n in lens]
        torch.cuda.synchronize()
        for i, (kn, vn, q) in enumerate(parts):
            # (the C calls, which wait for nothing)
            args = (s.h, ctypes.byref(caches[i]), kn.data_ptr(), vn.data_ptr(), 128, 3, 1)
            assert s.lib.pz_tree_attention(*args, None, None, 4, c.scale, q.data_ptr(), 256,
                                           outs[i].data_ptr(), 256) == 0
            if wait:
                s.sync()
            assert s.lib.pz_cache_append(*args, None, None) == 0
            if wait:
                s.sync()
        s.sync()
        return torch.cat(outs, 1), d["k"], d["v"]

    with pz.Sampler(1, 16) as s:
        apart, together = loop(s, True), loop(s, False)
    for a, b in zip(apart, together):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    exp, tol = c.want()  # (a chain: node i sees the cache and nodes 0 .. i)
    got = together[0].double().cpu().numpy().reshape(exp.shape)
    assert (np.abs(got - exp) <= tol).all()
