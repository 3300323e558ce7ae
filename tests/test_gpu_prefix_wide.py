"""Prefix attention's kernel for many rows with several nodes a sequence and several query
heads a key head (test_prefix_wide_plan.py: these cases take it).  Reference and bound: those
of test_gpu_prefix.py, on some of the sequences of each batch."""
import copy

import numpy as np
import pytest

import pzsample as pz
from test_gpu_prefix import Shared

pytestmark = pytest.mark.gpu

HEADS, KV = 32, 8
FIRST = [3, 70, 75, 75, 138]  # (the first three and the last two have none, one range none)
LENS = [200, 0, 129, 65]


@pytest.fixture(scope="module")
def sampler(torch_cuda):
    with pz.Sampler(1, 16) as s:
        yield s


def some(c, bs):
    """The case of sequences bs alone, as its check() needs it."""
    p = copy.copy(c)
    p.B, p.of, p.lens = len(bs), [c.of[b] for b in bs], c.lens[bs]
    p.table = c.table[bs]
    for n in ("q", "kn", "vn"):
        setattr(p, n, getattr(c, n)[bs])
    p.tree = None if c.tree is None else c.tree[bs]
    p.n_nodes = None if c.n_nodes is None else [c.n_nodes[b] for b in bs]
    return p


def attend(s, c):
    d = c.device()
    c.call(s, d)
    s.sync()
    return d["out"]


def counts(B, T, seed):
    """Nodes of B sequences: all, some, none, and counts outside 0 .. T."""
    n = np.random.default_rng(seed).integers(-1, T + 2, B)
    n[::3] = T
    return [int(x) if x <= T else 99 for x in n]


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [3, 5])  # (16 and 32 own rows a wave)
def test_nodes_of_many_sequences(torch_cuda, sampler, kind, D, T):
    """Trees, counts, ranges with gaps, a prefix of no position, pages that are missing."""
    c = Shared(torch_cuda, kind, LENS, FIRST, [b % 45 for b in range(140)], T, HEADS, KV, D, 16,
               seed=T + D).random_tree(T)
    bs = [0, 2, 3, 4, 37, 69, 70, 71, 74, 75, 76, 100, 101, 136, 137, 138, 139]
    some(c, bs).check(attend(sampler, c)[bs], "whole")
    c.n_nodes = counts(140, T, D)
    c.tree[5, 0] = 0
    for b in range(140):  # (queries behind the last node may be anything)
        c.q[b, max(c.n_nodes[b], 0):] = float("nan")
    c.ptable[0, 1] = -1
    c.ptable[3, 0] = c.n_pages
    c.table[4, 0] = 2 ** 31 - 1
    some(c, bs + [5]).check(attend(sampler, c)[bs + [5]], "counts, missing pages")


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("fp16", 64)])
def test_drafts_under_prompts(torch_cuda, sampler, kind, D):
    """64 sequences of 5 drafts under four prompts, in splits."""
    c = Shared(torch_cuda, kind, [2100, 1024, 1987, 33], None, [7 * b % 50 for b in range(64)], 5,
               HEADS, KV, D, 16, seed=D).random_tree(8)
    bs = [0, 15, 16, 31, 32, 47, 48, 63]
    some(c, bs).check(attend(sampler, c)[bs], "trees")
    c.tree = None
    c.ptable[0, 40:45] = -1
    some(c, bs).check(attend(sampler, c)[bs], "chains, missing pages")


def test_own_positions_in_splits(torch_cuda, sampler):
    """128 units of waves, two splits of the sequences' own keys; most sequences have one."""
    lens = [(600, 3, 257, 511, 0, 64, 512, 40)[b % 8] for b in range(128)]
    for kind, D in (("bf16", 64), ("fp16", 128)):
        c = Shared(torch_cuda, kind, [2100], None, lens, 3, HEADS, KV, D, 16,
                   seed=D + 1).random_tree(9)
        c.n_nodes = counts(128, 3, 1)
        bs = [0, 1, 2, 3, 4, 5, 6, 64, 65, 66, 120, 126, 127]
        some(c, bs).check(attend(sampler, c)[bs], (kind, D))


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_nodes_that_are_not_seen(torch_cuda, sampler, kind):
    """NaN and infinities of nodes that a row does not see leave it within its bound; a row
    that sees a NaN is one."""
    torch, T = torch_cuda, 5
    c = Shared(torch, kind, LENS, FIRST, [b % 45 for b in range(140)], T, HEADS, KV, 64, 16,
               seed=21).random_tree(5)
    bs = list(range(0, 140, 6))
    want, tol = some(c, bs).want()
    c.vn[:, 1] = float("nan")
    c.vn[:, 2, ::3] = float("inf")
    c.kn[:, 3] = float("nan")
    got = attend(sampler, c)[bs].double().cpu().numpy().reshape(want.shape)
    blind = hit = 0
    for i, b in enumerate(bs):
        for t in range(T):
            bits = int(c.tree[b, t])
            if not bits & 0b01110:
                blind += 1
                assert (np.abs(got[i, t] - want[i, t]) <= tol[i, t]).all(), (b, t)
            elif bits & 0b01010:
                hit += 1
                assert np.isnan(got[i, t]).any(), (b, t)
    assert blind > 20 and hit > 20


def test_more_rows_than_the_workspace(torch_cuda, sampler):
    """403 sequences are as many as its two parts hold: the others follow, from inside a
    prefix on."""
    B, T, D = 500, 5, 128
    assert (64 << 20) // (2 * (D + 2) * 4) // (T * HEADS) == 403
    c = Shared(torch_cuda, "bf16", [150, 90, 33], [2, 380, 450, 499], [b % 20 for b in range(B)],
               T, HEADS, KV, D, 16, seed=61).random_tree(7)
    c.n_nodes = counts(B, T, 3)
    bs = [0, 1, 2, 379, 380, 402, 403, 404, 449, 450, 498, 499]
    some(c, bs).check(attend(sampler, c)[bs])


def test_replayed(torch_cuda, sampler):
    """Captured, then replayed on new rows and longer sequences and prefixes, eager calls
    between: every replay against an eager call, the last against the reference."""
    torch, T = torch_cuda, 5
    c = Shared(torch, "bf16", [150, 90, 33, 60], FIRST, [b % 40 for b in range(140)], T, HEADS, KV,
               64, 16, seed=99, spare=2, pspare=2).random_tree(9)
    for name in ("k", "v"):  # (positions that lengths reach later)
        t = getattr(c, name)
        t[torch.isnan(t)] = 0.5
    d = c.device()
    c.call(sampler, d)
    sampler.sync()
    cache, prefix = c.cache(d), c.prefix(d)
    row, q = KV * 64, HEADS * 64

    def call(out):
        assert sampler.lib.pz_prefix_attention(
            sampler.h, pz.ctypes.byref(cache), pz.ctypes.byref(prefix), d["kn"].data_ptr(),
            d["vn"].data_ptr(), row, 140, T, None, d["tree"].data_ptr(), HEADS, c.scale,
            d["q"].data_ptr(), q, out.data_ptr(), q) == 0
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(sampler.stream)):
        call(d["out"])
    eager = torch.empty_like(d["out"])
    for i in range(4):
        for n in ("kn", "vn", "q"):
            d[n].normal_()
        d["lens"] += 2
        d["plens"] += 3
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager.zero_()
        torch.cuda.synchronize()
        call(eager)
        sampler.sync()
        assert torch.equal(eager, d["out"]), i
    for n in ("kn", "vn", "q"):
        setattr(c, n, d[n].cpu())
    c.lens, c.plens = d["lens"].cpu().numpy(), d["plens"].cpu().numpy()
    bs = [0, 3, 69, 70, 74, 75, 137, 139]
    some(c, bs).check(d["out"][bs], "the last")


@pytest.mark.parametrize("kv,B,positions", [(1, 2, 300), (1, 2, 700), (512, 1, 300), (256, 1, 700)])
def test_the_most_rows_of_a_sequence(torch_cuda, sampler, kv, B, positions):
    """32768 of 64 elements, and no more: 512 heads of 64 nodes, over one key head to one
    each."""
    T, heads, D = 64, 512, 64
    c = Shared(torch_cuda, "bf16", [positions], None, [40, 0][:B], T, heads, kv, D, 16,
               seed=kv + positions).random_tree(3)
    c.run(sampler, (kv, positions))
