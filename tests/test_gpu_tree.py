"""Attention of drafted trees over a paged cache (pz_tree_attention) and the
append that fills the pages (pz_cache_append).

Reference: 64-bit softmax attention of the same 16-bit inputs.  Bound per
result, with h = eps / 2 of the type (a rounding to it, relative), P the exact
softmax weights of the row:
  |got - o| <= h |o| + (h + d) (1 + h) sum_p P |v|  + tiny
The result is rounded once (h |o|); every weight is rounded once (h) and its
relative error before that is at most d = 2 max_p |s_p error| + 2^-20 + n 2^-23,
where the score (base e) is an fp32 sum of D exact products, off by at most
(D + 2) 2^-24 scale sum_j |q_j k_j|, its use as exp2(fma(s, c, -m)) adds
2 |s c| 2^-24 (c and the fma rounded) and the hardware's exp2 a few ulp; n 2^-23
bounds the fp32 sums of weights and products over n keys.  The factor 2: the
weight's own error and the normaliser's.  fp16 weights below 2^-14 (relative to
a row maximum scaled to 2^8 or more) lose at most 2^-25 each, 2^-33 of the
maximum, which n keys and the largest |v| bound; fp16 results below 2^-14 lose
2^-25."""
import numpy as np
import pytest

import pzsample as pz

pytestmark = pytest.mark.gpu

KINDS = {"bf16": (pz.PZ_BF16, 2.0 ** -8, "bfloat16"), "fp16": (pz.PZ_F16, 2.0 ** -11, "float16")}


class Case:
    """B sequences over a shuffled paged cache whose other slots hold NaN."""

    def __init__(self, torch, kind, lens, T, heads, kv, D, page, seed, sigma=1.0, spare=2,
                 extra=0):
        self.torch, self.kind, self.T, self.heads, self.kv = torch, kind, T, heads, kv
        self.D, self.page = D, page
        B = self.B = len(lens)
        self.lens = np.asarray(lens, np.int32)
        self.dt = getattr(torch, KINDS[kind][2])
        g = torch.Generator().manual_seed(seed)
        self.per = (max(max(lens), 1) + T + page - 1) // page + spare
        n_pages = B * self.per + 3
        self.table = torch.randperm(n_pages, generator=g)[:B * self.per].reshape(B, self.per)
        self.table = self.table.to(torch.int32)
        self.n_pages = n_pages
        nan = float("nan")
        row = kv * D + extra
        self.k = torch.full((n_pages * page, row), nan, dtype=self.dt)
        self.v = torch.full((n_pages * page, row), nan, dtype=self.dt)
        for b in range(B):
            p = torch.arange(int(lens[b]))
            at = self.slots(b, p)
            self.k[at, :kv * D] = (torch.randn((len(p), kv * D), generator=g)).to(self.dt)
            self.v[at, :kv * D] = (torch.randn((len(p), kv * D), generator=g)).to(self.dt)
        self.kn = torch.randn((B, T, row), generator=g).to(self.dt)
        self.vn = torch.randn((B, T, row), generator=g).to(self.dt)
        self.q = (torch.randn((B, T, heads * D + extra), generator=g) * sigma).to(self.dt)
        self.scale = D ** -0.5
        self.n_nodes = None
        self.tree = None

    def slots(self, b, p):
        return self.table[b].long()[p // self.page] * self.page + p % self.page

    def random_tree(self, seed):
        rng = np.random.default_rng(seed)
        sees = np.zeros((self.B, self.T), np.uint64)
        for b in range(self.B):
            for t in range(self.T):
                sees[b, t] = np.uint64(1) << np.uint64(t)
                if t:
                    sees[b, t] |= sees[b, rng.integers(0, t)]
        self.tree = sees
        return self

    def want(self):
        """(results, bounds) float64 [B, T, heads, D]; NaN-marked where no row
        is written."""
        T, D, group = self.T, self.D, self.heads // self.kv
        _, h, _ = KINDS[self.kind]
        out = np.full((self.B, T, self.heads, D), np.nan)
        tol = np.zeros_like(out)
        for b in range(self.B):
            nn = T if self.n_nodes is None else min(max(int(self.n_nodes[b]), 0), T)
            ctx = min(max(int(self.lens[b]), 0), self.per * self.page)
            pos = np.arange(ctx)
            pages = self.table[b].numpy()[pos // self.page]
            ok = (pages >= 0) & (pages < self.n_pages)
            at = np.where(ok, pages, 0) * self.page + pos % self.page
            for hk in range(self.kv):
                sl = slice(hk * D, hk * D + D)
                k = np.concatenate([self.k[at, sl].double().numpy(),
                                    self.kn[b, :, sl].double().numpy()])
                v = np.concatenate([self.v[at, sl].double().numpy(),
                                    self.vn[b, :, sl].double().numpy()])
                for t in range(nn):
                    bits = (int(self.tree[b, t]) if self.tree is not None else (2 << t) - 1)
                    see = np.concatenate([ok, [(bits >> u & 1) == 1 and u < nn for u in range(T)]])
                    if not see.any():
                        out[b, t, hk * group:(hk + 1) * group] = 0.0
                        continue
                    ks, vs = k[see], v[see]
                    for j in range(hk * group, (hk + 1) * group):
                        q = self.q[b, t, j * D:(j + 1) * D].double().numpy()
                        s = ks @ q * self.scale
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        o = p @ vs
                        n = len(ks)
                        err = ((D + 2) * 2.0 ** -24 * self.scale * (np.abs(ks) @ np.abs(q)).max()
                               + 2 * np.abs(s).max() * 2.0 ** -24)
                        d = 2 * err + 2.0 ** -20 + n * 2.0 ** -23
                        out[b, t, j] = o
                        tol[b, t, j] = (h * np.abs(o) + (h + d) * (1 + h) * (p @ np.abs(vs))
                                        + (n * 2.0 ** -33 * np.abs(vs).max() + 2.0 ** -25
                                           if self.kind == "fp16" else 0.0))
        return out, tol

    def cache(self, d):
        return pz.kv_cache(type=KINDS[self.kind][0], n_kv_heads=self.kv, head_dim=self.D,
                           d_k=d["k"], d_v=d["v"], ld=self.k.shape[1], n_blocks=self.n_pages,
                           block_size=self.page, d_blocks=d["table"], max_blocks=self.per,
                           d_len=d["lens"])

    def device(self):
        t = self.torch
        d = {n: getattr(self, n).cuda() for n in ("k", "v", "kn", "vn", "q", "table")}
        d["lens"] = t.from_numpy(self.lens).cuda()
        d["n_nodes"] = None if self.n_nodes is None else t.tensor(self.n_nodes,
                                                                  dtype=t.int32).cuda()
        d["tree"] = None if self.tree is None else t.from_numpy(self.tree.view(np.int64)).cuda()
        d["out"] = t.full_like(d["q"], 77.0)
        return d

    def call(self, s, d):
        s.tree_attention(self.cache(d), d["kn"], d["vn"], self.kn.shape[2], self.B, self.T,
                         self.heads, self.scale, d["q"], self.q.shape[2], d["out"],
                         self.q.shape[2], d["n_nodes"], d["tree"])

    def check(self, out, label=""):
        exp, tol = self.want()
        w = self.heads * self.D
        got = out[:, :, :w].double().cpu().numpy().reshape(exp.shape)
        idle = np.isnan(exp).all(3) & (tol.max(3) == 0)
        for b in range(self.B):
            nn = self.T if self.n_nodes is None else min(max(int(self.n_nodes[b]), 0), self.T)
            idle[b, :nn] = False
        assert (got[idle] == 77.0).all(), (label, "rows behind the last node")
        assert (out[:, :, w:].float() == 77.0).all(), (label, "past the heads")
        g, e, t = got[~idle], exp[~idle], tol[~idle]
        assert (np.isnan(g) == np.isnan(e)).all(), (label, "NaN")
        fin = ~np.isnan(e)
        off = np.abs(g - e)[fin] - t[fin]
        assert (off <= 0).all(), (label, off.max(), (np.abs(g - e)[fin] / (t[fin] + 1e-30)).max())

    def run(self, s, label=""):
        d = self.device()
        self.call(s, d)
        s.sync()
        self.check(d["out"], label)
        return d["out"]


@pytest.fixture(scope="module")
def sampler(torch_cuda):
    with pz.Sampler(1, 16) as s:
        yield s


SHAPES = [(8, 2), (4, 4), (20, 5), (16, 1), (3, 1)]


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 2, 5, 17, 33, 64])
def test_trees(torch_cuda, sampler, kind, D, T):
    for i, (heads, kv) in enumerate(SHAPES):
        lens = [0, 1, 31, 33, 100][i % 2:]
        Case(torch_cuda, kind, lens, T, heads, kv, D, 16, 100 * T + i).random_tree(T + i).run(
            sampler, (kind, D, T, heads, kv))


@pytest.mark.parametrize("kind,D", [("bf16", 64), ("bf16", 128), ("fp16", 128), ("bf16", 256)])
def test_chains_over_long_contexts(torch_cuda, sampler, kind, D):
    """d_tree NULL, lengths of every remainder, split and unsplit."""
    Case(torch_cuda, kind, [2049, 777, 4000, 5], 5, 8, 2, D, 32, 3).run(sampler, "split")
    Case(torch_cuda, kind, list(range(60, 100)), 3, 4, 2, D, 8, 4).run(sampler, "remainders")
    Case(torch_cuda, kind, [9001], 1, 4, 4, D, 256, 5, sigma=4.0).run(sampler, "one token")
    Case(torch_cuda, kind, [300] * 150, 1, 8, 8, D, 64, 6).run(sampler, "no split")


@pytest.mark.parametrize("page", [8, 16, 64, 512])
def test_pages_and_strides(torch_cuda, sampler, page):
    Case(torch_cuda, "bf16", [1, 7, 8, 9, 515], 4, 6, 3, 64, page, page, extra=24).random_tree(
        1).run(sampler, page)


def test_lengths_and_counts_outside_their_range(torch_cuda, sampler):
    c = Case(torch_cuda, "bf16", [40, 40, 40, 40, 40, 40], 6, 4, 2, 64, 16, 11).random_tree(2)
    c.n_nodes = [0, -1, 1, 5, 6, 99]
    c.run(sampler, "counts")
    c.lens = np.array([-4, 0, 1, 40, 39, 17], np.int32)
    c.run(sampler, "lengths")
    full = Case(torch_cuda, "bf16", [48, 48], 2, 4, 2, 64, 16, 12, spare=0)
    full.per = 3
    full.table = full.table[:, :3].contiguous()
    full.run(sampler, "a full table")
    full.lens = np.array([48, 2 ** 31 - 1], np.int32)  # as long as the table at most
    full.run(sampler, "a length past it")


def test_pages_outside_the_cache_hold_nothing(torch_cuda, sampler):
    c = Case(torch_cuda, "fp16", [100, 100, 100], 3, 4, 2, 128, 16, 21).random_tree(3)
    c.table[0, 2] = -1
    c.table[1, 0] = c.n_pages
    c.table[1, 6] = 2 ** 31 - 1
    c.table[2, :] = -(2 ** 31)
    c.run(sampler)


def test_rows_that_see_nothing(torch_cuda, sampler):
    for T in (3, 40):
        c = Case(torch_cuda, "bf16", [0, 0, 50], T, 4, 2, 64, 16, 31).random_tree(4)
        c.tree[0, :] = 0
        c.tree[1, 1:] = 0
        c.tree[2, ::2] = 0
        # bits past the last node count for nothing
        c.n_nodes = [T, T, T - 1]
        c.tree[1, 0] |= np.uint64(~((1 << T) - 1) & (2 ** 64 - 1))
        c.run(sampler, T)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("spare", [2, 1400])
def test_what_is_not_seen_has_no_influence(torch_cuda, sampler, kind, spare):
    """NaN and infinities in nodes that a row does not see leave it as it is;
    rows that see them get what the sum gives."""
    torch = torch_cuda
    for T, D in ((6, 64), (40, 128), (33, 256)):
        c = Case(torch, kind, [70, 0, 33], T, 8, 2, D, 16, 41, spare=spare).random_tree(5)
        clean = c.run(sampler, "clean")
        c.vn[:, 2] = float("nan")
        c.vn[:, 3, ::3] = float("inf")
        c.kn[:, 4] = float("nan")
        c.kn[:, 5] = float("inf")
        d = c.device()
        c.call(sampler, d)
        sampler.sync()
        got = d["out"]
        for b in range(3):
            for t in range(T):
                bits = int(c.tree[b, t])
                if not bits & 0b111100:
                    assert torch.equal(got[b, t], clean[b, t]), (T, b, t)
                elif bits & 0b010100:
                    assert torch.isnan(got[b, t].float()).any(), (T, b, t)
        # one row by hand: it sees an infinite value and no NaN
        for b in range(3):
            for t in range(T):
                bits = int(c.tree[b, t])
                if bits & 8 and not bits & 0b110100:
                    o = got[b, t, :8 * D].float().reshape(8, D)
                    at = torch.arange(2 * D).reshape(2, D).repeat_interleave(4, 0) % 3 == 0
                    assert torch.isinf(o.cpu()[at]).all() and (o.cpu()[at] > 0).all(), (b, t)
                    assert torch.isfinite(o.cpu()[~at]).all(), (b, t)


@pytest.mark.parametrize("kind,D", [("bf16", 64), ("bf16", 128), ("fp16", 128), ("fp16", 64)])
@pytest.mark.parametrize("T", [6, 16, 17, 40, 64])
@pytest.mark.parametrize("spare", [2, 900])
def test_many_rows_in_splits(torch_cuda, sampler, kind, D, T, spare):
    """Sequences of several splits, of one and of none, tiles that end early and
    pages that are missing in the middle, at a range's ends and throughout, for
    rows that fill their waves and rows that do not, in tables that are short
    and long."""
    c = Case(torch_cuda, kind, [1500, 0, 31, 1000, 257], T, 16, 2, D, 16, 7 * T,
             spare=spare).random_tree(T)
    c.n_nodes = [T, T - 1, T, 1, T // 2]
    c.table[0, 20] = -1
    c.table[0, 93] = c.n_pages
    c.table[3, 0] = 2 ** 31 - 1
    c.table[4, 16] = -5
    c.run(sampler, (kind, D, T))
    c.table[3, :] = -1
    c.run(sampler, "a sequence without pages")


def test_many_rows_of_long_tables(torch_cuda, sampler):
    """Tables of more entries than a workgroup keeps at hand."""
    c = Case(torch_cuda, "bf16", [300, 7] * 16, 9, 64, 8, 64, 8, 77)
    small = c.per
    c.per = 4500
    table = torch_cuda.full((32, c.per), -1, dtype=torch_cuda.int32)
    table[:, :small] = c.table
    c.table = table
    c.run(sampler)
    c.lens[3] = 2 ** 31 - 1  # all of the table: entries of no page from the first ones on
    c.run(sampler, "the whole table")


def test_many_sequences_of_long_tables(torch_cuda, sampler):
    """As many entries in tables of many sequences."""
    c = Case(torch_cuda, "bf16", [40, 7] * 32, 33, 32, 32, 64, 8, 79)
    c.n_nodes = [0] * 64
    c.n_nodes[5], c.n_nodes[62] = 33, 20
    small = c.per
    c.per = 4500
    table = torch_cuda.full((64, c.per), -1, dtype=torch_cuda.int32)
    table[:, :small] = c.table
    c.table = table
    c.run(sampler)


def test_many_rows_of_a_long_sequence(torch_cuda, sampler):
    """Positions whose table entries lie past those at hand, some without a page."""
    c = Case(torch_cuda, "bf16", [16700, 7, 7, 7, 7, 7, 7, 40], 33, 32, 32, 64, 8, 80)
    c.n_nodes = [2, 0, 0, 0, 0, 0, 0, 33]
    c.table[0, 2050] = -1
    c.table[0, 2087] = c.n_pages
    c.run(sampler)


def test_many_rows_of_far_slots(torch_cuda, sampler):
    """Slots 128 MiB apart: a tile's rows pass 32 bits of offsets."""
    torch = torch_cuda
    c = Case(torch, "bf16", [13], 12, 8, 2, 64, 8, 78, spare=0)
    d = c.device()
    ld, pages = 1 << 26, c.per
    pool = torch.empty(((pages * 8 - 1) * ld + 1024,), dtype=torch.bfloat16, device="cuda")
    at = torch.arange(pages)
    for name, first in (("k", 0), ("v", 512)):
        rows = getattr(c, name)[c.slots(0, torch.arange(pages * 8))].cuda()
        pool[first:].as_strided((pages * 8, 128), (ld, 1)).copy_(rows)
    cache = pz.kv_cache(type=pz.PZ_BF16, n_kv_heads=2, head_dim=64, d_k=pool, d_v=pool[512:], ld=ld,
                        n_blocks=pages, block_size=8, d_blocks=at.int().reshape(1, -1).cuda(),
                        max_blocks=pages, d_len=d["lens"])
    sampler.tree_attention(cache, d["kn"], d["vn"], 128, 1, 12, 8, c.scale, d["q"], 512, d["out"],
                           512)
    sampler.sync()
    c.check(d["out"])


def test_large_scores(torch_cuda, sampler):
    """Scores far apart: one key takes all the weight, wherever it lies."""
    for kind in KINDS:
        c = Case(torch_cuda, kind, [500, 1000], 4, 4, 2, 64, 16, 51, sigma=40.0).random_tree(6)
        c.run(sampler, kind)
        c = Case(torch_cuda, kind, [500], 1, 2, 2, 64, 16, 52)
        c.k[c.slots(0, c.torch.arange(500))] *= 0.0
        c.run(sampler, (kind, "equal scores"))


def test_same_inputs_same_bits(torch_cuda, sampler):
    c = Case(torch_cuda, "bf16", [3000, 10, 700], 7, 8, 2, 128, 16, 61).random_tree(7)
    d = c.device()
    c.call(sampler, d)
    sampler.sync()
    first = d["out"].clone()
    for _ in range(3):
        d["out"].fill_(5.0)
        c.call(sampler, d)
        sampler.sync()
        assert torch_cuda.equal(d["out"], first)


def test_a_far_cache(torch_cuda, sampler):
    """Slots whose byte offsets pass 2^32 (a cache of 6 GiB, used at its end)."""
    torch = torch_cuda
    c = Case(torch, "bf16", [90], 2, 4, 2, 64, 16, 71)
    d = c.device()
    ld, pages = 2048, 1 << 16  # 2^20 slots of 4 KiB and more
    k = torch.empty((pages * 16 * ld + (2 << 30),), dtype=torch.bfloat16, device="cuda")
    far = pages - 1 - torch.arange(c.per, dtype=torch.int32)
    for name in ("k", "v"):
        at = (far.long()[:, None] * 16 + torch.arange(16)).reshape(-1)
        rows = getattr(c, name)[c.slots(0, torch.arange(c.per * 16))].cuda()
        dst = k[(0 if name == "k" else 1024):].as_strided((pages * 16, 128), (ld, 1))
        dst[at.cuda()] = rows
    cache = pz.kv_cache(type=pz.PZ_BF16, n_kv_heads=2, head_dim=64, d_k=k, d_v=k[1024:], ld=ld,
                        n_blocks=pages, block_size=16, d_blocks=far.reshape(1, -1).cuda(),
                        max_blocks=c.per, d_len=d["lens"])
    sampler.tree_attention(cache, d["kn"], d["vn"], 128, 1, 2, 4, c.scale, d["q"], 256, d["out"],
                           256)
    sampler.sync()
    c.check(d["out"])


# ---- append --------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("D,kv,page,extra", [(64, 1, 8, 0), (128, 8, 16, 8), (256, 3, 64, 0)])
def test_append(torch_cuda, sampler, kind, D, kv, page, extra):
    torch = torch_cuda
    T = 7
    c = Case(torch, kind, [0, 5, page - 1, page, 40, 11, 3], T, kv, kv, D, page, 81, extra=extra,
             spare=0)
    rng = np.random.default_rng(81)
    count = np.array([7, 0, 3, 99, -2, 5, 4], np.int32)
    take = np.stack([rng.permutation(T) for _ in range(7)]).astype(np.int32)
    take[5, 1:4] = [-1, T, 2 ** 31 - 1]       # no such nodes: skipped
    take[6, :4] = 2                           # one node at four positions
    c.table[3, 1] = c.n_pages                 # a page outside the cache: skipped
    for with_take, with_count in ((True, True), (False, True), (True, False), (False, False)):
        d = c.device()
        exp = {"k": c.k.clone(), "v": c.v.clone()}
        for b in range(7):
            n = min(max(int(count[b]), 0), T) if with_count else T
            for i in range(n):
                node = int(take[b, i]) if with_take else i
                p = int(c.lens[b]) + i
                if not 0 <= node < T or p >= c.per * page:
                    continue
                blk = int(c.table[b, p // page])
                if not 0 <= blk < c.n_pages:
                    continue
                at = blk * page + p % page
                exp["k"][at, :kv * D] = c.kn[b, node, :kv * D]
                exp["v"][at, :kv * D] = c.vn[b, node, :kv * D]
        sampler.cache_append(c.cache(d), d["kn"], d["vn"], c.kn.shape[2], 7, T,
                             torch.from_numpy(take).cuda() if with_take else None,
                             torch.from_numpy(count).cuda() if with_count else None)
        sampler.sync()
        for n in ("k", "v"):
            assert torch.equal(d[n].cpu().view(torch.int16), exp[n].view(torch.int16)), (
                n, with_take, with_count)


def test_append_stops_at_the_tables_end(torch_cuda, sampler):
    torch = torch_cuda
    c = Case(torch, "bf16", [14], 6, 1, 1, 64, 8, 91, spare=0)
    c.per = 2
    c.table = c.table[:, :2].contiguous()
    d = c.device()
    sampler.cache_append(c.cache(d), d["kn"], d["vn"], 64, 1, 6)
    sampler.sync()
    exp = c.k.clone()
    exp[c.slots(0, torch.tensor([14, 15]))] = c.kn[0, :2]
    assert torch.equal(d["k"].cpu().view(torch.int16), exp.view(torch.int16))


def test_attention_after_append_is_attention_over_the_nodes(torch_cuda, sampler):
    """A token attended as a node, then appended and attended as part of the
    cache: a second token's result against the reference both ways."""
    torch = torch_cuda
    c = Case(torch, "bf16", [37, 64], 2, 4, 2, 64, 16, 95)
    chain = c.run(sampler, "chain of two")
    d = c.device()
    sampler.cache_append(c.cache(d), d["kn"], d["vn"], 128, 2, 2,
                         d_count=torch.tensor([1, 1], dtype=torch.int32).cuda())
    one = Case(torch, "bf16", [37, 64], 1, 4, 2, 64, 16, 95)
    d["lens"] += 1
    kn, vn, q = (d[n][:, 1:].contiguous() for n in ("kn", "vn", "q"))
    out = torch.zeros_like(q)
    sampler.tree_attention(c.cache(d), kn, vn, 128, 2, 1, 4, c.scale, q, 256, out, 256)
    sampler.sync()
    exp, tol = c.want()
    got = out.double().cpu().numpy().reshape(2, 4, 64)
    assert (np.abs(got - exp[:, 1]) <= tol[:, 1]).all()
    assert one.T == 1 and chain.shape[1] == 2


def test_refused_calls(torch_cuda, sampler):
    c = Case(torch_cuda, "bf16", [5], 2, 4, 2, 64, 16, 1)
    d = c.device()
    before = d["out"].clone()
    good = dict(type=pz.PZ_BF16, n_kv_heads=2, head_dim=64, d_k=d["k"], d_v=d["v"], ld=128,
                n_blocks=c.n_pages, block_size=16, d_blocks=d["table"], max_blocks=c.per,
                d_len=d["lens"])
    for kw, code in ((dict(type=pz.PZ_F32), pz.PZ_ENOTSUP), (dict(head_dim=80), pz.PZ_ENOTSUP),
                     (dict(block_size=12), pz.PZ_EINVAL), (dict(ld=100), pz.PZ_EINVAL),
                     (dict(d_len=None), pz.PZ_EINVAL)):
        cache = pz.kv_cache(**dict(good, **kw))
        with pytest.raises(pz.PzError) as e:
            sampler.tree_attention(cache, d["kn"], d["vn"], 128, 1, 2, 4, 0.1, d["q"], 256,
                                   d["out"], 256)
        assert e.value.code == code, kw
        with pytest.raises(pz.PzError):
            sampler.cache_append(cache, d["kn"], d["vn"], 128, 1, 2)
    with pytest.raises(pz.PzError) as e:
        sampler.tree_attention(pz.kv_cache(**good), d["kn"], d["vn"], 128, 1, 65, 4, 0.1, d["q"],
                               256, d["out"], 256)
    assert e.value.code == pz.PZ_ERANGE
    sampler.sync()
    assert torch_cuda.equal(d["out"], before)


def test_captured_and_replayed(torch_cuda, sampler):
    """Append and attention in one graph, replayed with longer sequences and
    new nodes, eager calls between: every replay against an eager call."""
    torch = torch_cuda
    c = Case(torch, "bf16", [2000, 100, 7], 4, 8, 2, 128, 16, 99).random_tree(9)
    d = c.device()
    count = torch.tensor([2, 4, 1], dtype=torch.int32).cuda()
    c.call(sampler, d)  # (the workspace exists before the capture)
    sampler.sync()
    import ctypes
    lib, h = sampler.lib, sampler.h
    cache = c.cache(d)

    def calls(out):
        assert lib.pz_cache_append(h, ctypes.byref(cache), d["kn"].data_ptr(), d["vn"].data_ptr(),
                                   256, 3, 4, None, count.data_ptr()) == 0
        assert lib.pz_tree_attention(h, ctypes.byref(cache), d["kn"].data_ptr(),
                                     d["vn"].data_ptr(), 256, 3, 4, None, d["tree"].data_ptr(), 8,
                                     c.scale, d["q"].data_ptr(), 1024, out.data_ptr(), 1024) == 0

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(sampler.stream)):
        calls(d["out"])
    eager = torch.empty_like(d["out"])
    for i in range(4):
        d["kn"].normal_()
        d["vn"].normal_()
        d["q"].normal_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager.zero_()
        torch.cuda.synchronize()
        calls(eager)
        sampler.sync()
        assert torch.equal(eager, d["out"]), i
        assert torch.isfinite(eager.float()).all()
        d["lens"] += count
