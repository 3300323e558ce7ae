"""Attention over shared prefixes (pz_prefix_attention).

Reference and bound: those of test_gpu_tree.py, with the prefix's positions before
each sequence's own.  A weight is rounded against the largest score of its part of the
keys, so its half step is relative to the weight itself as there; the parts' sums meet
in fp32 (a few 2^-24 more, within the bound's 2^-20)."""
import numpy as np
import pytest

import pzsample as pz
from test_gpu_tree import KINDS, Case

pytestmark = pytest.mark.gpu


class Shared(Case):
    """Case whose sequences b with of[b] = i have prefix i (or none, -1); `first` the
    ranges as the call takes them (None: even)."""

    def __init__(self, torch, kind, prefix_lens, first, lens, *args, pspare=1, **kw):
        super().__init__(torch, kind, lens, *args, **kw)
        g = torch.Generator().manual_seed(kw.get("seed", 0) + 999)
        self.plens = np.asarray(prefix_lens, np.int32)
        P = self.P = len(prefix_lens)
        self.first = first
        cut = first if first is not None else [i * (self.B // P) for i in range(P + 1)]
        self.of = [-1] * self.B
        for i in range(P):
            for b in range(max(cut[i], 0), min(cut[i + 1], self.B)):
                self.of[b] = i
        self.pper = (max(max(prefix_lens), 1) + self.page - 1) // self.page + pspare
        # pages behind the sequences' own, in no order
        more = P * self.pper
        self.ptable = (self.n_pages + torch.randperm(more, generator=g)).reshape(P, self.pper)
        self.ptable = self.ptable.to(torch.int32)
        self.n_pages += more
        for name in ("k", "v"):
            old = getattr(self, name)
            new = torch.full((self.n_pages * self.page, old.shape[1]), float("nan"), dtype=self.dt)
            new[:old.shape[0]] = old
            setattr(self, name, new)
        row = self.kv * self.D
        for i in range(P):
            p = torch.arange(int(min(max(prefix_lens[i], 0), self.pper * self.page)))
            at = self.pslots(i, p)
            self.k[at, :row] = torch.randn((len(p), row), generator=g).to(self.dt)
            self.v[at, :row] = torch.randn((len(p), row), generator=g).to(self.dt)

    def pslots(self, i, p):
        return self.ptable[i].long()[p // self.page] * self.page + p % self.page

    def want(self):
        T, D, group = self.T, self.D, self.heads // self.kv
        _, h, _ = KINDS[self.kind]
        out = np.full((self.B, T, self.heads, D), np.nan)
        tol = np.zeros_like(out)

        def cached(table, n, per):
            pos = np.arange(min(max(int(n), 0), per * self.page))
            pages = table.numpy()[pos // self.page]
            ok = (pages >= 0) & (pages < self.n_pages)
            return np.where(ok, pages, 0).astype(np.int64) * self.page + pos % self.page, ok
        for b in range(self.B):
            nn = T if self.n_nodes is None else min(max(int(self.n_nodes[b]), 0), T)
            at, ok = cached(self.table[b], self.lens[b], self.per)
            if self.of[b] >= 0:
                i = self.of[b]
                pat, pok = cached(self.ptable[i], self.plens[i], self.pper)
                at, ok = np.concatenate([pat, at]), np.concatenate([pok, ok])
            for hk in range(self.kv):
                sl = slice(hk * D, hk * D + D)
                k = np.concatenate([self.k[at, sl].double().numpy(),
                                    self.kn[b, :, sl].double().numpy()])
                v = np.concatenate([self.v[at, sl].double().numpy(),
                                    self.vn[b, :, sl].double().numpy()])
                js = slice(hk * group, (hk + 1) * group)
                for t in range(nn):
                    bits = int(self.tree[b, t]) if self.tree is not None else (2 << t) - 1
                    see = np.concatenate([ok, [(bits >> u & 1) == 1 and u < nn for u in range(T)]])
                    if not see.any():
                        out[b, t, js] = 0.0
                        continue
                    ks, vs = k[see], v[see]
                    q = self.q[b, t, hk * group * D:(hk + 1) * group * D].double().numpy()
                    q = q.reshape(group, D)
                    s = q @ ks.T * self.scale
                    p = np.exp(s - s.max(1, keepdims=True))
                    p /= p.sum(1, keepdims=True)
                    o = p @ vs
                    n = len(ks)
                    err = ((D + 2) * 2.0 ** -24 * self.scale * (np.abs(q) @ np.abs(ks).T).max(1)
                           + 2 * np.abs(s).max(1) * 2.0 ** -24)
                    d = (2 * err + 2.0 ** -20 + n * 2.0 ** -23)[:, None]
                    out[b, t, js] = o
                    tol[b, t, js] = (h * np.abs(o) + (h + d) * (1 + h) * (p @ np.abs(vs))
                                     + (n * 2.0 ** -33 * np.abs(vs).max() + 2.0 ** -25
                                        if self.kind == "fp16" else 0.0))
        return out, tol

    def check_tokens(self, out, label=""):
        """check() for T = 1 without a tree, computed on the GPU, a key head of a prefix's
        sequences at a time."""
        t, D, group = self.torch, self.D, self.heads // self.kv
        _, h, _ = KINDS[self.kind]
        q = self.q[:, 0, :self.heads * D].cuda().double().reshape(self.B, self.kv, group, D)
        got = out[:, 0, :self.heads * D].double().reshape(self.B, self.kv, group, D)
        k, v = self.k.cuda(), self.v.cuda()
        kn, vn = (x[:, 0].cuda() for x in (self.kn, self.vn))

        def cached(table, n, per):
            n = min(max(int(n), 0), per * self.page)
            p = t.arange(n)
            page = table.long()[p // self.page]
            ok = (page >= 0) & (page < self.n_pages)
            return ((t.where(ok, page, 0) * self.page + p % self.page)[ok]).cuda()
        own = [cached(self.table[b], self.lens[b], self.per) for b in range(self.B)]
        most = max(len(a) for a in own) + 1
        at = t.zeros((self.B, most), dtype=t.long, device="cuda")
        on = t.zeros((self.B, most), dtype=t.bool, device="cuda")
        for b, a in enumerate(own):
            at[b, :len(a)], on[b, :len(a) + 1] = a, True
        for i in sorted(set(self.of)):
            bs = t.tensor([b for b in range(self.B) if self.of[b] == i]).cuda()
            pat = cached(self.ptable[i], self.plens[i], self.pper) if i >= 0 else at[0, :0]
            for hk in range(self.kv):
                sl = slice(hk * D, hk * D + D)
                Q = q[bs, hk]                                              # [n, group, D]
                kp, vp = k[pat, sl].double(), v[pat, sl].double()
                ko, vo = k[at[bs], sl].double(), v[at[bs], sl].double()    # [n, most, D]
                last = (on[bs].sum(1) - 1)
                rows = t.arange(len(bs), device="cuda")
                ko[rows, last], vo[rows, last] = kn[bs, sl].double(), vn[bs, sl].double()
                dead = ~on[bs]
                ko[dead], vo[dead] = 0.0, 0.0

                def over(f, a, b):  # of the prefix's keys, then of its own
                    x = f(Q).reshape(-1, D) @ f(a).t()
                    y = f(Q) @ f(b).transpose(1, 2).contiguous()
                    return t.cat([x.reshape(len(bs), group, -1), y], 2)

                def mix(p, a, b):
                    n = a.shape[0]
                    x = p[..., :n].reshape(len(bs) * group, n) @ a
                    return x.reshape(len(bs), group, D) + p[..., n:].contiguous() @ b
                s = over(lambda x: x, kp, ko) * self.scale
                live = t.cat([t.ones((len(bs), len(pat)), dtype=t.bool, device="cuda"), on[bs]], 1)
                s = t.where(live[:, None], s, -t.inf)
                p = t.softmax(s, 2)
                o = mix(p, vp, vo)
                n = s.shape[2]
                err = ((D + 2) * 2.0 ** -24 * self.scale * over(t.abs, kp, ko).amax(2)
                       + 2 * t.where(live[:, None], s.abs(), 0.0).amax(2) * 2.0 ** -24)
                d = (2 * err + 2.0 ** -20 + n * 2.0 ** -23)[..., None]
                tol = h * o.abs() + (h + d) * (1 + h) * mix(p, vp.abs(), vo.abs())
                # (bf16: a part's weights are 2^-40 times those against a score m of the row, so
                # that its largest is at least 2^-40; one below 2^-126, the least normal number,
                # may be lost, and with it at most 2^-126 / 2^-40 of that part's mean times its
                # value: for all n keys n 2^-86 max|v|)
                big = max(float(vp.abs().max()) if len(pat) else 0.0, float(vo.abs().max()))
                if self.kind == "fp16":
                    tol = tol + n * 2.0 ** -33 * big + 2.0 ** -25
                else:
                    tol = tol + n * 2.0 ** -86 * big
                off = (got[bs, hk] - o).abs() - tol
                assert (off <= 0).all(), (label, i, hk, off.max())

    def run_tokens(self, s, label=""):
        d = self.device()
        self.call(s, d)
        s.sync()
        self.check_tokens(d["out"], label)
        return d["out"]

    def device(self):
        d = super().device()
        t = self.torch
        d["ptable"] = self.ptable.cuda()
        d["plens"] = t.from_numpy(self.plens).cuda()
        d["first"] = None if self.first is None else t.tensor(self.first, dtype=t.int32).cuda()
        return d

    def prefix(self, d):
        return pz.kv_prefix(d_blocks=d["ptable"], max_blocks=self.pper, d_len=d["plens"],
                            n_prefixes=self.P, d_first=d["first"])

    def call(self, s, d):
        s.prefix_attention(self.cache(d), self.prefix(d), d["kn"], d["vn"], self.kn.shape[2],
                           self.B, self.T, self.heads, self.scale, d["q"], self.q.shape[2],
                           d["out"], self.q.shape[2], d["n_nodes"], d["tree"])


@pytest.fixture(scope="module")
def sampler(torch_cuda):
    with pz.Sampler(1, 16) as s:
        yield s


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 3, 17, 64])
def test_prefixes(torch_cuda, sampler, kind, D, T):
    for i, (heads, kv) in enumerate([(8, 2), (4, 4), (16, 1), (3, 1)]):
        Shared(torch_cuda, kind, [100, 0, 33], None, [0, 1, 31, 33, 100, 5], T, heads, kv, D, 16,
               seed=100 * T + i).random_tree(T + i).run(sampler, ("even", heads, kv))
        Shared(torch_cuda, kind, [65, 1, 40, 32], [0, 1, 1, 4, 5], [3, 0, 16, 50, 2, 7], T, heads,
               kv, D, 16, seed=100 * T + i + 50).random_tree(T).run(sampler, ("ranges", heads, kv))


@pytest.mark.parametrize("kind,D", [("bf16", 64), ("bf16", 128), ("fp16", 128), ("bf16", 256)])
@pytest.mark.parametrize("B,T,heads,kv", [(2, 1, 8, 2), (6, 1, 8, 2), (24, 1, 8, 2), (40, 1, 8, 1),
                                          (40, 2, 16, 2), (96, 1, 16, 2), (7, 5, 16, 1)])
def test_long_prefixes(torch_cuda, sampler, kind, D, B, T, heads, kv):
    """In splits, for few rows and many, chains."""
    for c in (Shared(torch_cuda, kind, [3001], None, [1 + 7 * b % 40 for b in range(B)], T, heads,
                     kv, D, 32, seed=B + T),
              # (the first sequence without one)
              Shared(torch_cuda, kind, [2049, 777], [1, 1 + B // 2, B],
                     [7 * b % 40 for b in range(B)], T, heads, kv, D, 16, seed=B + T + 7)):
        (c.run_tokens if T == 1 else c.run)(sampler, c.P)


@pytest.mark.parametrize("kind,D", [("bf16", 64), ("bf16", 128), ("fp16", 128), ("fp16", 64)])
@pytest.mark.parametrize("each", [35, 70, 300])
def test_many_rows_of_many_heads(torch_cuda, sampler, kind, D, each):
    """A workgroup for every CU: rows that share keys in LDS, of prefixes that end
    anywhere in a tile, in one, and before the first; with pages that are missing."""
    lens = [33, 1, 64, 0] if each == 300 else [200, 129, 1, 64]
    c = Shared(torch_cuda, kind, lens, None, [b % 3 for b in range(4 * each)], 1, 64, 64, D, 16,
               seed=each + D)
    c.run_tokens(sampler, "whole")
    c.ptable[0, 1] = -1
    c.ptable[2, 0] = c.n_pages
    c.run_tokens(sampler, "missing pages")


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("fp16", 64)])
def test_many_rows_of_a_long_prefix(torch_cuda, sampler, kind, D):
    """In splits, whose borders are anywhere in a tile of 64; tables of more entries than a
    workgroup keeps at hand."""
    torch = torch_cuda
    c = Shared(torch, kind, [8500 + 37], None, [5, 0] * 45, 1, 32, 16, D, 8, seed=D, pspare=0)
    c.run_tokens(sampler, "splits")
    c.plens[0] = 8192
    c.run_tokens(sampler, "whole tiles")
    c.ptable[0, 700:720] = -1
    c.ptable[0, 1023] = 2 ** 31 - 1
    c.run_tokens(sampler, "missing pages")


@pytest.mark.parametrize("pspare", [120, 250])  # (the table's length tells the kernel)
@pytest.mark.parametrize("kind,D", [("bf16", 128), ("fp16", 64)])
def test_one_infinite_value(torch_cuda, sampler, kind, D, pspare):
    """Every score alike, and two elements of one value infinite: of that column alone."""
    torch = torch_cuda
    c = Shared(torch, kind, [4200], None, [0] * 40, 1, 32, 16, D, 16, seed=D + 1, pspare=pspare)
    c.q.zero_()
    clean = c.run_tokens(sampler, "alike")
    at = c.pslots(0, torch.tensor([4199]))
    c.v[at, 3] = float("inf")
    c.v[at, 2 * D + 1] = float("-inf")
    d = c.device()
    c.call(sampler, d)
    sampler.sync()
    got, clean = (x.reshape(40, 32, D).float() for x in (d["out"], clean))
    for h, i, v in ((0, 3, 1.0), (1, 3, 1.0), (4, 1, -1.0), (5, 1, -1.0)):
        assert (got[:, h, i] == v * float("inf")).all()
        got[:, h, i] = clean[:, h, i]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("page", [8, 16, 64, 512])
def test_pages_and_strides(torch_cuda, sampler, page):
    Shared(torch_cuda, "bf16", [515, 9], None, [1, 7, 8, 9, 515, 0], 4, 6, 3, 64, page, seed=page,
           extra=24).random_tree(1).run(sampler, page)


def test_long_own_positions(torch_cuda, sampler):
    """Sequences whose own part is split, too, and longer than the prefix."""
    for T, heads, kv in ((1, 8, 2), (20, 8, 4), (64, 8, 2)):
        Shared(torch_cuda, "bf16", [50], None, [2500, 17], T, heads, kv, 128, 16,
               seed=T).random_tree(T).run(sampler, T)


def test_counts_and_lengths_outside_their_range(torch_cuda, sampler):
    c = Shared(torch_cuda, "bf16", [40, 40, 40], None, [40] * 6, 6, 4, 2, 64, 16,
               seed=11).random_tree(2)
    c.n_nodes = [0, -1, 1, 5, 6, 99]
    c.run(sampler, "counts")
    c.lens = np.array([-4, 0, 1, 40, 39, 17], np.int32)
    c.plens = np.array([-7, 0, 17], np.int32)
    c.run(sampler, "lengths")
    full = Shared(torch_cuda, "bf16", [64, 64], None, [48, 48], 2, 4, 2, 64, 16, seed=12, pspare=0)
    full.plens = np.array([2 ** 31 - 1, 64], np.int32)
    full.run(sampler, "as long as the table")


def test_ranges_outside_the_batch(torch_cuda, sampler):
    for first in ([-3, 2, 9], [2, 2, 2], [0, 0, 5], [4, 5, 5], [-9, -1, 0], [7, 8, 9]):
        Shared(torch_cuda, "bf16", [70, 33], first, [20, 0, 5, 9, 33], 2, 4, 2, 64, 16,
               seed=13).run(sampler, first)


def test_many_prefixes(torch_cuda, sampler):
    """More than a wave looks at together, most of them without a sequence."""
    P = 150
    first = sorted(int(x) for x in np.random.default_rng(1).integers(0, 9, P + 1))
    for T, heads in ((1, 2), (40, 8)):
        Shared(torch_cuda, "bf16", [1 + 5 * i % 60 for i in range(P)], first, [3] * 8, T, heads, 2,
               64, 16, seed=14).run(sampler, T)


def test_pages_outside_the_cache_hold_nothing(torch_cuda, sampler):
    for B, T in ((6, 3), (40, 4)):
        c = Shared(torch_cuda, "fp16", [700, 100], None, [100] * B, T, 16, 2, 128, 16,
                   seed=21).random_tree(3)
        c.ptable[0, 2] = -1
        c.ptable[0, 40] = 2 ** 31 - 1
        c.table[0, 2] = -1
        c.table[1, 0] = c.n_pages
        c.ptable[1, :] = -(2 ** 31)
        c.run(sampler, B)


def test_rows_that_see_nothing(torch_cuda, sampler):
    for T in (3, 40):
        c = Shared(torch_cuda, "bf16", [0, 30], None, [0, 0, 0, 50], T, 4, 2, 64, 16,
                   seed=31).random_tree(4)
        c.tree[0, :] = 0
        c.tree[1, 1:] = 0
        c.tree[2, ::2] = 0
        c.run(sampler, T)
        # a prefix of no page is nothing, too
        c.plens[0] = 20
        c.ptable[0, :] = -1
        c.run(sampler, (T, "no page"))


def test_scores_that_are_infinite(torch_cuda, sampler):
    """Rows whose every score is -infinity are NaN, wherever the keys are."""
    torch = torch_cuda
    for D in (64, 256):
        c = Shared(torch, "bf16", [10, 5], None, [3, 0, 4, 6], 1, 2, 1, D, 16, seed=5)
        c.q.zero_()
        c.q[:, :, ::D] = 1.0   # the first element of each head
        c.kn.zero_()
        c.kn[..., 0] = 1.0
        for i, n in enumerate(c.plens):
            c.k[c.pslots(i, torch.arange(int(n))), 0] = float("-inf")
        clean = c.want()[0]
        assert np.isfinite(clean[1]).all()  # (its own node is what it attends)
        d = c.device()
        c.call(sampler, d)
        sampler.sync()
        assert torch.isfinite(d["out"].float()).all()
        c.tree = np.zeros((4, 1), np.uint64)
        c.lens[:] = [0, 0, 4, 6]
        d = c.device()
        c.call(sampler, d)
        sampler.sync()
        got = d["out"].float()
        assert torch.isnan(got[:2]).all() and torch.isfinite(got[2:]).all()


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_what_is_not_seen_has_no_influence(torch_cuda, sampler, kind):
    """Another prefix's NaN, other sequences' and those behind lengths (every slot
    that holds nothing is NaN in these cases) change no bit."""
    torch = torch_cuda
    for B, T in ((4, 2), (32, 8)):
        c = Shared(torch, kind, [300, 90], None, [20 + b for b in range(B)], T, 8, 2, 128, 16,
                   seed=41).random_tree(5)
        clean = c.run(sampler, "clean").clone()
        c.k[c.pslots(1, torch.arange(90))] = float("nan")
        c.v[c.pslots(1, torch.arange(90))] = float("inf")
        d = c.device()
        c.call(sampler, d)
        sampler.sync()
        assert torch.equal(d["out"][:B // 2], clean[:B // 2])
        assert torch.isnan(d["out"][B // 2:].float()).any()


def test_ends_of_the_range(torch_cuda, sampler):
    """Values and scores at the types' ends: results stay finite where the mean is."""
    torch = torch_cuda
    for kind, most in (("bf16", 3.38953138925153547590e38), ("fp16", 65504.0)):
        for B in (2, 40):
            c = Shared(torch, kind, [200], None, [20] * B, 1, 8, 2, 64, 16, seed=51)
            c.v[torch.isfinite(c.v)] = most
            c.vn[:] = most
            d = c.device()
            c.call(sampler, d)
            sampler.sync()
            assert (d["out"].double() >= most * (1 - 2.0 ** -7)).all()
            assert torch.isfinite(d["out"].float()).all()
            # scores far from zero, apart by what the type holds of them
            c = Shared(torch, kind, [200], None, [20] * B, 1, 8, 2, 64, 16, seed=52, sigma=40.0)
            c.run(sampler, (kind, B, "far"))


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("fp16", 64)])
def test_scores_of_many_rows(torch_cuda, sampler, kind, D):
    """The kernel for many rows: scores far from zero and apart, infinite ones of some rows,
    rows that are NaN."""
    torch = torch_cuda
    c = Shared(torch, kind, [200, 129, 1, 64], None, [b % 3 for b in range(280)], 1, 64, 64, D, 16,
               seed=81, sigma=80.0 if kind == "bf16" else 60.0)
    c.run_tokens(sampler, "far")
    c = Shared(torch, kind, [200, 129, 1, 64], None, [b % 3 for b in range(280)], 1, 64, 64, D, 16,
               seed=82)
    at = c.pslots(0, torch.tensor([150]))
    c.k[at, :D] = 0.0

    def run(first, q=None):
        c.k[at, 0] = first
        d = c.device()
        if q is not None:
            d["q"][5] = q
        c.call(sampler, d)
        sampler.sync()
        return d["out"][:, 0].reshape(280, 64, D).float()
    clean, got = run(60000.0), run(float("inf"))
    up = (c.q[:70, 0, 0] > 0).cuda()
    assert up.any() and not up.all()
    assert torch.isnan(got[:70, 0][up]).all() and torch.isfinite(got[:70, 0][~up]).all()
    # (a score of -infinity is a weight of 0, as one far below the others is)
    far = (c.q[:70, 0, 0] < -0.5).cuda()
    assert torch.equal(got[:70, 0][far], clean[:70, 0][far])
    assert torch.equal(got[:70, 1:], clean[:70, 1:]) and torch.equal(got[70:], clean[70:])
    # (another row's scores may change which m its neighbours' weights are taken against, and
    # so their rounding: within the bound)
    got = run(60000.0, float("nan"))
    assert torch.isnan(got[5]).all()
    got[5] = clean[5]
    c.check_tokens(got.reshape(280, 1, -1), "beside a NaN")


def test_more_rows_than_the_workspace(torch_cuda, sampler):
    """64 MiB hold two parts of 32513 rows of 256: the sequences are taken in turns,
    whose borders lie inside prefixes."""
    torch = torch_cuda
    B, T, heads, D = 70, 64, 16, 256
    assert B * T * heads > 2 * 32513
    c = Shared(torch, "bf16", [40, 3, 20], [3, 30, 31, 68], [b % 20 for b in range(B)], T, heads,
               1, D, 16, seed=61)
    d = c.device()
    c.call(sampler, d)
    sampler.sync()
    # against the same sequences in small batches
    lib_first = c.first
    for b0 in (0, 29, 33, 66):
        small = Shared(torch, "bf16", [40, 3, 20], None, [0, 0, 0], T, heads, 1, D, 16, seed=61)
        for n in ("k", "v", "page", "pper", "ptable", "plens", "n_pages", "per"):
            setattr(small, n, getattr(c, n))
        small.first = [min(max(x - b0, 0), 3) for x in lib_first]
        small.of = c.of[b0:b0 + 3]
        small.lens = c.lens[b0:b0 + 3]
        small.table = c.table[b0:b0 + 3].contiguous()
        for n in ("q", "kn", "vn"):
            setattr(small, n, getattr(c, n)[b0:b0 + 3].contiguous())
        small.check(d["out"][b0:b0 + 3], b0)


def test_more_rows_than_the_workspace_in_even_parts(torch_cuda, sampler):
    """Alike without ranges: turns that begin and end inside a prefix, and hold many; and
    more prefixes than ranges may name."""
    T, heads, D = 64, 16, 256
    for P, B in ((3, 72), (36, 72)):
        c = Shared(torch_cuda, "bf16", [40, 3, 20] * (P // 3), None, [b % 20 for b in range(B)], T,
                   heads, 1, D, 16, seed=62)
        d = c.device()
        c.call(sampler, d)
        sampler.sync()
        each, step = B // P, 2 * 32513 // (2 * T * heads)
        for b0 in (0, step - 1, step, 2 * step - 1, B - 3):
            small = Shared(torch_cuda, "bf16", [40] * P, [0] * (P + 1), [0, 0, 0], T, heads, 1, D,
                           16, seed=62)
            for n in ("k", "v", "page", "pper", "ptable", "plens", "n_pages", "per"):
                setattr(small, n, getattr(c, n))
            small.first = [min(max(i * each - b0, 0), 3) for i in range(P + 1)]
            small.of = c.of[b0:b0 + 3]
            small.lens = c.lens[b0:b0 + 3]
            small.table = c.table[b0:b0 + 3].contiguous()
            for n in ("q", "kn", "vn"):
                setattr(small, n, getattr(c, n)[b0:b0 + 3].contiguous())
            small.check(d["out"][b0:b0 + 3], (P, b0))
    B = 6000
    c = Shared(torch_cuda, "bf16", [1 + b % 70 for b in range(B)], None, [b % 3 for b in range(B)],
               1, 2, 1, 64, 16, seed=63)
    c.run(sampler, B)


def test_as_tree_attention(torch_cuda, sampler):
    """The prefix's pages in each sequence's own table give the same results, within
    both bounds."""
    torch = torch_cuda
    c = Shared(torch, "bf16", [96], None, [0] * 4, 2, 8, 2, 64, 16, seed=71, spare=8)
    got = c.run(sampler)
    d = c.device()
    d["table"] = d["ptable"].repeat(4, 1).contiguous()
    d["lens"] = torch.full((4,), 96, dtype=torch.int32).cuda()
    cache = pz.kv_cache(type=pz.PZ_BF16, n_kv_heads=2, head_dim=64, d_k=d["k"], d_v=d["v"], ld=128,
                        n_blocks=c.n_pages, block_size=16, d_blocks=d["table"], max_blocks=c.pper,
                        d_len=d["lens"])
    out = torch.zeros_like(got)
    sampler.tree_attention(cache, d["kn"], d["vn"], 128, 4, 2, 8, c.scale, d["q"], 512, out, 512)
    sampler.sync()
    c.check(out, "tree attention")


def test_replayed(torch_cuda, sampler):
    """Captured with an append, replayed on longer sequences and prefixes, eager calls
    between: every replay against an eager call."""
    torch = torch_cuda
    c = Shared(torch, "bf16", [500, 60], None, [100, 7, 0, 30], 2, 8, 2, 128, 16, seed=99,
               spare=4).random_tree(9)
    for name in ("k", "v"):  # (positions that lengths reach later)
        t = getattr(c, name)
        t[torch.isnan(t)] = 0.5
    d = c.device()
    c.call(sampler, d)
    sampler.sync()
    lib, h = sampler.lib, sampler.h
    cache, prefix = c.cache(d), c.prefix(d)

    def calls(out):
        assert lib.pz_cache_append(h, pz.ctypes.byref(cache), d["kn"].data_ptr(),
                                   d["vn"].data_ptr(), 256, 4, 2, None, None) == 0
        assert lib.pz_prefix_attention(h, pz.ctypes.byref(cache), pz.ctypes.byref(prefix),
                                       d["kn"].data_ptr(), d["vn"].data_ptr(), 256, 4, 2, None,
                                       d["tree"].data_ptr(), 8, c.scale, d["q"].data_ptr(), 1024,
                                       out.data_ptr(), 1024) == 0
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(sampler.stream)):
        calls(d["out"])
    eager = torch.empty_like(d["out"])
    for i in range(4):
        for n in ("kn", "vn", "q"):
            d[n].normal_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager.zero_()
        torch.cuda.synchronize()
        calls(eager)
        sampler.sync()
        assert torch.equal(eager, d["out"]), i
        assert torch.isfinite(eager.float()).all()
        d["lens"] += 2
        d["plens"] += 3


def test_refusals(torch_cuda, sampler):
    c = Shared(torch_cuda, "bf16", [20, 20], None, [3, 3, 3, 3], 1, 4, 2, 64, 16, seed=1)
    d = c.device()
    c.P = 3
    with pytest.raises(pz.PzError) as e:
        c.call(sampler, d)
    assert e.value.code == pz.PZ_EINVAL and "divides" in str(e.value)
    c.P, c.T = 2, 65
    with pytest.raises(pz.PzError) as e:
        c.call(sampler, d)
    assert e.value.code == pz.PZ_ERANGE
    c.T, c.B = 1, 0
    c.call(sampler, d)
    sampler.sync()
    assert (d["out"] == 77).all()
