"""Selections of a beam search (pz_beam_select) and the reordering of the beams'
caches (pz_beam_reorder).

Selection, reference in 64 bits: parents, ids and flags are equal; a score is the
reference's rounded to fp32, whose 64-bit value is off by at most 2^-40 (1 + |score|):
the exponentials by 2^-42, their sum's logarithm and the sums by a few 2^-53 of the
values.  Inputs are random, so that no two candidates of different logits lie that close
(a draw that did would fail here without a fault; none does).  Reordering is exact."""
import numpy as np
import pytest

import pzsample as pz
from conftest import to_dev

pytestmark = pytest.mark.gpu


def select(x, score, done, pad, K, eos=()):
    """(parent, ids, scores, done) of [G, W, V] logits."""
    G, W, V = x.shape
    parent, ids = np.full((G, K), -1, np.int32), np.full((G, K), -1, np.int32)
    out, ended = np.full((G, K), -np.inf), np.zeros((G, K), np.uint8)
    for g in range(G):
        cands = []
        for w in range(W):
            s = np.float64(score[g, w])
            if not np.isfinite(s):
                continue
            if done is not None and done[g, w]:
                cands.append((-s, w, 0.0, pad, 1))
                continue
            row = x[g, w].astype(np.float64)
            if not (row < np.inf).all() or not np.isfinite(row).any():
                continue
            m = row.max()
            lse = m + np.log(np.exp(row - m).sum())
            top = np.lexsort((np.arange(V), -row))[:K]
            cands += [(-(s + (row[i] - lse)), w, -row[i], int(i), 0) for i in top
                      if np.isfinite(row[i])]
        cands.sort()
        for k, (s, w, _, i, e) in enumerate(cands[:K]):
            parent[g, k], ids[g, k], out[g, k] = w, i, -s
            ended[g, k] = e or i in eos
    return parent, ids, out, ended


class Selection:
    def __init__(self, torch, G, W, V, seed, pad=0, off=0, sigma=3.0):
        rng = np.random.default_rng(seed)
        self.torch, self.G, self.W, self.V, self.off = torch, G, W, V, off
        self.ld = V + pad
        self.x = (rng.standard_normal((G, W, V)) * sigma).astype(np.float32)
        self.score = (-20 * rng.random((G, 1)) - 3 * rng.random((G, W))).astype(np.float32)
        self.done = None
        self.pad_id = 0

    def device(self):
        t = self.torch
        flat = t.full((self.G * self.W * self.ld + self.off,), float("nan"), device="cuda")
        x = flat[self.off:].reshape(self.G * self.W, self.ld)
        x[:, :self.V] = to_dev(t, self.x.reshape(-1, self.V))
        return x, to_dev(t, self.score), None if self.done is None else to_dev(t, self.done)

    def run(self, s, K, eos=(), label="", want_done=True):
        t, G = self.torch, self.G
        s.set_eos(list(eos))
        x, score, done = self.device()
        out = [t.full((G, K), 55, dtype=d, device="cuda")
               for d in (t.int32, t.int32, t.float32, t.uint8)]
        s.beam_select(x, self.ld, G, self.W, self.V, score, K, *out[:3], d_done=done,
                      pad_id=self.pad_id, d_done_out=out[3] if want_done else None)
        s.sync()
        self.check(out if want_done else out[:3], K, eos, label)
        return out

    def check(self, out, K, eos=(), label=""):
        want = select(self.x, self.score, self.done, self.pad_id, K, eos)
        got = [o.cpu().numpy() for o in out]
        for n, a, b in zip(("parent", "ids"), got, want):
            assert (a == b).all(), (label, n, np.argwhere(a != b)[:4], a[a != b][:4], b[a != b][:4])
        if len(got) > 3:
            assert (got[3] == want[3]).all(), (label, "done")
        there = want[0] >= 0
        assert (got[2][~there] == -np.inf).all(), (label, "pads")
        w = want[2][there]
        off = np.abs(got[2][there].astype(np.float64) - w)
        assert (off <= 2.0 ** -24 * np.abs(w) * (1 + 2.0 ** -20) + 2.0 ** -39 * (1 + np.abs(w))).all(), (
            label, "scores", off.max())


@pytest.fixture(scope="module")
def sampler(torch_cuda):
    with pz.Sampler(1, 16) as s:
        yield s


@pytest.mark.parametrize("V", [1, 2, 3, 5, 63, 257, 1000, 2048, 2049, 8192, 8193, 50257])
@pytest.mark.parametrize("W", [1, 2, 5, 16])
def test_sizes(torch_cuda, sampler, V, W):
    for K in sorted({1, W, 2 * W, 33}):
        Selection(torch_cuda, 3, W, V, V + W).run(sampler, K, eos=[0, 7], label=K)


@pytest.mark.parametrize("G,W,V,K", [(1, 4, 128256, 4), (8, 8, 128256, 16), (16, 4, 151936, 8),
                                     (40, 16, 8191, 32), (1, 64, 20000, 128), (2, 64, 130000, 64),
                                     (130, 4, 20001, 4), (1, 1, 1 << 22, 128)])
def test_large(torch_cuda, sampler, G, W, V, K):
    Selection(torch_cuda, G, W, V, G + K).run(sampler, K)


def test_strides_and_addresses(torch_cuda, sampler):
    for pad, off in ((0, 1), (3, 0), (61, 2), (1, 3)):
        Selection(torch_cuda, 2, 3, 9001, pad, pad=pad, off=off).run(sampler, 6, label=(pad, off))


def test_first_step_and_ended_beams(torch_cuda, sampler):
    c = Selection(torch_cuda, 4, 4, 3001, 1)
    c.score[:, 1:] = -np.inf
    c.score[:, 0] = 0.0
    c.run(sampler, 8, label="first")
    c = Selection(torch_cuda, 6, 5, 3001, 2)
    c.done = (np.random.default_rng(3).random((6, 5)) < 0.4).astype(np.uint8)
    c.done[1], c.done[2] = 0, 255
    for pad in (0, 2999, -1, 2 ** 31 - 1):
        c.pad_id = pad
        c.run(sampler, 10, eos=[pad, 5], label=pad)
    c.run(sampler, 10, want_done=False)
    # an ended beam's row is not looked at
    c.x[c.done != 0] = np.nan
    c.run(sampler, 10)


def test_fewer_candidates_than_asked_for(torch_cuda, sampler):
    c = Selection(torch_cuda, 5, 3, 700, 4)
    c.x[0] = -np.inf
    c.x[1, :, 2:] = -np.inf
    c.x[2, 1, 5], c.x[2, 0, 699] = np.nan, np.inf
    c.score[3] = [np.nan, np.inf, -np.inf]
    c.x[4, :2] = np.nan
    c.x[4, 2, 1:] = -np.inf
    c.run(sampler, 20)
    c.done = np.ones((5, 3), np.uint8)
    c.run(sampler, 20, label="ended")  # (scores that are not finite offer nothing all the same)


def test_masks_and_outliers(torch_cuda, sampler):
    low = np.finfo(np.float32).min
    rng = np.random.default_rng(5)
    for V in (3000, 60000):
        for value in (-np.inf, low, -1e9):
            c = Selection(torch_cuda, 3, 4, V, V)
            c.x[rng.random(c.x.shape) < 0.999] = value
            c.run(sampler, 8, label=(V, value))
        c = Selection(torch_cuda, 3, 4, V, V + 1)
        c.x[:, :, 17] = 1e30
        c.run(sampler, 8, label="one far above")
        c = Selection(torch_cuda, 3, 4, V, V + 2, sigma=1e-3)
        c.x += 1000.0
        c.run(sampler, 8, label="far from zero")
        c = Selection(torch_cuda, 3, 4, V, V + 3, sigma=1e-30)
        c.run(sampler, 8, label="almost equal")


@pytest.mark.parametrize("G,W,V", [(1, 4, 20000), (2, 48, 60000)])
def test_not_a_number_among_masked_ids(torch_cuda, sampler, G, W, V):
    """A NaN rules its row out, also where its part of the row has no other logit."""
    c = Selection(torch_cuda, G, W, V, 5)
    c.x[:, 1, 100:] = -np.inf
    c.run(sampler, 4, label="masked")
    c.x[:, 1, V - 7] = np.nan
    c.run(sampler, 4, label="and a NaN")
    c.x[:, 0, 20:] = -np.inf
    c.x[:, 0, 11000] = np.inf
    c.run(sampler, 2 * W, label="and an infinity")


@pytest.mark.parametrize("V", [5, 2500, 40000])
def test_ties(torch_cuda, sampler, V):
    """Equal logits, equal beams: lower beams, then lower ids."""
    for K in (1, 4, 9, 128):
        c = Selection(torch_cuda, 3, 4, V, 6)
        c.x[0] = 0.25
        c.x[1] = np.round(c.x[1])
        c.x[2, 1:], c.score[2, 1:] = c.x[2, 0], c.score[2, 0]
        c.score[0, 1] = c.score[0, 0]
        c.run(sampler, K, label=(V, K))
        c.x[:] = -0.0
        c.x[:, :, ::3] = 0.0
        c.score[:] = -1.5
        c.run(sampler, K, label="zeros")


def test_many_groups(torch_cuda, sampler):
    """More than the workspace holds at a time."""
    c = Selection(torch_cuda, 1100, 64, 40, 7)
    assert 1100 * 64 * (16 + 128 * 8) > pz.PZ_BEAM_WORKSPACE
    c.done = (np.random.default_rng(8).random((1100, 64)) < 0.1).astype(np.uint8)
    c.run(sampler, 128)


def test_more_logits_than_32_bits_count(torch_cuda, sampler):
    """Rows past 2^31 elements, with NaN between them."""
    torch = torch_cuda
    ld, V = (1 << 29) + 4, 5000
    c = Selection(torch, 3, 2, V, 9)
    flat = torch.empty((5 * ld + V,), device="cuda")
    for r in range(6):
        flat[r * ld:r * ld + V] = to_dev(torch, c.x.reshape(6, V)[r])
        if r < 5:
            flat[r * ld + V:r * ld + V + 64] = float("nan")
    out = [torch.zeros((3, 4), dtype=d, device="cuda") for d in (torch.int32, torch.int32,
                                                                 torch.float32)]
    sampler.beam_select(flat, ld, 3, 2, V, to_dev(torch, c.score), 4, *out)
    sampler.sync()
    c.check(out, 4)


def test_selection_replayed(torch_cuda, sampler):
    torch = torch_cuda
    c = Selection(torch, 4, 4, 20000, 10)
    x, score, _ = c.device()
    done = torch.zeros((4, 4), dtype=torch.uint8, device="cuda")
    outs = [[torch.zeros((4, 8), dtype=d, device="cuda")
             for d in (torch.int32, torch.int32, torch.float32, torch.uint8)] for _ in range(2)]
    sampler.set_eos([11])

    def call(o):
        assert sampler.lib.pz_beam_select(sampler.h, x.data_ptr(), c.ld, 4, 4, c.V,
                                          score.data_ptr(), done.data_ptr(), 3, 8,
                                          *(t.data_ptr() for t in o)) == 0
    call(outs[0])
    sampler.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(sampler.stream)):
        call(outs[0])
    c.pad_id = 3
    for i in range(4):
        x.normal_()
        done.copy_(torch.rand((4, 4), device="cuda") < 0.2 * i)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        call(outs[1])
        sampler.sync()
        assert all(torch.equal(a, b) for a, b in zip(*outs)), i
        c.x, c.done = x[:, :c.V].cpu().numpy().reshape(4, 4, -1), done.cpu().numpy()
        c.check(outs[0], 8, [11], i)


# ---- reordering ----------------------------------------------------------------
def reorder(table, lens, parent, pool, ahead, page):
    """(table, lens, missing, copies (from, to, positions)) of [G, W, per] tables."""
    G, W, per = table.shape
    new, length = np.full_like(table, -1), np.zeros_like(lens)
    missing, copies = np.zeros(G, np.int32), []
    for g in range(G):
        eldest, used, asks = {}, set(), []
        for w in range(W):
            p = int(parent[g, w])
            if not 0 <= p < W:
                continue
            n = min(max(int(lens[g, p]), 0), per * page)
            length[g, w] = n
            keep = n // page
            if p not in eldest and n % page:
                keep += 1
            eldest.setdefault(p, w)
            new[g, w, :keep] = table[g, p, :keep]
            used.update(table[g, p, :keep].tolist())
            asks += [(w, c) for c in range(keep, min(per, -(-(n + ahead) // page)))]
        free = [int(p) for p in pool[g] if int(p) not in used]
        for i, (w, c) in enumerate(asks):
            if i >= len(free):
                missing[g] += 1
                continue
            new[g, w, c] = free[i]
            p = int(parent[g, w])
            n = int(length[g, w])
            if n % page and c == n // page:
                copies.append((int(table[g, p, c]), free[i], n % page))
    return new, length, missing, copies


class Reordering:
    """Groups whose beams share pages at random, over caches of several layers."""

    def __init__(self, torch, G, W, per, page, kv, D, layers, seed, ahead=1, pool=None, extra=0,
                 kind="bf16", shared=0):
        rng = np.random.default_rng(seed)
        self.torch, self.G, self.W, self.per, self.page = torch, G, W, per, page
        self.kv, self.D, self.ahead, self.kind = kv, D, ahead, kind
        n_pool = W * per if pool is None else pool
        self.n_pages = G * n_pool + shared + 2
        ids = rng.permutation(self.n_pages)[:G * n_pool + shared].astype(np.int32)
        self.pool = np.sort(ids[:G * n_pool].reshape(G, n_pool), 1)
        self.common = ids[G * n_pool:]  # pages of no pool
        self.lens = np.repeat(rng.integers(0, per * page - ahead + 1, (G, 1)), W, 1).astype(np.int32)
        self.table = np.full((G, W, per), -1, np.int32)
        for g in range(G):
            spare = list(rng.permutation(self.pool[g]))
            for w in range(W):
                full = self.lens[g, w] // page
                top = -(-self.lens[g, w] // page)
                old = rng.integers(0, w) if w else 0
                share = rng.integers(0, full + 1) if w else 0
                for c in range(top):
                    if c < min(shared, full):
                        self.table[g, w, c] = self.common[c]
                    elif c < share:
                        self.table[g, w, c] = self.table[g, old, c]
                    else:
                        self.table[g, w, c] = spare.pop() if spare else -1
        self.parent = rng.integers(0, W, (G, W)).astype(np.int32)
        self.dt = torch.bfloat16 if kind == "bf16" else torch.float16
        gen = torch.Generator().manual_seed(seed)
        shape = (layers, 2, self.n_pages * page, kv * D + extra)
        self.kvs = torch.randn(shape, generator=gen).to(self.dt)

    def caches(self, d):
        return [pz.kv_cache(type=pz.PZ_BF16 if self.kind == "bf16" else pz.PZ_F16,
                            n_kv_heads=self.kv, head_dim=self.D, d_k=d["kvs"][i, 0],
                            d_v=d["kvs"][i, 1], ld=self.kvs.shape[3], n_blocks=self.n_pages,
                            block_size=self.page, d_blocks=d["table"], max_blocks=self.per,
                            d_len=d["lens"]) for i in range(self.kvs.shape[0])]

    def device(self):
        t = self.torch
        d = {n: to_dev(t, getattr(self, n)) for n in ("table", "lens", "parent", "pool")}
        d["kvs"] = self.kvs.cuda()
        d["out"] = t.full_like(d["table"], 99)
        d["len_out"] = t.full_like(d["lens"], 99)
        d["missing"] = t.full((self.G,), 99, dtype=t.int32, device="cuda")
        return d

    def run(self, s, label="", missing=True):
        d = self.device()
        s.beam_reorder(self.caches(d), self.G, self.W, d["parent"], d["pool"], self.pool.shape[1],
                       self.ahead, d["out"], d["len_out"], d["missing"] if missing else None)
        s.sync()
        table, lens, lacks, copies = reorder(self.table, self.lens, self.parent, self.pool,
                                             self.ahead, self.page)
        assert (d["len_out"].cpu().numpy() == lens).all(), (label, "lengths")
        got = d["out"].cpu().numpy()
        assert (got == table).all(), (label, "tables", np.argwhere(got != table)[:5])
        if missing:
            assert (d["missing"].cpu().numpy() == lacks).all(), (label, "missing")
        want = self.kvs.clone()
        for a, b, n in copies:
            if 0 <= a < self.n_pages and 0 <= b < self.n_pages:
                w = self.kv * self.D
                want[:, :, b * self.page:b * self.page + n, :w] = \
                    self.kvs[:, :, a * self.page:a * self.page + n, :w]
        assert self.torch.equal(d["kvs"].cpu().view(self.torch.int16),
                                want.view(self.torch.int16)), (label, "contents")
        return d


@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("W", [1, 2, 3, 8, 64])
def test_reorderings(torch_cuda, sampler, page, W):
    for i, (G, per, ahead) in enumerate([(1, 1, 0), (3, 4, 1), (2, 9, 5), (5, 3, 2 * page)]):
        if ahead > per * page:
            continue
        Reordering(torch_cuda, G, W, per, page, 2, 64, 2, 10 * page + W + i, ahead=ahead).run(
            sampler, (G, per, ahead))


@pytest.mark.parametrize("D,kv,extra,kind", [(64, 1, 0, "bf16"), (128, 3, 24, "fp16"),
                                             (256, 2, 8, "bf16")])
def test_shapes_and_strides(torch_cuda, sampler, D, kv, extra, kind):
    Reordering(torch_cuda, 3, 4, 5, 16, kv, D, 3, D, extra=extra, kind=kind).run(sampler)


def test_more_layers_than_a_launch_takes(torch_cuda, sampler):
    Reordering(torch_cuda, 2, 3, 3, 8, 1, 64, 131, 1).run(sampler)


def test_parents_without_a_beam_and_odd_lengths(torch_cuda, sampler):
    c = Reordering(torch_cuda, 5, 4, 4, 16, 2, 64, 2, 2)
    c.parent[0] = [-1, 4, 2 ** 31 - 1, -(2 ** 31)]
    c.parent[1] = [2, -1, 2, 2]
    c.lens[2] = [-5, 0, 2 ** 31 - 1, 64]
    c.lens[3] = [1, 16, 17, 63]
    c.run(sampler, "parents")
    c.ahead = 2 ** 31 - 1
    c.run(sampler, "as far as the tables go", missing=False)
    c.ahead = 0
    c.run(sampler, "nothing ahead")


def test_pools_that_lack_pages(torch_cuda, sampler):
    for pool in (0, 1, 3, 7, 31, 32, 33):
        c = Reordering(torch_cuda, 3, 4, 6, 8, 1, 64, 2, 3 + pool, pool=pool)
        c.parent[0] = 1
        c.run(sampler, pool)


def test_pages_outside_the_pool_or_the_cache(torch_cuda, sampler):
    c = Reordering(torch_cuda, 3, 4, 8, 8, 1, 64, 2, 4, shared=3)
    c.run(sampler, "a prompt's pages")
    c.table[0, :, 0] = -1
    c.table[1, 2] = 2 ** 31 - 1
    c.table[2, 1, -1] = c.n_pages
    c.lens[:] = 61
    c.parent[:] = [[2, 2, 2, 1]] * 3
    c.run(sampler, "no pages")


def test_large_pools(torch_cuda, sampler):
    """Pools of more words than the workgroup has threads; long tables; and the last sizes
    that one launch takes."""
    for W, per, pool in ((64, 64, 8192), (64, 65, 8192), (2, 3, 8193)):
        Reordering(torch_cuda, 2, W, per, 8, 1, 64, 2, W + per, pool=pool).run(sampler, pool)
    c = Reordering(torch_cuda, 2, 16, 1200, 8, 1, 64, 1, 5)
    c.run(sampler)
    c = Reordering(torch_cuda, 1, 2, 3, 8, 1, 64, 1, 6, pool=50000)
    c.run(sampler)


def test_long_searches_keep_their_histories(torch_cuda, sampler):
    """60 steps of appends and reorderings, tables in turns: every beam's cache holds what
    its hypothesis appended, whatever was shared, copied, given up and given out again."""
    torch = torch_cuda
    G, W, per, page, D = 3, 5, 9, 8, 64
    rng = np.random.default_rng(7)
    c = Reordering(torch, G, W, per, page, 1, D, 2, 7)
    c.lens[:] = 0
    c.table[:] = -1
    d = c.device()
    d["table"].fill_(-1)
    # an empty cache's first pages
    ident = to_dev(torch, np.tile(np.arange(W, dtype=np.int32), (G, 1)))
    names = [("table", "lens"), ("out", "len_out")]
    history = [[[] for _ in range(W)] for _ in range(G)]

    def step(parent):
        (a, al), (b, bl) = names
        at = dict(d, table=d[a], lens=d[al])
        sampler.beam_reorder(c.caches(at), G, W, parent, d["pool"], c.pool.shape[1], 1, d[b],
                             d[bl], d["missing"])
        sampler.sync()
        assert (d["missing"] == 0).all()
        names.reverse()
    step(ident)
    for t in range(60):
        a, al = names[0]
        kn = torch.randn((G * W, 1, D)).to(torch.bfloat16)
        now = c.caches(dict(d, table=d[a], lens=d[al]))
        for i, cache in enumerate(now):
            sampler.cache_append(cache, (kn + i).cuda(), (kn - i).cuda(), D, G * W, 1)
            sampler.sync()
        for g in range(G):
            for w in range(W):
                history[g][w] = history[g][w] + [kn[g * W + w, 0]]
        d[al] += 1
        torch.cuda.synchronize()
        parent = rng.integers(0, W, (G, W)).astype(np.int32)
        if t % 7 == 0:
            parent[:] = np.arange(W)
        step(to_dev(torch, parent))
        history = [[history[g][parent[g, w]] for w in range(W)] for g in range(G)]
        if t % 9 == 8 or t == 59:
            a, al = names[0]
            table, lens = d[a].cpu().reshape(G, W, per).long(), d[al].cpu()
            for i in range(2):
                k, v = d["kvs"][i, 0].cpu(), d["kvs"][i, 1].cpu()
                for g in range(G):
                    for w in range(W):
                        n = int(lens[g, w])
                        assert n == t + 1
                        p = torch.arange(n)
                        at = table[g, w, p // page] * page + p % page
                        want = torch.stack(history[g][w])
                        assert torch.equal(k[at], want + i) and torch.equal(v[at], want - i)


def test_reordering_replayed(torch_cuda, sampler):
    torch = torch_cuda
    c = Reordering(torch, 3, 4, 5, 16, 2, 64, 3, 8)
    d = c.device()
    caches = c.caches(d)
    arr = (pz.KvCache * 3)(*caches)

    def call():
        assert sampler.lib.pz_beam_reorder(sampler.h, arr, 3, 3, 4, d["parent"].data_ptr(),
                                           d["pool"].data_ptr(), c.pool.shape[1], 1,
                                           d["out"].data_ptr(), d["len_out"].data_ptr(),
                                           d["missing"].data_ptr()) == 0
    call()
    sampler.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(sampler.stream)):
        call()
    for i in range(4):
        d["parent"].random_(0, 4)
        d["kvs"].normal_()
        torch.cuda.synchronize()
        was = d["kvs"].clone()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = [d[n].clone() for n in ("out", "len_out", "missing", "kvs")]
        d["kvs"].copy_(was)
        torch.cuda.synchronize()
        call()
        sampler.sync()
        assert all(torch.equal(a, d[n]) for a, n in zip(got, ("out", "len_out", "missing", "kvs"))), i
        want = reorder(c.table, c.lens, d["parent"].cpu().numpy(), c.pool, 1, 16)
        assert (got[0].cpu().numpy() == want[0]).all()


def test_refusals(torch_cuda, sampler):
    c = Reordering(torch_cuda, 2, 2, 2, 8, 1, 64, 2, 9)
    d = c.device()
    caches = c.caches(d)

    def call(layers=caches, G=2, W=2, n_pool=4, out="out", ahead=1):
        sampler.beam_reorder(layers, G, W, d["parent"], d["pool"], n_pool, ahead, d[out],
                             d["len_out"])
    for code, kw in ((pz.PZ_EINVAL, dict(W=0)), (pz.PZ_ERANGE, dict(W=65)),
                     (pz.PZ_ERANGE, dict(n_pool=pz.PZ_BEAM_MAX_POOL + 1)),
                     (pz.PZ_EINVAL, dict(ahead=-1)), (pz.PZ_EINVAL, dict(out="table"))):
        with pytest.raises(pz.PzError) as e:
            call(**kw)
        assert e.value.code == code, kw
    other = c.caches(dict(d, table=d["out"]))
    with pytest.raises(pz.PzError) as e:
        call(layers=[caches[0], other[1]])
    assert e.value.code == pz.PZ_EINVAL and "layers" in str(e.value)
    call(G=0)
    sampler.sync()
    assert (d["out"] == 99).all()
    x = Selection(torch_cuda, 1, 2, 10, 1)
    for K, code in ((0, pz.PZ_EINVAL), (129, pz.PZ_ERANGE)):
        with pytest.raises(pz.PzError) as e:
            x.run(sampler, K)
        assert e.value.code == code
