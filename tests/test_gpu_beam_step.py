"""A beam search over shared prompts as a program runs it: queries' and keys' norms and
rotation, attention over the prompts and the beams' own pages, the new positions' way into
them, the LM head, the selection of the next beams and the reordering of their caches.

Every stage is checked on what the stage before left on the device, each within the bound
of its own tests; which keys and values a beam has is known from the choices alone (a
history a beam, permuted with the parents), so that a wrong page or a lost position shows
in the next step's attention."""
import numpy as np
import pytest

import pzsample as pz
import test_gpu_beam as be
import test_gpu_rope as ro

pytestmark = pytest.mark.gpu

G, W, LAYERS, HEADS, KV, D, PAGE, V = 3, 4, 2, 4, 2, 64, 8, 1003
N, ROW, KROW, B = HEADS * D, (HEADS + 2 * KV) * D, KV * D, G * W
PROMPTS, MOST, STEPS, EOS = [37, 16, 0], 4, 26, list(range(7, V, 60))
POOL = W * MOST
H = 2.0 ** -8  # half a step of bf16


class Search:
    """The state of a search on the device, and a step of it."""

    def __init__(self, torch, s, seed):
        self.torch, self.s = torch, s
        g = torch.Generator().manual_seed(seed)

        def rand(*shape):
            return torch.randn(shape, generator=g)
        self.emb = rand(V, N).cuda()
        self.w_qkv = [(rand(ROW, N) / N ** 0.5).to(torch.bfloat16).cuda() for _ in range(LAYERS)]
        self.w_o = [(rand(N, N) / N ** 0.5).to(torch.bfloat16).cuda() for _ in range(LAYERS)]
        self.head = (3 * rand(V, N) / N ** 0.5).to(torch.bfloat16).cuda()
        self.norms = [(1 + 0.1 * rand(2, D)).cuda() for _ in range(LAYERS)]
        self.freq = torch.tensor(10000.0 ** (-np.arange(D // 2) / (D / 2)),
                                 dtype=torch.float32).cuda()
        per = max(-(-n // PAGE) for n in PROMPTS)
        n_blocks = G * (per + POOL)
        pages = torch.randperm(n_blocks, generator=g).to(torch.int32)
        self.prompt = pages[:G * per].reshape(G, per)
        pool = pages[G * per:].reshape(G, POOL).sort(1).values.contiguous()
        self.k, self.v = ([torch.full((n_blocks * PAGE, KROW), float("nan"),
                                      dtype=torch.bfloat16) for _ in range(LAYERS)]
                          for _ in range(2))
        for i, n in enumerate(PROMPTS):
            p = torch.arange(n)
            at = self.prompt[i].long()[p // PAGE] * PAGE + p % PAGE
            for t in self.k + self.v:
                t[at] = rand(n, KROW).to(torch.bfloat16)
        self.prompts = [[(k[at].double().numpy(), v[at].double().numpy())
                         for k, v in zip(self.k, self.v)]
                        for at in [self.prompt[i].long()[torch.arange(n) // PAGE] * PAGE
                                   + torch.arange(n) % PAGE for i, n in enumerate(PROMPTS)]]
        self.k, self.v = [t.cuda() for t in self.k], [t.cuda() for t in self.v]
        i32 = dict(dtype=torch.int32, device="cuda")
        # each group starts from one hypothesis with a page of its own
        table = torch.full((B, MOST), -1, dtype=torch.int32)
        table[::W, 0] = pool[:, 0]
        self.tables = [table.cuda(), torch.full((B, MOST), -2, **i32)]
        self.lens = [torch.zeros(B, **i32), torch.full((B,), -2, **i32)]
        score = torch.full((G, W), -np.inf)
        score[:, 0] = 0.0
        self.score, self.done = score.cuda(), torch.zeros(B, dtype=torch.uint8, device="cuda")
        self.ids = torch.tensor([11, 12, 13], **i32).repeat_interleave(W).contiguous()
        self.plens = torch.tensor(PROMPTS, **i32)
        self.base = self.plens.repeat_interleave(W).contiguous()
        self.prefix = pz.kv_prefix(d_blocks=self.prompt.cuda(), max_blocks=per, d_len=self.plens,
                                   n_prefixes=G)
        self.pool = pool.cuda()
        self.caches = [[pz.kv_cache(type=pz.PZ_BF16, n_kv_heads=KV, head_dim=D, d_k=k, d_v=v,
                                    ld=KROW, n_blocks=n_blocks, block_size=PAGE,
                                    d_blocks=self.tables[a], max_blocks=MOST, d_len=self.lens[a])
                        for k, v in zip(self.k, self.v)] for a in range(2)]
        self.ropes = [pz.qk_rope(type=pz.PZ_BF16, n_heads=HEADS, n_kv_heads=KV, head_dim=D,
                                 d_q_norm=w[0], d_k_norm=w[1], eps=1e-6, rot_dim=D,
                                 layout=pz.PZ_ROPE_HALVES, d_freq=self.freq, amplitude=1.0)
                      for w in self.norms]
        f32 = dict(dtype=torch.float32, device="cuda")
        self.x, self.y = torch.empty((B, N), **f32), torch.empty((B, N), **f32)
        self.qkv32 = torch.empty((B, ROW), **f32)
        self.raw, self.qkv = ([torch.empty((B, ROW), dtype=torch.bfloat16, device="cuda")
                               for _ in range(LAYERS)] for _ in range(2))
        self.att = [torch.empty((B, N), dtype=torch.bfloat16, device="cuda")
                    for _ in range(LAYERS)]
        self.o32 = torch.empty((B, N), **f32)
        self.logits = torch.empty((B, V), **f32)
        self.parent, self.nid = torch.empty((G, W), **i32), torch.empty((G, W), **i32)
        self.nscore = torch.empty((G, W), **f32)
        self.ndone = torch.empty(B, dtype=torch.uint8, device="cuda")
        self.missing = torch.empty(G, **i32)
        self.pos = torch.empty(B, **i32)

    def step(self, a):
        """One step on the sampler's stream, from tables a to 1 - a."""
        torch, s, lib = self.torch, self.s, self.s.lib
        ref, ptr = pz.ctypes.byref, lambda t: t.data_ptr()
        with torch.cuda.stream(torch.cuda.ExternalStream(s.stream)):
            torch.add(self.base, self.lens[a], out=self.pos)
            self.x.copy_(self.emb[self.ids.clamp(min=0).long()])
            for i in range(LAYERS):
                w = self.raw[i]
                assert lib.pz_lm_head_bf16(s.h, ptr(self.w_qkv[i]), ROW, N, ptr(self.x), B, N,
                                           ptr(self.qkv32), ROW) == 0
                w.copy_(self.qkv32)
                o = self.qkv[i]
                o.copy_(w)
                q, k, v = ptr(o), ptr(o) + 2 * N, ptr(o) + 2 * (N + KROW)
                assert lib.pz_qk_norm_rope(s.h, ref(self.ropes[i]), q, ROW, k, ROW, q, ROW, k,
                                           ROW, B, ptr(self.pos)) == 0
                c = self.caches[a][i]
                assert lib.pz_prefix_attention(s.h, ref(c), ref(self.prefix), k, v, ROW, B, 1,
                                               None, None, HEADS, D ** -0.5, q, ROW,
                                               ptr(self.att[i]), N) == 0
                assert lib.pz_cache_append(s.h, ref(c), k, v, ROW, B, 1, None, None) == 0
                self.y.copy_(self.att[i])
                assert lib.pz_lm_head_bf16(s.h, ptr(self.w_o[i]), N, N, ptr(self.y), B, N,
                                           ptr(self.o32), N) == 0
                self.x.add_(self.o32)
            self.x.mul_(0.3)
            assert lib.pz_lm_head_bf16(s.h, ptr(self.head), V, N, ptr(self.x), B, N,
                                       ptr(self.logits), V) == 0
            assert lib.pz_beam_select(s.h, ptr(self.logits), V, G, W, V, ptr(self.score),
                                      ptr(self.done), 0, W, ptr(self.parent), ptr(self.nid),
                                      ptr(self.nscore), ptr(self.ndone)) == 0
            self.lens[a].add_(1)  # (the position that was appended)
            arr = (pz.KvCache * LAYERS)(*self.caches[a])
            assert lib.pz_beam_reorder(s.h, arr, LAYERS, G, W, ptr(self.parent), ptr(self.pool),
                                       POOL, 1, ptr(self.tables[1 - a]), ptr(self.lens[1 - a]),
                                       ptr(self.missing)) == 0
            self.ids.copy_(self.nid.reshape(-1))

    def carry(self):
        """The chosen beams' scores and flags are the next step's."""
        with self.torch.cuda.stream(self.torch.cuda.ExternalStream(self.s.stream)):
            self.score.copy_(self.nscore)
            self.done.copy_(self.ndone)


def attend(q, keys, values):
    """(result, bound) of HEADS rows q over one beam's keys: test_gpu_prefix.py's."""
    out, tol = np.zeros((HEADS, D)), np.zeros((HEADS, D))
    n, scale = len(keys), D ** -0.5
    for h in range(HEADS):
        hk = h // (HEADS // KV)
        k, v = keys[:, hk * D:hk * D + D], values[:, hk * D:hk * D + D]
        s = k @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        err = ((D + 2) * 2.0 ** -24 * scale * (np.abs(k) @ np.abs(q[h])).max()
               + 2 * np.abs(s).max() * 2.0 ** -24)
        d = 2 * err + 2.0 ** -20 + n * 2.0 ** -23
        out[h] = p @ v
        tol[h] = H * np.abs(out[h]) + (H + d) * (1 + H) * (p @ np.abs(v))
    return out, tol


def test_search(torch_cuda):
    torch = torch_cuda
    with pz.Sampler(B, V) as s:
        s.set_eos(EOS)
        c = Search(torch, s, 3)
        hist = [[[(np.empty((0, KROW)), np.empty((0, KROW))) for _ in range(LAYERS)]
                 for _ in range(W)] for _ in range(G)]
        ended = 0
        torch.cuda.synchronize()
        for step in range(STEPS):
            a = step & 1
            score, done = c.score.cpu().numpy(), c.done.cpu().numpy()
            lens = c.lens[a].cpu().numpy()
            assert (lens == [len(hist[b // W][b % W][0][0]) for b in range(B)]).all(), step
            c.step(a)
            s.sync()
            assert (c.missing == 0).all(), step
            live = np.isfinite(score.reshape(-1))
            for i in range(LAYERS):
                raw, qkv = (t[i].cpu().double().numpy() for t in (c.raw, c.qkv))
                w = c.norms[i].cpu().numpy()
                for x, y, heads, at, wi in ((raw, qkv, HEADS, 0, 0), (raw, qkv, KV, N, 1)):
                    sl = slice(at, at + heads * D)
                    want, tol = ro.reference(x[:, sl], heads, D, D, pz.PZ_ROPE_HALVES,
                                             c.freq.cpu().numpy(), c.pos.cpu().numpy(), w[wi],
                                             1e-6, 1.0)
                    assert (np.abs(y[:, sl] - want) <= H * np.abs(want) + tol * (1 + H)).all(), (
                        step, i, "rotation")
                assert (raw[:, N + KROW:] == qkv[:, N + KROW:]).all()
                got = c.att[i].cpu().double().numpy().reshape(B, HEADS, D)
                for b in range(B):
                    own = hist[b // W][b % W][i]
                    new = qkv[b:b + 1, N:N + KROW], qkv[b:b + 1, N + KROW:]
                    k, v = (np.concatenate([p, o, n]) for p, o, n in
                            zip(c.prompts[b // W][i], own, new))
                    if live[b]:
                        want, tol = attend(qkv[b, :N].reshape(HEADS, D), k, v)
                        assert (np.abs(got[b] - want) <= tol).all(), (step, i, b, "attention")
                    hist[b // W][b % W][i] = tuple(np.concatenate([o, n])
                                                   for o, n in zip(own, new))
            want = be.select(c.logits.cpu().numpy().reshape(G, W, V), score, done.reshape(G, W), 0,
                             W, EOS)
            parent, ids, nscore, nd = (t.cpu().numpy().reshape(G, W)
                                       for t in (c.parent, c.nid, c.nscore, c.ndone))
            assert (parent == want[0]).all() and (ids == want[1]).all(), step
            assert (nd == want[3]).all(), step
            assert np.allclose(nscore, want[2], rtol=2.0 ** -23, atol=2.0 ** -39)
            ended += int(nd.sum())
            hist = [[[tuple(x.copy() for x in layer) for layer in hist[g][parent[g, w]]]
                     for w in range(W)] for g in range(G)]
            # what the pages hold is each beam's history, and what goes on has a page
            table, nl = c.tables[1 - a].cpu().numpy(), c.lens[1 - a].cpu().numpy()
            for b in range(B):
                n = len(hist[b // W][b % W][0][0])
                assert nl[b] == n and (table[b, :min(n // PAGE + 1, MOST)] >= 0).all()
                at = torch.from_numpy(table[b].astype(np.int64)[np.arange(n) // PAGE] * PAGE
                                      + np.arange(n) % PAGE).cuda()
                for i in range(LAYERS):
                    for t, x in zip((c.k[i], c.v[i]), hist[b // W][b % W][i]):
                        assert (t[at].cpu().double().numpy() == x).all(), (step, b, i, "pages")
            c.carry()
            s.sync()
        assert 0 < ended


def test_search_replayed(torch_cuda):
    """Two steps captured into a graph (the tables change places), replayed to the end of
    the search: the eager search's beams, bit for bit."""
    torch = torch_cuda

    def run(captured):
        with pz.Sampler(B, V) as s:
            s.set_eos(EOS)
            c = Search(torch, s, 3)
            torch.cuda.synchronize()
            said = []

            def pair():
                for a in (0, 1):
                    c.step(a)
                    c.carry()
            for i in range(STEPS // 2):
                if captured and i == 1:
                    torch.cuda.synchronize()
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(s.stream)):
                        pair()
                if captured and i >= 1:
                    g.replay()
                else:
                    pair()
                torch.cuda.synchronize()
                said.append([t.cpu().clone() for t in (c.parent, c.nid, c.nscore, c.ndone,
                                                       c.logits, c.tables[0], c.lens[0])])
                assert int(torch.zeros(64, device="cuda").sum()) == 0  # (eager work between)
            return said

    eager, replayed = run(False), run(True)
    for i, (x, y) in enumerate(zip(eager, replayed)):
        for j, (p, q) in enumerate(zip(x, y)):
            assert ro.same_bits(torch, p, q), (i, j)


def test_two_searches_at_once(torch_cuda):
    """Two samplers, their steps under way together: each search as alone."""
    torch = torch_cuda

    def run(seeds):
        samplers = [pz.Sampler(B, V) for _ in seeds]
        for s in samplers:
            s.set_eos(EOS)
        searches = [Search(torch, s, seed) for s, seed in zip(samplers, seeds)]
        torch.cuda.synchronize()
        for step in range(STEPS):
            for c in searches:
                c.step(step & 1)
                c.carry()
        torch.cuda.synchronize()
        said = [[t.cpu().clone() for t in (c.parent, c.nid, c.nscore, c.ndone, c.logits, c.lens[0],
                                           c.tables[0])] for c in searches]
        for s in samplers:
            s.close()
        return said

    both, alone = run([3, 4]), run([3]) + run([4])
    for i, (x, y) in enumerate(zip(both, alone)):
        for j, (p, q) in enumerate(zip(x, y)):
            assert ro.same_bits(torch, p, q), (i, j)
