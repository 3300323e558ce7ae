"""The operators together, as a decode loop uses them: drafted trees attend a
paged cache, the 8-bit LM head scores every node, grammar masks and penalties
change the scores, the sampler picks, the accepted path goes into the cache.

Every stage is checked on what the stage before left on the device: attention
within the bound of its own tests, the rest bit for bit."""
import numpy as np
import pytest

import pz_oracle as po
import pzsample as pz
import test_gpu_lmhead_i8 as i8
import test_gpu_rules as ru
from conftest import to_dev
from test_gpu_tree import Case

pytestmark = pytest.mark.gpu

HEADS, KV, D, PAGE, V = 4, 2, 64, 16, 3001
N = HEADS * D


def bits(tree):
    """Ancestor masks of parent lists."""
    sees = np.zeros(tree.shape, np.uint64)
    for b, row in enumerate(tree):
        for t, p in enumerate(row):
            sees[b, t] = np.uint64(1 << t) | (sees[b, p] if p >= 0 else np.uint64(0))
    return sees


@pytest.mark.parametrize("mode", [dict(temperature=0.0), dict(temperature=0.8, top_p=0.9)])
def test_constrained_tree_decode(torch_cuda, mode):
    torch = torch_cuda
    B, T, steps, H = 3, 5, 6, 16
    rng = np.random.default_rng(4)
    g = torch.Generator().manual_seed(4)
    # a toy model: token embeddings and projections, an int8 LM head
    emb = torch.randn((V, N), generator=g)
    proj = {n: torch.randn((N, w), generator=g) / N ** 0.5
            for n, w in (("q", N), ("kn", KV * D), ("vn", KV * D))}
    w8, sw = i8.quant(rng.standard_normal((V, N)).astype(np.float32))
    grammar = rng.random((4, V)) < 0.3          # four automaton states
    c = Case(torch, "bf16", [20, 0, 33], T, HEADS, KV, D, PAGE, 5, spare=3)
    d = c.device()
    cache = c.cache(d)
    host_k, host_v = c.k.clone(), c.v.clone()
    d_w, d_sw = to_dev(torch, w8), to_dev(torch, sw)
    d_mask = to_dev(torch, ru.pack(grammar).view(np.int32))
    last = rng.integers(0, V, B)
    hist = np.full((B, H), -1, np.int32)
    rows = B * T
    lens = c.lens.copy()
    accepted_total = 0
    with pz.Sampler(rows, V, max_hist=H) as s:
        xq = torch.empty((rows, N), dtype=torch.int8, device="cuda")
        sx = torch.empty(rows, device="cuda")
        y = torch.empty((rows, V), device="cuda")
        allowed = torch.empty(rows, dtype=torch.int32, device="cuda")
        guess = rng.integers(0, V, (B, T))
        for step in range(steps):
            # node 0 the input token, then a tree of guesses
            parent = np.array([[-1] + [int(rng.integers(0, t)) for t in range(1, T)]
                               for _ in range(B)])
            tokens = guess.copy()
            tokens[:, 0] = last
            e = emb[torch.from_numpy(tokens)]
            c.q, c.kn, c.vn = ((e @ proj[n]).to(torch.bfloat16) for n in ("q", "kn", "vn"))
            c.tree, c.lens = bits(parent), lens
            for n in ("q", "kn", "vn"):
                d[n].copy_(getattr(c, n))
            d["tree"] = torch.from_numpy(c.tree.view(np.int64)).cuda()
            d["out"].fill_(77.0)
            c.call(s, d)
            # the LM head on every node
            s.sync()
            x = d["out"].reshape(rows, N).float()
            s.quant_rows_i8(x, pz.PZ_F32, N, rows, N, xq, N, sx)
            s.lm_head_i8(d_w, d_sw, V, N, xq, sx, rows, N, y, V)
            raw = None
            s.sync()
            raw = y.cpu().numpy().copy()
            # each node's grammar state and history (its sequence's)
            state = rng.integers(-1, 4, rows).astype(np.int32)
            node_hist = np.repeat(hist, T, 0)
            rules = pz.logit_rules(1.1, 0.2, 0.1, d_hist=to_dev(torch, node_hist), H=H,
                                   d_mask=d_mask, ld_mask=d_mask.shape[1], n_masks=4,
                                   d_mask_row=to_dev(torch, state), d_allowed=allowed)
            s.rules(y, y, rows, V, V, V, rules)
            u = pz.synth_draws(rows, 100 + step)
            ids, _ = s.sample(y, rows, V, V, [pz.row_params(**mode)], u=u)

            c.check(d["out"], step)
            q, sc = i8.quant(x.cpu().numpy())
            i8.same(raw, i8.product(w8, sw, q, sc), step)
            exp, n_on = ru.want(raw, V, [(1.1, 0.2, 0.1)] * rows, node_hist, None, None, None,
                                grammar, state)
            ru.same(y.cpu().numpy(), exp, step)
            assert (allowed.cpu().numpy() == n_on).all()
            pick, _, _, _ = po.sample_batch(exp, [po.params(**mode)], u=u)
            assert (ids == pick).all(), step

            # walk each tree as far as a child holds its parent's token; make the
            # next step's guesses good ones so that paths are accepted
            take = np.full((B, T), -1, np.int32)
            count = np.zeros(B, np.int32)
            ids = ids.reshape(B, T)
            for b in range(B):
                at, path = 0, [0]
                while True:
                    kids = [t for t in range(T) if parent[b, t] == at and
                            (tokens[b, t] == ids[b, at] or (step % 2 and t == at + 1))]
                    if not kids:
                        break
                    at = kids[0]
                    path.append(at)
                take[b, :len(path)], count[b] = path, len(path)
                last[b] = ids[b, at]
                hist[b] = np.concatenate([hist[b][1:], [last[b]]])
                for i, t in enumerate(path):
                    slot = c.slots(b, torch.tensor([int(lens[b]) + i]))
                    host_k[slot, :KV * D] = c.kn[b, t]
                    host_v[slot, :KV * D] = c.vn[b, t]
            accepted_total += int(count.sum())
            s.cache_append(cache, d["kn"], d["vn"], KV * D, B, T, to_dev(torch, take),
                           to_dev(torch, count))
            s.sync()
            lens = lens + count
            d["lens"].copy_(torch.from_numpy(lens))
            c.k, c.v = host_k, host_v
            for n, want in (("k", host_k), ("v", host_v)):
                assert torch.equal(d[n].cpu().view(torch.int16), want.view(torch.int16)), (step, n)
            guess = rng.integers(0, V, (B, T))
    assert accepted_total > B * steps  # (some drafts were accepted)
