"""Operators of a beam search that decodes over a paged cache, as cases that can be
timed.

A case's "op":
  rope     queries and keys of the new tokens, as the projection leaves them in one
           row a token: the RMS norm of each head and the rotation to the token's
           position (pz_qk_norm_rope)
  prefix   attention of the new tokens over a prefix that sequences share (a prompt
           and its beams, a system prompt and a batch), over each sequence's own
           positions and over the new tokens (pz_prefix_attention)
  select   the best continuations of every group of beams, over its beams and the
           vocabulary (pz_beam_select)
  reorder  the chosen beams' caches: tables of pages that beams share, and copies of
           the pages that two beams would write (pz_beam_reorder)

Sizes are those of the bench's workloads (vocabularies 49152, 128256, 151936) and of
the attention cases beside them (32 heads over 8 of 128, 20 over 5).  With `own` false
run() computes a case by elementary torch operations; with it true, by the library's
calls.
"""
import ctypes
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

_MOST_ROPE = 16384 * 40 * 128          # elements of the largest rope case
_MOST_PRODUCTS = 256 * 32 * 128 * 32768  # query elements times prefix positions
_MOST_OWN = 256 * 512 * 8 * 128        # elements of the largest own cache
_MOST_LOGITS = 256 * 151936            # logits of the largest selection
_MOST_COPY = 8 * 8 * 8 * 16 * 8 * 128  # elements that the largest reordering could copy
_EOS = 2


def listed():
    return [
        # one token of one sequence
        dict(name="rope_1", op="rope", n=1, heads=32, kv=8, dim=128, rot=128, layout="halves",
             norm=True, type="bf16", far=4096),
        # a batch's target forward over drafts: 64 sequences of 5 tokens, half of each head
        # rotated, in neighbouring pairs, positions of a scaled long context
        dict(name="rope_320_partial", op="rope", n=320, heads=20, kv=5, dim=128, rot=64,
             layout="pairs", norm=True, type="fp16", far=1 << 20),
        # a chunk of prompts
        dict(name="rope_16384", op="rope", n=16384, heads=32, kv=8, dim=128, rot=128,
             layout="halves", norm=True, type="bf16", far=32768),
        # one prompt and its four beams: latency
        dict(name="prefix_1x4_ctx500", op="prefix", P=1, B=4, T=1, heads=32, kv=8, dim=128,
             page=16, ctx=500, tail=20, even=True, ragged=False, type="bf16"),
        # eight prompts of eight beams each, every prompt of its own length
        dict(name="prefix_8x8_ctx4096", op="prefix", P=8, B=64, T=1, heads=32, kv=8, dim=128,
             page=16, ctx=4096, tail=128, even=True, ragged=True, type="bf16"),
        # groups of uneven sizes that verify drafts
        dict(name="prefix_5x48x5_ctx2000", op="prefix", P=5, B=48, T=5, heads=20, kv=5, dim=128,
             page=32, ctx=2000, tail=300, even=False, ragged=True, type="fp16"),
        # a batch under one long system prompt
        dict(name="prefix_1x256_ctx32768", op="prefix", P=1, B=256, T=1, heads=32, kv=8, dim=128,
             page=64, ctx=32768, tail=512, even=True, ragged=True, type="bf16"),
        # the beams of one sequence
        dict(name="select_1x4x49152", op="select", G=1, W=4, V=49152, ld=49152, K=4, done=0.0,
             first=False),
        # twice the beams, so that ended hypotheses leave enough that go on
        dict(name="select_8x8x128256", op="select", G=8, W=8, V=128256, ld=128256, K=16,
             done=0.1, first=False),
        # the largest batch
        dict(name="select_64x4x151936", op="select", G=64, W=4, V=151936, ld=151936, K=4,
             done=0.1, first=False),
        # one sequence's beams, every layer's cache
        dict(name="reorder_1x4", op="reorder", G=1, W=4, layers=16, kv=8, dim=128, page=16,
             ctx=120, ahead=1, type="bf16"),
        # a batch of beam searches
        dict(name="reorder_8x8", op="reorder", G=8, W=8, layers=8, kv=8, dim=128, page=16,
             ctx=250, ahead=1, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "prefix", "prefix", "prefix", "select", "select", "reorder"])
    heads, kv = rng.choice([(32, 8), (20, 5), (32, 32), (16, 2), (8, 8), (24, 8)])
    dim, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 256])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rope":
        dim = rng.choice([64, 128, 128, 256, 80, 96])
        n = min(_log(rng, 1, 16384), _MOST_ROPE // ((heads + kv) * dim))
        kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if kind == "fp32":
            n = max(1, n // 2)
        rot = rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])
        return dict(op=op, n=n, heads=heads, kv=kv, dim=dim, rot=rot // 2 * 2,
                    layout=rng.choice(["halves", "pairs"]), norm=rng.random() < 0.7, type=kind,
                    far=_log(rng, 64, 1 << 20))
    if op == "prefix":
        ctx, T = _log(rng, 1, 32768), rng.choice([1, 1, _log(rng, 1, 8), _log(rng, 1, 64)])
        tail = rng.choice([1, _log(rng, 1, 512)])
        B = max(1, min(_log(rng, 1, 256), _MOST_PRODUCTS // (T * heads * dim * (ctx + tail + T)),
                       _MOST_OWN // ((tail + T) * kv * dim)))
        P = min(B, rng.choice([1, 1, _log(rng, 1, 32)]), max(1, (1 << 27) // (ctx * kv * dim)))
        return dict(op=op, P=P, B=B, T=T, heads=heads, kv=kv, dim=dim, page=page, ctx=ctx,
                    tail=tail, even=B % P == 0 and rng.random() < 0.5,
                    ragged=rng.random() < 0.6, type=kind)
    if op == "select":
        V, W = _log(rng, 1000, 200000), rng.choice([1, 2, 3, 4, 5, 8, 16])
        G = max(1, min(_log(rng, 1, 64), _MOST_LOGITS // (V * W)))
        return dict(op=op, G=G, W=W, V=V, ld=V if rng.random() < 0.5 else (V + 63) // 64 * 64,
                    K=rng.choice([W, 2 * W, W + 1]), done=rng.choice([0.0, 0.1, 0.5]),
                    first=rng.random() < 0.2)
    dim, W = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 5, 8, 16])
    G = max(1, min(_log(rng, 1, 64), 64 // W))
    layers = max(1, min(_log(rng, 1, 32), _MOST_COPY // (G * W * page * kv * dim)))
    return dict(op=op, G=G, W=W, layers=layers, kv=kv, dim=dim, page=page,
                ctx=_log(rng, 1, min(512, max(1, (1 << 28) // (G * W * layers * kv * dim)))),
                ahead=rng.choice([1, 1, 5]), type=kind)


def _normal(g, shape, sigma):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(sigma)


def _ints(g, lo, hi, shape):
    """Whole numbers from lo to hi."""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda").int()


def _type(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["type"]]


def _prepare_rope(case, g):
    n, heads, kv, dim, rot = (case[k] for k in ("n", "heads", "kv", "dim", "rot"))
    # queries, keys and values of a token side by side, as the fused projection
    # leaves them
    st = {"qkv": _normal(g, (n, (heads + 2 * kv) * dim), 1.5).to(_type(case))}
    # a run of positions for each of a few sequences
    run = max(1, min(n, 64))
    start = _ints(g, 0, max(0, case["far"] - run), ((n + run - 1) // run, 1))
    st["pos"] = (start + torch.arange(run, device="cuda")).reshape(-1)[:n].int().contiguous()
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    st["freq"] = torch.pow(500000.0, -2.0 * i / rot).float()
    if case["norm"]:
        st["q_norm"] = 1 + _normal(g, (dim,), 0.1)
        st["k_norm"] = 1 + _normal(g, (dim,), 0.1)
    st["q_out"] = torch.empty((n, heads, dim), dtype=_type(case), device="cuda")
    st["k_out"] = torch.empty((n, kv, dim), dtype=_type(case), device="cuda")
    return st


def _prepare_prefix(case, g):
    P, B, T, ctx, tail = (case[k] for k in ("P", "B", "T", "ctx", "tail"))
    heads, kv, dim, page, t = *(case[k] for k in ("heads", "kv", "dim", "page")), _type(case)
    per, own_per = (ctx + page - 1) // page, (tail + page - 1) // page
    n_pages = P * per + B * own_per
    pages = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    st = {"shared": pages[:P * per].reshape(P, per).contiguous(),
          "table": pages[P * per:].reshape(B, own_per).contiguous()}
    st["k"] = torch.empty((n_pages * page, kv, dim), dtype=t, device="cuda")
    st["v"] = torch.empty_like(st["k"])
    st["k"].normal_(generator=g)
    st["v"].normal_(generator=g)
    st["q"] = _normal(g, (B, T, heads, dim), 1.5).to(t)
    st["kn"] = _normal(g, (B, T, kv, dim), 1.0).to(t)
    st["vn"] = _normal(g, (B, T, kv, dim), 1.0).to(t)
    if case["ragged"]:
        st["shared_len"] = _ints(g, (ctx + 1) // 2, ctx, (P,))
        st["len"] = _ints(g, 0, tail, (B,))
    else:
        st["shared_len"] = torch.full((P,), ctx, dtype=torch.int32, device="cuda")
        st["len"] = torch.full((B,), tail, dtype=torch.int32, device="cuda")
    if case["even"]:
        cut = torch.arange(P + 1, device="cuda") * (B // P)
    else:  # each prefix has a sequence at least, the rest fall where they fall
        inner = 1 + torch.randperm(B - 1, generator=g, device="cuda")[:P - 1].sort().values
        cut = torch.cat([torch.zeros(1, device="cuda").long(), inner,
                         torch.full((1,), B, device="cuda")])
    st["first"], st["cut"] = cut.int().contiguous(), cut.tolist()
    # node 0 is the input token, every later node the child of an earlier one
    at = torch.rand((B, T), generator=g, device="cuda")
    rows = torch.arange(B, device="cuda")
    sees = torch.zeros((B, T), dtype=torch.int64, device="cuda")
    for i in range(T):
        sees[:, i] = 1 << i if i < 63 else -(1 << 63)  # (the sign bit is node 63's)
        if i:
            sees[:, i] |= sees[rows, (at[:, i] * i).long().clamp_(max=i - 1)]
    st["sees"] = sees
    st["out"] = torch.zeros((B, T, heads, dim), dtype=t, device="cuda")
    return st


def _prepare_select(case, g):
    G, W, K = case["G"], case["W"], case["K"]
    st = {"x": _normal(g, (G * W, case["ld"]), 3.0)}
    if case["first"]:  # a prompt's first step: one beam, the others not there yet
        score = torch.full((G, W), -math.inf, device="cuda")
        score[:, 0] = 0.0
    else:  # beams of a group lie close together
        score = (_normal(g, (G, 1), 1.0).abs() * -30 + _normal(g, (G, W), 2.0)).clamp_(max=0.0)
    st["score"] = score.reshape(-1).contiguous()
    st["done"] = (torch.rand(G * W, generator=g, device="cuda") < case["done"]).to(torch.uint8)
    for name, t in (("parent", torch.int32), ("ids", torch.int32), ("score_out", torch.float32),
                    ("done_out", torch.uint8)):
        st[name] = torch.zeros((G, K), dtype=t, device="cuda")
    return st


def _prepare_reorder(case, g):
    G, W, page, ctx, layers = (case[k] for k in ("G", "W", "page", "ctx", "layers"))
    per = (ctx + case["ahead"] + page - 1) // page
    n_pool = W * per
    n_pages = G * n_pool + 3
    # each group's own pages, in ascending order; its beams' tables as selections have
    # left them: an older beam's first pages, then pages of its own
    pool = torch.randperm(n_pages, generator=g, device="cuda")[:G * n_pool].reshape(G, n_pool)
    mixed = pool.reshape(G, W, per)
    length = _ints(g, 1, ctx, (G, 1)).long()
    full = length // page
    col = torch.arange(per, device="cuda")
    table = torch.empty((G, W, per), dtype=torch.int64, device="cuda")
    for w in range(W):
        old = _ints(g, 0, max(0, w - 1), (G,)).long()
        share = (torch.rand((G, 1), generator=g, device="cuda") * (full + 1)).long()
        from_old = (col < share) & (col < full) if w else torch.zeros_like(col < share)
        table[:, w] = torch.where(from_old, table[torch.arange(G, device="cuda"), old],
                                  mixed[:, w])
    table = torch.where(col < (length + page - 1)[..., None] // page, table, -1)
    st = {"table": table.reshape(G * W, per).int().contiguous(),
          "pool": pool.sort(1).values.int().contiguous(),
          "len": length.expand(G, W).reshape(-1).int().contiguous()}
    st["k"] = torch.empty((layers, n_pages * page, case["kv"] * case["dim"]), dtype=_type(case),
                          device="cuda")
    st["v"] = torch.empty_like(st["k"])
    st["k"].normal_(generator=g)
    st["v"].normal_(generator=g)
    st["parent"] = _ints(g, 0, W - 1, (G * W,))
    st["table_out"] = torch.empty_like(st["table"])
    st["len_out"] = torch.empty_like(st["len"])
    st["missing"] = torch.empty(G, dtype=torch.int32, device="cuda")
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2654435761 % (1 << 62) + 1)
    st = {"rope": _prepare_rope, "prefix": _prepare_prefix, "select": _prepare_select,
          "reorder": _prepare_reorder}[case["op"]](case, g)
    st["case"] = case
    return st


# ---- the plain forms ---------------------------------------------------------
_EPS = 1e-6


def _plain_rope(st):
    c = st["case"]
    n, heads, kv, dim, rot = (c[k] for k in ("n", "heads", "kv", "dim", "rot"))
    x = st["qkv"][:, :(heads + kv) * dim].float().reshape(n, heads + kv, dim)
    if c["norm"]:
        w = torch.cat([st["q_norm"].expand(heads, dim), st["k_norm"].expand(kv, dim)])
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
    # (angles of far positions need 64 bits)
    angle = st["pos"].double()[:, None] * st["freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    y = x.clone()
    if c["layout"] == "halves":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2] = a * cos - b * sin
        y[..., rot // 2:rot] = b * cos + a * sin
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2] = a * cos - b * sin
        y[..., 1:rot:2] = b * cos + a * sin
    y = y.to(st["qkv"].dtype)
    return y[:, :heads].contiguous(), y[:, heads:].contiguous()


def _plain_prefix(st):
    c = st["case"]
    T, heads, kv, dim, page, tail = (c[k] for k in ("T", "heads", "kv", "dim", "page", "tail"))
    group, ctx = heads // kv, c["ctx"]
    pos, late = torch.arange(ctx, device="cuda"), torch.arange(tail, device="cuda")
    node = torch.arange(T, device="cuda")
    out = []
    for p in range(c["P"]):
        b0, b1 = st["cut"][p], st["cut"][p + 1]
        n = b1 - b0
        at = st["shared"].long()[p, pos // page] * page + pos % page
        k, v = st["k"][at].float(), st["v"][at].float()             # [ctx, kv, dim]
        mine = st["table"].long()[b0:b1, late // page] * page + late % page
        ko = torch.cat([st["k"][mine], st["kn"][b0:b1]], 1).float()  # [n, tail + T, kv, dim]
        vo = torch.cat([st["v"][mine], st["vn"][b0:b1]], 1).float()
        q = st["q"][b0:b1].float().reshape(n, T, kv, group, dim)
        qs = q.permute(2, 0, 1, 3, 4).reshape(kv, n * T * group, dim)
        s = torch.matmul(qs, k.permute(1, 2, 0).contiguous())
        s = s.reshape(kv, n, T, group, ctx).permute(1, 0, 2, 3, 4)
        qo = q.permute(0, 2, 1, 3, 4).reshape(n, kv, T * group, dim)
        so = torch.matmul(qo, ko.permute(0, 2, 3, 1).contiguous())
        s = torch.cat([s, so.reshape(n, kv, T, group, tail + T)], -1) / math.sqrt(dim)
        on = torch.cat([(pos < st["shared_len"][p]).expand(n, T, ctx),
                        (late < st["len"][b0:b1, None])[:, None].expand(n, T, tail),
                        ((st["sees"][b0:b1, :, None] >> node) & 1) != 0], 2)
        s = s.masked_fill_(~on[:, None, :, None], -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True))
        e /= e.sum(-1, keepdim=True)
        es = e[..., :ctx].permute(1, 0, 2, 3, 4).reshape(kv, n * T * group, ctx)
        o = torch.matmul(es, v.transpose(0, 1).contiguous())
        o = o.reshape(kv, n, T, group, dim).permute(1, 2, 0, 3, 4)
        eo = e[..., ctx:].reshape(n, kv, T * group, tail + T)
        oo = torch.matmul(eo, vo.transpose(1, 2).contiguous())
        o = o + oo.reshape(n, kv, T, group, dim).permute(0, 2, 1, 3, 4)
        out.append(o.reshape(n, T, heads, dim).to(st["q"].dtype))
    return torch.cat(out)


def _plain_select(st):
    c = st["case"]
    G, W, V, K = c["G"], c["W"], c["V"], c["K"]
    # (scores of beams lie close together: 64 bits)
    x = st["x"][:, :V].double()
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    score = st["score"].double()[:, None] + (x - lse)
    done = st["done"] != 0
    score = torch.where(done[:, None], -math.inf, score)
    score[:, 0] = torch.where(done, st["score"].double(), score[:, 0])  # (0 pads)
    best, at = torch.sort(score.reshape(G, W * V), dim=1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    there = best > -math.inf
    parent = torch.where(there, at // V, -1).int()
    ids = torch.where(there, at % V, -1).int()
    ended = done.reshape(G, W).gather(1, parent.long().clamp(min=0)) | (ids == _EOS)
    return parent, ids, best.float(), (ended & there).to(torch.uint8)


def _reordered(st):
    """Tables and lengths of the chosen beams, what each group lacks, and the pairs of
    slots to copy."""
    c = st["case"]
    G, W, page = c["G"], c["W"], c["page"]
    per = st["table"].shape[1]
    g, w, col = (torch.arange(n, device="cuda") for n in (G, W, per))
    parent = st["parent"].long().reshape(G, W)
    length = st["len"].long().reshape(G, W).gather(1, parent)
    full, rem = length // page, length % page
    need = ((length + c["ahead"] + page - 1) // page).clamp(max=per)
    old = st["table"].long().reshape(G, W, per)[g[:, None], parent]
    eldest = ~((parent[:, :, None] == parent[:, None]) & (w < w[:, None])).any(2)
    keep = (col < full[..., None]) | ((col == full[..., None]) & (rem > 0)[..., None]
                                      & eldest[..., None])
    fresh = (col < need[..., None]) & ~keep
    n_pages = st["k"].shape[1] // page
    used = torch.zeros((G, n_pages + 1), dtype=torch.bool, device="cuda")
    used.scatter_(1, torch.where(keep, old, n_pages).reshape(G, -1), True)
    pool = st["pool"].long()
    free = ~used.gather(1, pool)
    order = torch.sort((~free).int(), dim=1, stable=True).indices
    rank = fresh.reshape(G, -1).long().cumsum(1) - 1
    there = rank < free.sum(1, keepdim=True)
    page_of = pool.gather(1, order).gather(1, rank.clamp(0, pool.shape[1] - 1))
    new = torch.where(there, page_of, -1).reshape(G, W, per)
    table = torch.where(keep, old, torch.where(fresh, new, -1))
    missing = (fresh.reshape(G, -1).sum(1) - free.sum(1)).clamp(min=0)
    i = torch.arange(page, device="cuda")
    at = full.clamp(max=per - 1)[..., None]
    src, dst = old.gather(2, at), table.gather(2, at)
    moved = (~eldest & (rem > 0) & (dst[..., 0] >= 0))[..., None] & (i < rem[..., None])
    return table, length, missing, (src * page + i)[moved], (dst * page + i)[moved]


def _plain_reorder(st):
    table, length, missing, src, dst = _reordered(st)
    st["k"][:, dst] = st["k"][:, src]
    st["v"][:, dst] = st["v"][:, src]
    return table.reshape(st["table"].shape).int(), length.reshape(-1).int(), missing.int(), \
        st["k"], st["v"]


# ---- the library's calls -----------------------------------------------------
@functools.lru_cache(maxsize=1)
def _library():
    """The binding and one handle per program: its stream and workspaces outlive
    the inputs."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "project-zero_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import pzsample as pz
    s = pz.Sampler(1024, 1024)
    s.set_eos([_EOS])
    return pz, s


def _call(st):
    """The C call of one pass with its arguments, marshalled once as a C program
    has them."""
    pz, s = _library()
    c, lib, h = st["case"], s.lib, s.h
    kind = {"bf16": pz.PZ_BF16, "fp16": pz.PZ_F16, "fp32": pz.PZ_F32}.get(c.get("type"))
    if c["op"] == "rope":
        n, heads, kv, dim = c["n"], c["heads"], c["kv"], c["dim"]
        how = pz.qk_rope(type=kind, n_heads=heads, n_kv_heads=kv, head_dim=dim,
                         d_q_norm=st.get("q_norm"), d_k_norm=st.get("k_norm"), eps=_EPS,
                         rot_dim=c["rot"], d_freq=st["freq"], amplitude=1.0,
                         layout=pz.PZ_ROPE_HALVES if c["layout"] == "halves"
                         else pz.PZ_ROPE_PAIRS)
        ld, q = (heads + 2 * kv) * dim, st["qkv"].data_ptr()
        return lib.pz_qk_norm_rope, (h, ctypes.byref(how), q, ld,
                                     q + heads * dim * st["qkv"].element_size(), ld,
                                     st["q_out"].data_ptr(), heads * dim,
                                     st["k_out"].data_ptr(), kv * dim, n,
                                     st["pos"].data_ptr()), how
    if c["op"] == "select":
        return lib.pz_beam_select, (h, st["x"].data_ptr(), c["ld"], c["G"], c["W"], c["V"],
                                    st["score"].data_ptr(), st["done"].data_ptr(), 0, c["K"],
                                    st["parent"].data_ptr(), st["ids"].data_ptr(),
                                    st["score_out"].data_ptr(), st["done_out"].data_ptr()), None
    row = c["kv"] * c["dim"]

    def cache(k, v):
        return pz.kv_cache(type=kind, n_kv_heads=c["kv"], head_dim=c["dim"], d_k=k, d_v=v, ld=row,
                           n_blocks=k.shape[0] // c["page"], block_size=c["page"],
                           d_blocks=st["table"], max_blocks=st["table"].shape[1],
                           d_len=st["len"])
    if c["op"] == "reorder":
        kept = [cache(st["k"][i], st["v"][i]) for i in range(c["layers"])]
        layers = (pz.KvCache * c["layers"])(*kept)
        return lib.pz_beam_reorder, (h, layers, c["layers"], c["G"], c["W"],
                                     st["parent"].data_ptr(), st["pool"].data_ptr(),
                                     st["pool"].shape[1], c["ahead"], st["table_out"].data_ptr(),
                                     st["len_out"].data_ptr(), st["missing"].data_ptr()), kept
    one = cache(st["k"], st["v"])
    shared = pz.kv_prefix(d_blocks=st["shared"], max_blocks=st["shared"].shape[1],
                          d_len=st["shared_len"], n_prefixes=c["P"],
                          d_first=None if c["even"] else st["first"])
    q = c["heads"] * c["dim"]
    return lib.pz_prefix_attention, (h, ctypes.byref(one), ctypes.byref(shared),
                                     st["kn"].data_ptr(), st["vn"].data_ptr(), row, c["B"],
                                     c["T"], None, st["sees"].data_ptr(), c["heads"],
                                     1.0 / math.sqrt(c["dim"]), st["q"].data_ptr(), q,
                                     st["out"].data_ptr(), q), (one, shared)


def _own(st):
    if "call" not in st:
        *st["call"], st["kept"] = _call(st)
    f, args = st["call"]
    rc = f(*args)
    if rc:
        raise RuntimeError(f"{f.__name__} returned {rc}")
    op = st["case"]["op"]
    if op == "rope":
        return st["q_out"], st["k_out"]
    if op == "prefix":
        return st["out"]
    if op == "select":
        return st["parent"], st["ids"], st["score_out"], st["done_out"]
    return st["table_out"], st["len_out"], st["missing"], st["k"], st["v"]


def run(st):
    if own:
        return _own(st)
    return {"rope": _plain_rope, "prefix": _plain_prefix, "select": _plain_select,
            "reorder": _plain_reorder}[st["case"]["op"]](st)


def work(case):
    op = case["op"]
    size = 4 if case.get("type") == "fp32" else 2
    if op == "rope":
        n, dim, rows = case["n"], case["dim"], case["n"] * (case["heads"] + case["kv"])
        norms = 2 * 4 * dim if case["norm"] else 0
        return {"bytes": 2 * rows * dim * size + 4 * n + 2 * case["rot"] + norms,
                "flops": rows * ((4 * dim if case["norm"] else 0) + 3 * case["rot"])}
    if op == "select":
        rows = case["G"] * case["W"]
        live = rows * (1 - case["done"]) / (case["W"] if case["first"] else 1)
        return {"bytes": 4 * live * case["V"] + 5 * rows + 13 * case["G"] * case["K"],
                "flops": 0}
    if op == "reorder":
        G, W, page = case["G"], case["W"], case["page"]
        twins = W * (1 - 1 / W) ** W  # beams whose parent has an elder child, on average
        half = (min(page, case["ctx"]) - 1) / 2 if page <= case["ctx"] else case["ctx"] / 2
        pages = (case["ctx"] / 2 + case["ahead"]) / page
        return {"bytes": G * (twins * half * 2 * 2 * size * case["layers"] * case["kv"]
                              * case["dim"] + W * (8 * pages + 12)), "flops": 0}
    B, T, row = case["B"], case["T"], 2 * case["kv"] * case["dim"]
    ctx, tail = case["ctx"], case["tail"]
    if case["ragged"]:
        ctx, tail = ((ctx + 1) // 2 + ctx) / 2, tail / 2
    q = 2 * case["heads"] * case["dim"]
    return {"bytes": 2 * row * (case["P"] * ctx + B * (tail + T)) + B * T * (2 * q + 8)
            + 4 * (case["P"] * ctx + B * tail) / case["page"],
            "flops": 2 * q * B * T * (ctx + tail + (T + 1) / 2)}


# ---- the definitions in 64 bits ----------------------------------------------
def _exact_rope(case, st):
    n, heads, kv, dim, rot = (case[k] for k in ("n", "heads", "kv", "dim", "rot"))
    # pairs of a head's elements as complex numbers times exp(i angle)
    one = torch.arange(rot // 2, device="cuda")
    first, second = (one, one + rot // 2) if case["layout"] == "halves" else (2 * one, 2 * one + 1)
    angle = torch.outer(st["pos"].double(), st["freq"].double())
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    out = []
    for part, m, name in ((st["qkv"][:, :heads * dim], heads, "q_norm"),
                          (st["qkv"][:, heads * dim:(heads + kv) * dim], kv, "k_norm")):
        y = part.double().reshape(n, m, dim)
        if case["norm"]:
            y = y / (y.pow(2).sum(-1, keepdim=True) / dim + float(np.float32(_EPS))).sqrt()
            y = y * st[name].double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y = y.index_copy(2, first, z.real).index_copy(2, second, z.imag)
        out.append(y)
    return tuple(out)


def _exact_prefix(case, st):
    B, T, heads, kv, dim, page = (case[k] for k in ("B", "T", "heads", "kv", "dim", "page"))
    if B * heads > 8192:
        return None
    group = heads // kv
    out = torch.empty((B, T, heads, dim), dtype=torch.float64, device="cuda")
    sl, tl = st["shared_len"].tolist(), st["len"].tolist()

    def slots(pages, n):
        p = torch.arange(n, device="cuda")
        return pages.long()[p // page] * page + p % page
    for p in range(case["P"]):
        at = slots(st["shared"][p], sl[p])
        ks, vs = st["k"][at].double(), st["v"][at].double()
        for b in range(st["cut"][p], st["cut"][p + 1]):
            mine = slots(st["table"][b], tl[b])
            k = torch.cat([ks, st["k"][mine].double(), st["kn"][b].double()])
            v = torch.cat([vs, st["v"][mine].double(), st["vn"][b].double()])
            see = torch.ones((T, len(k)), dtype=torch.bool, device="cuda")
            for i in range(T):
                see[:, len(k) - T + i] = (st["sees"][b] >> i) & 1 == 1
            for h in range(kv):
                kh, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
                q = st["q"][b, :, h * group:(h + 1) * group].double().reshape(T * group, dim)
                s = (q @ kh * dim ** -0.5).reshape(T, group, -1)
                w = torch.softmax(torch.where(see[:, None], s, -math.inf), -1)
                out[b, :, h * group:(h + 1) * group] = (w.reshape(T * group, -1) @ vh).reshape(
                    T, group, dim)
    return out


def _exact_select(case, st):
    G, W, V, K = (case[k] for k in ("G", "W", "V", "K"))
    out = torch.full((G, K), -math.inf, dtype=torch.float64)
    score, done = st["score"].double().cpu(), st["done"].cpu()
    for g in range(G):
        of_group = []
        for r in range(g * W, (g + 1) * W):
            if done[r]:
                of_group.append(score[r:r + 1])
            else:
                row = torch.log_softmax(st["x"][r, :V].double(), 0)
                of_group.append(score[r] + row.topk(min(K, V)).values.cpu())
        best = torch.cat(of_group).sort(descending=True).values[:K]
        out[g, :len(best)] = best
    return None, None, out, None


def _exact_reorder(case, st):
    G, W, page, per = case["G"], case["W"], case["page"], st["table"].shape[1]
    table, pool = st["table"].reshape(G, W, per).tolist(), st["pool"].tolist()
    parent, length = st["parent"].reshape(G, W).tolist(), st["len"].reshape(G, W).tolist()
    k, v = st["k"].double(), st["v"].double()
    for g in range(G):
        used, heirs = set(), set()
        for p in parent[g]:
            used.update(table[g][p][:(length[g][p] + page - 1) // page])
        spare = [p for p in pool[g] if p not in used]
        for w in range(W):
            p, n = parent[g][w], length[g][parent[g][w]]
            at = n // page
            most = min(per, (n + case["ahead"] + page - 1) // page)
            if p not in heirs:
                heirs.add(p)
                at += n % page > 0
                spare = spare[max(0, most - at):]
                continue
            if n % page:
                a, b = table[g][p][at] * page, spare[0] * page
                k[:, b:b + n % page] = k[:, a:a + n % page].clone()
                v[:, b:b + n % page] = v[:, a:a + n % page].clone()
            spare = spare[max(0, most - at):]
    return None, None, None, k, v


def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "prefix": _exact_prefix, "select": _exact_select,
            "reorder": _exact_reorder}[case["op"]](case, st)
