"""Caches, rows and strides past 2^32 bytes: prefix attention's kernels, reordering in its two
forms, the rotation's."""
import numpy as np
import pytest

import pzsample as pz
import test_gpu_rope as ro
from test_gpu_prefix import Shared

pytestmark = pytest.mark.gpu

FAR = (1 << 33) + (1 << 30)  # bytes


@pytest.mark.parametrize("form", ["few", "some", "wide"])
def test_prefix_attention_of_far_pages(torch_cuda, form):
    """The pages of a small cache at equal distances in a large one."""
    torch = torch_cuda
    B, heads, kv, lens = {"few": (4, 8, 2, [200, 90]), "some": (20, 8, 2, [200, 90]),
                          "wide": (140, 64, 64, [200, 129])}[form]
    c = Shared(torch, "bf16", lens, None, [b % 3 for b in range(B)], 1, heads, kv, 64, 16, seed=3)
    d = c.device()
    page = c.page * d["k"].shape[1]
    apart = FAR // (2 * page * c.n_pages) + 1
    for n in ("k", "v"):
        far = torch.empty((c.n_pages * apart, page), dtype=torch.bfloat16, device="cuda")
        far[::apart] = d[n].reshape(c.n_pages, page)
        d[n] = far
    for n in ("table", "ptable"):
        d[n] = torch.where(d[n] < 0, d[n], d[n] * apart)
    assert int(d["ptable"].max()) * page * 2 > 1 << 33
    cache = c.cache(d)
    cache.n_blocks = c.n_pages * apart
    with pz.Sampler(1, 16) as s:
        s.prefix_attention(cache, c.prefix(d), d["kn"], d["vn"], c.kn.shape[2], B, 1, heads,
                           c.scale, d["q"], c.q.shape[2], d["out"], c.q.shape[2])
        s.sync()
        c.check_tokens(d["out"], form)


@pytest.mark.parametrize("n_pool", [40, 9000])  # (in one launch, in two)
def test_reordering_of_far_pages(torch_cuda, n_pool):
    torch = torch_cuda
    page, row = 16, 128
    n_blocks = FAR // (2 * page * row)
    k, v = (torch.zeros((n_blocks, page, row), dtype=torch.bfloat16, device="cuda")
            for _ in range(2))
    last = n_blocks - n_pool
    pool = torch.arange(last, n_blocks, dtype=torch.int32, device="cuda")[None].contiguous()
    table = torch.tensor([[last + 3, last], [5, 6], [last + 1, -1]], dtype=torch.int32).cuda()
    lens = torch.tensor([21, 32, 9], dtype=torch.int32).cuda()
    for t in (k, v):
        t[last] = torch.randn((page, row), device="cuda").to(torch.bfloat16)
        t[last + 1] = torch.randn((page, row), device="cuda").to(torch.bfloat16)
    cache = pz.kv_cache(type=pz.PZ_BF16, n_kv_heads=1, head_dim=row, d_k=k, d_v=v, ld=row,
                        n_blocks=n_blocks, block_size=page, d_blocks=table, max_blocks=2,
                        d_len=lens)
    out = torch.zeros_like(table)
    nl, missing = torch.zeros_like(lens), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pz.Sampler(1, 16) as s:
        s.beam_reorder([cache], 1, 3, torch.tensor([0, 0, 0], dtype=torch.int32).cuda(), pool,
                       n_pool, 1, out, nl, missing)
        s.sync()
        assert out.tolist() == [[last + 3, last], [last + 3, last + 1], [last + 3, last + 2]]
        assert nl.tolist() == [21] * 3 and missing.tolist() == [0]
        for t in (k, v):
            for to in (last + 1, last + 2):
                assert torch.equal(t[to, :5], t[last, :5])
            assert (t[last + 2, 5:] == 0).all()


@pytest.mark.parametrize("D", [128, 66])
def test_rotation_of_far_rows(torch_cuda, D):
    torch = torch_cuda
    n, ld = 150, 1 << 25
    x = torch.zeros((n, ld), dtype=torch.bfloat16, device="cuda")
    g = np.random.default_rng(1)
    rows = torch.from_numpy(g.standard_normal((n, 3 * D)).astype(np.float32)).to(torch.bfloat16)
    x[:, :3 * D] = rows.cuda()
    freq = (10000.0 ** (-np.arange(D // 2) / (D / 2))).astype(np.float32)
    pos = g.integers(0, 5000, n).astype(np.int32)
    w = (1 + 0.1 * g.standard_normal(D)).astype(np.float32)
    dw, df, dp = (torch.from_numpy(a).cuda() for a in (w, freq, pos))
    rope = pz.qk_rope(type=pz.PZ_BF16, n_heads=2, n_kv_heads=1, head_dim=D, d_q_norm=dw,
                      d_k_norm=dw, eps=1e-6, rot_dim=D, layout=pz.PZ_ROPE_HALVES, d_freq=df,
                      amplitude=1.0)
    with pz.Sampler(1, 16) as s:
        k = x[:, 2 * D:]
        s.qk_norm_rope(rope, x, ld, k, ld, x, ld, k, ld, n, dp)
        s.sync()
    got = x[:, :3 * D].cpu().double().numpy()
    want, tol = ro.reference(rows.double().numpy(), 3, D, D, pz.PZ_ROPE_HALVES, freq, pos, w, 1e-6,
                             1.0)
    h = 2.0 ** -8
    assert (np.abs(got - want) <= h * np.abs(want) + tol * (1 + h)).all()
    assert (x[:, 3 * D:4 * D] == 0).all()
