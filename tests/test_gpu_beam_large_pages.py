"""Reordering copies of a page that has more than 2^31 pieces of 16 bytes."""
import pytest

import pzsample as pz

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_pool", [2, 9000])  # (in one launch, in two)
def test_a_page_of_more_than_2_31_pieces(torch_cuda, n_pool):
    torch = torch_cuda
    page, kv, D = 1 << 24, 9, 128
    row, length = kv * D, (1 << 24) - 5
    assert length * row // 8 > 1 << 31
    # keys and values in one buffer: two pages are 77 GB
    k = torch.empty((2, page, row), dtype=torch.int16, device="cuda")
    slab = torch.empty((1 << 16, row), dtype=torch.int16, device="cuda").random_(-30000, 30000)
    parts = page // len(slab)
    for i in range(parts):  # (each part of the first page its own, the second page 7)
        k[0, i * len(slab):(i + 1) * len(slab)] = slab + i
        k[1, i * len(slab):(i + 1) * len(slab)] = 7
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens = torch.tensor([[0], [-1]], **i32), torch.tensor([length, 0], **i32)
    out, nl, missing = torch.zeros_like(table), torch.zeros_like(lens), torch.zeros(1, **i32)
    cache = pz.kv_cache(type=pz.PZ_BF16, n_kv_heads=kv, head_dim=D, d_k=k, d_v=k, ld=row,
                        n_blocks=2, block_size=page, d_blocks=table, max_blocks=1, d_len=lens)
    with pz.Sampler(1, 16) as s:
        s.beam_reorder([cache], 1, 2, torch.zeros(2, **i32), torch.arange(n_pool, **i32), n_pool,
                       0, out, nl, missing)
        s.sync()
    assert out.tolist() == [[0], [1]] and nl.tolist() == [length] * 2 and missing.tolist() == [0]
    for i in range(parts):
        sl = slice(i * len(slab), (i + 1) * len(slab))
        if i < parts - 1:
            assert torch.equal(k[1, sl], slab + i), i
        assert torch.equal(k[0, sl], slab + i), i
    assert torch.equal(k[1, (parts - 1) * len(slab):length],
                       (slab + parts - 1)[:length - (parts - 1) * len(slab)])
    assert (k[1, length:] == 7).all()
    del k, cache
    torch.cuda.empty_cache()
