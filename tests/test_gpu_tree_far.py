"""Tree attention of many rows over slots and nodes that lie far apart
(pz_tree_attention): the kernel that shares keys takes 32-bit offsets within a
load, up to strides just below 2^26 and 2^24 elements."""
import pytest

import pzsample as pz
from test_gpu_tree import Case

pytestmark = pytest.mark.gpu

POSITIONS = 37
# name: nodes, heads, key heads, ld, ld_n, whether the kernel that shares keys takes it
FAR = {
    "slots, 16 rows a wave": (40, 2, 2, (1 << 26) - 8, 128, True),
    "slots, 32 rows a wave": (20, 8, 2, (1 << 26) - 8, 128, True),
    "slots past it": (40, 2, 2, 1 << 26, 128, False),
    "nodes, 16 rows a wave": (64, 2, 2, 128, (1 << 24) - 8, True),
    "nodes, 32 rows a wave": (64, 4, 2, 128, (1 << 24) - 8, True),
    "nodes past it": (64, 2, 2, 128, 1 << 24, False),
}


def table_of(kv):
    """Entries of pages of 8 that make 16 tiles a CU of kv key heads."""
    return 16 * 256 * 4 // kv


def spread(torch, rows, ld, other):
    """Two tensors [n, 128] as rows `ld` apart of one buffer: (buffer, offset of
    the second); ld 128: a buffer each."""
    if ld < 1024:
        return rows, other
    n = len(rows)
    pool = torch.empty(((n - 1) * ld + 1024,), dtype=rows.dtype, device="cuda")
    for first, r in ((0, rows), (512, other)):
        pool[first:].as_strided((n, 128), (ld, 1)).copy_(r)
    return pool, pool[512:]


@pytest.mark.parametrize("form", list(FAR))
def test_far_strides(torch_cuda, form):
    torch = torch_cuda
    T, heads, kv, ld, ld_n, _ = FAR[form]
    c = Case(torch, "bf16", [POSITIONS], T, heads, kv, 64, 8, 17, spare=0).random_tree(3)
    d = c.device()
    pages = (POSITIONS + 7) // 8
    slots = c.slots(0, torch.arange(pages * 8))
    k, v = spread(torch, c.k[slots].cuda(), ld, c.v[slots].cuda())
    kn, vn = spread(torch, d["kn"][0], ld_n, d["vn"][0])
    table = torch.full((1, table_of(kv)), -1, dtype=torch.int32)
    table[0, :pages] = torch.arange(pages)
    cache = pz.kv_cache(type=pz.PZ_BF16, n_kv_heads=kv, head_dim=64, d_k=k, d_v=v, ld=ld,
                        n_blocks=pages, block_size=8, d_blocks=table.cuda(),
                        max_blocks=table.shape[1], d_len=d["lens"])
    with pz.Sampler(1, 16) as s:
        s.tree_attention(cache, kn, vn, ld_n, 1, T, heads, c.scale, d["q"], heads * 64, d["out"],
                         heads * 64, d_tree=d["tree"])
        s.sync()
    c.check(d["out"], form)
