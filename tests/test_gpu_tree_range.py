"""The ends of tree attention's ranges (pz_tree_attention): scores far from zero.

Every case runs through both kernels: the one of few rows or little work, whole
and in splits, and the one of many rows, whole and in splits."""
import numpy as np
import pytest

import pzsample as pz
from test_gpu_tree import Case, KINDS

pytestmark = pytest.mark.gpu

# name: sequences, nodes, heads, key heads, positions of the longest sequence
FORMS = {
    "one tile": (2, 3, 4, 2, 20),
    "two row tiles": (1, 12, 8, 2, 60),
    "splits": (1, 2, 4, 1, 3000),
    "many splits of more rows": (1, 20, 2, 1, 5000),
    "many rows": (32, 33, 8, 8, 50),
    "many rows, two tiles a wave": (32, 40, 16, 8, 50),
    "many rows in splits": (8, 36, 8, 8, 4000),
    "many rows in splits, two tiles a wave": (2, 70 // 2, 32, 8, 9000),
}


@pytest.fixture(scope="module")
def sampler(torch_cuda):
    with pz.Sampler(1, 16) as s:
        yield s


def case(torch, kind, form, D, seed, short=True):
    """A Case of a form whose sequences but the first are shorter, each node
    seeing itself alone besides the cache."""
    B, T, heads, kv, ctx = FORMS[form]
    lens = [ctx if b == 0 or not short else (17 * b) % (ctx + 1) for b in range(B)]
    c = Case(torch, kind, lens, T, heads, kv, D, 16, seed)
    c.tree = np.tile(np.uint64(1) << np.arange(T, dtype=np.uint64), (B, 1))
    return c


def call(s, c, scale=None):
    if scale is not None:
        c.scale = scale
    d = c.device()
    c.call(s, d)
    s.sync()
    return d["out"]


def only_first(c):
    """q and k whose products are those of their first elements."""
    for t in (c.q, c.kn):
        t.reshape(*t.shape[:-1], -1, c.D)[..., 1:] = 0
    c.k.reshape(len(c.k), -1, c.D)[..., 1:] = 0
    return [t.reshape(*t.shape[:-1], -1, c.D)[..., 0] for t in (c.q, c.kn, c.k)]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("product", [-1.125, 1.125])
def test_scores_at_the_ends_of_fp32(torch_cuda, sampler, kind, form, product):
    """scale 2e38, the largest: a node that attends itself alone gets its value,
    whatever its score, and of a longer sequence the largest score's position
    takes all the weight.  Products are exact, and scores of different keys lie
    0.0625 * 2e38 apart, so results are values of v, bit for bit."""
    torch = torch_cuda
    c = case(torch, kind, form, 64, 5)
    q, kn, k = only_first(c)
    q[:] = 1.0
    kn[:] = product - 0.0625
    k[:] = product - 0.125
    best = c.lens.copy()
    for b in range(c.B):
        if c.lens[b] and b % 2 == 0:  # a position that wins, in the last third
            best[b] = c.lens[b] - 1 - int(c.lens[b]) // 5
            k[c.slots(b, torch.tensor([int(best[b])]))] = product
    got = call(sampler, c, 2.0e38).reshape(c.B, c.T, c.kv, -1, 64).cpu()
    v = c.v.reshape(-1, c.kv, 64)
    for b in range(c.B):
        if best[b] < c.lens[b]:
            want = v[c.slots(b, torch.tensor([int(best[b])]))][0][None].expand(c.T, -1, -1)
        else:
            want = c.vn[b].reshape(c.T, c.kv, 64)
        assert torch.equal(got[b], want[:, :, None].expand_as(got[b])), b


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", [2.0 ** 18, 2.0 ** 24, 2.0 ** 60])
def test_scores_past_the_integers_of_fp32(torch_cuda, sampler, kind, form, scale):
    """Whole-number products times a large scale: exact scores, of which equal
    ones share the weight and others get none.  The result is the mean of the
    values at the largest product: n equal weights (exact in 16 bits, a power of
    two), fp32 sums (n 2^-24 of sum |v|) and one rounding to the type."""
    torch = torch_cuda
    c = case(torch, kind, form, 64, 6)
    g = torch.Generator().manual_seed(6)
    q, kn, k = only_first(c)
    q[:] = torch.randint(-3, 4, q.shape, generator=g).to(c.dt) * 31 + 1
    kn[:] = torch.randint(-40, 41, kn.shape, generator=g).to(c.dt)
    k[:] = torch.randint(-40, 41, k.shape, generator=g).to(c.dt)
    got = call(sampler, c, scale).reshape(c.B, c.T, c.kv, -1, 64).double().cpu().numpy()
    q = q.double().numpy().reshape(c.B, c.T, c.kv, -1)
    h = KINDS[kind][1]
    for b in range(c.B):
        at = c.slots(b, torch.arange(int(c.lens[b])))
        kc, vc = k[at].double().numpy(), c.v.reshape(-1, c.kv, 64)[at].double().numpy()
        for t in range(c.T):
            ks = np.concatenate([kc, kn[b, t][None].double().numpy()])
            vs = np.concatenate([vc, c.vn[b, t].reshape(1, c.kv, 64).double().numpy()])
            for hk in range(c.kv):
                s = ks[:, hk, None] * q[b, t, hk]                     # [keys, group]
                top = (s == s.max(0)).astype(np.float64)
                n = top.sum(0)[:, None]
                mean = top.T @ vs[:, hk] / n
                tol = h * np.abs(mean) + (1 + h) * n * 2.0 ** -23 * (top.T @ np.abs(vs[:, hk]) / n)
                tol += 2.0 ** -25 if kind == "fp16" else 0.0
                assert (np.abs(got[b, t, hk] - mean) <= tol).all(), (b, t, hk)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("form", list(FORMS))
def test_scores_around_the_choice(torch_cuda, sampler, kind, form):
    """Rows of one wave whose scores pass 2^12 and rows whose scores stay below,
    maxima that grow past it and away from it: within the usual bound."""
    c = case(torch_cuda, kind, form, 128, 7)
    g = torch_cuda.Generator().manual_seed(7)
    q, kn, k = only_first(c)
    q[:] = torch_cuda.randint(-2, 3, q.shape, generator=g).to(c.dt) * 20
    kn[:] = torch_cuda.randint(-90, 91, kn.shape, generator=g).to(c.dt)
    at = c.slots(0, torch_cuda.arange(int(c.lens[0])))
    k[at] = (torch_cuda.arange(len(at)) * 200 // len(at) - 100).to(c.dt)[:, None]
    c.check(call(sampler, c, 1.0))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("pages", ["all", "none", "last"])
def test_scores_of_minus_infinity(torch_cuda, sampler, kind, form, pages):
    """What a row attends with a score of -infinity takes no weight beside a
    finite score; a row that attends nothing else is NaN (the quotient of zeros
    that the formula gives), one that attends nothing is zeros."""
    torch = torch_cuda
    c = case(torch, kind, form, 64, 8)
    if c.B > 1:
        c.lens[1] = 0
    q, kn, k = only_first(c)
    q[:] = 1.0
    k[:] = -float("inf")
    kn[:] = 0.0
    kn[:, ::3] = -float("inf")
    c.tree[:, 2::3] = 0  # (these see the cache alone)
    if pages != "all":
        keep = c.table.clone()
        c.table[:] = -1
        if pages == "last":
            for b in range(c.B):
                last = max(int(c.lens[b]) - 1, 0) // 16
                c.table[b, last] = keep[b, last]
    got = call(sampler, c).reshape(c.B, c.T, c.kv, -1, 64).cpu()
    for b in range(c.B):
        assert torch.isnan(got[b, ::3]).all(), b
        value = c.vn[b].reshape(c.T, c.kv, 1, 64)[1::3]
        assert torch.equal(got[b, 1::3], value.expand_as(got[b, 1::3])), b
        if c.lens[b] > 0 and pages != "none":
            assert torch.isnan(got[b, 2::3]).all(), b
        else:
            assert (got[b, 2::3] == 0).all(), b


def most_of(torch, c):
    return torch.finfo(c.dt).max


@pytest.mark.parametrize("form", list(FORMS))
def test_saturated_values(torch_cuda, sampler, form):
    """fp16 values of +-65504 throughout, one key with most of the weight, whose
    rounding differs from row to row: a mean of such values is one of them, and
    must not become infinite by the weights' rounding."""
    torch = torch_cuda
    c = case(torch, "fp16", form, 64, 9)
    q, kn, k = only_first(c)
    q[:] = 1.0 + (torch.arange(q.numel()) % 80 / 1024.0).reshape(q.shape).to(c.dt)
    kn[:] = -1000.0
    k[:] = -1000.0
    for b in range(c.B):
        at = torch.arange(int(c.lens[b]))
        k[c.slots(b, at[::32])] = 0.0
        if len(at):
            k[c.slots(b, at[len(at) - 1 - len(at) // 5:][:1])] = 5.5
    sign = torch.randint(0, 2, (64,), generator=torch.Generator().manual_seed(9)) * 2 - 1
    top = sign.to(c.dt) * most_of(torch, c)
    for v in (c.v, c.vn):
        v[:] = top.repeat(c.kv)
    c.check(call(sampler, c, float(np.log(2.0))))


@pytest.mark.parametrize("form", list(FORMS))
def test_the_largest_bf16_values(torch_cuda, sampler, form):
    """bf16 values of +-3.39e38 throughout: sums of weighted values stay in
    fp32, and the mean is finite."""
    torch = torch_cuda
    c = case(torch, "bf16", form, 64, 10)
    sign = torch.randint(0, 2, (64,), generator=torch.Generator().manual_seed(10)) * 2 - 1
    top = sign.to(c.dt) * most_of(torch, c)
    for v in (c.v, c.vn):
        v[:] = top.repeat(c.kv)
    c.check(call(sampler, c))


@pytest.mark.parametrize("form", list(FORMS))
def test_small_bf16_values(torch_cuda, sampler, form):
    """Values around 2^-90, whose weighted sums are small: the bound of ordinary
    values, scaled, and half of fp32's least step (2^-150) for each product and
    partial sum, over a normaliser of at least 2^-40."""
    torch = torch_cuda
    c = case(torch, "bf16", form, 64, 11)
    small = 2.0 ** -90
    c.v, c.vn = (v * small for v in (c.v, c.vn))  # (a power of two: exact)
    got = call(sampler, c).reshape(c.B, c.T, c.heads, 64).double().cpu().numpy()
    exp, tol = c.want()
    tol = tol + 2 * (int(c.lens.max()) + c.T) * 2.0 ** -110
    assert (np.abs(got - exp) <= tol).all(), (np.abs(got - exp) / tol).max()
