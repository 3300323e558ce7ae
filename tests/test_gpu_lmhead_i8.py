"""The LM head in 8-bit integers (pz_quant_rows_i8, pz_lm_head_i8,
pz_lm_head_argmax_i8).  Everything is defined to the bit: scales and quotients
are correctly rounded fp32, the sum is exact, and two fp32 products follow, so
numpy's integers and fp32 operations give the expected values."""
import ctypes

import numpy as np
import pytest

import pz_oracle as po
import pzsample as pz
from conftest import to_dev

pytestmark = pytest.mark.gpu

F = np.float32


def quant(x):
    """Scales and int8 of fp32 rows."""
    x = np.asarray(x, F)
    with np.errstate(all="ignore"):
        fin = np.isfinite(x).all(1)
        sc = np.where(fin, np.abs(np.where(np.isfinite(x), x, 0)).max(1) / F(127), F(np.nan))
        sc = sc.astype(F)
        q = np.rint(x / sc[:, None]).clip(-127, 127)
        q = np.where((fin & (sc != 0))[:, None], q, 0)
    return np.nan_to_num(q).astype(np.int8), sc


def product(w, sw, xq, sx):
    acc = (xq.astype(np.float64) @ w.astype(np.float64).T)  # exact: below 2^31
    with np.errstate(all="ignore"):
        return (acc.astype(F) * sw[None, :]) * sx[:, None]


def argmax(row):
    row = np.ascontiguousarray(row, F)
    return po.oracle().orc_argmax(row.ctypes.data_as(ctypes.c_void_p), row.size)


def same(got, exp, label=""):
    ok = (got.view(np.uint32) == exp.view(np.uint32)) | (np.isnan(got) & np.isnan(exp))
    assert ok.all(), (label, np.argwhere(~ok)[:4], got[~ok][:4], exp[~ok][:4])


def bf16(a):
    u = np.ascontiguousarray(a, F).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def run_quant(torch, x, kind, ldx, ldq, offset, label=""):
    rows, n = x.shape
    if kind == pz.PZ_F32:
        raw, val = x, x
    elif kind == pz.PZ_BF16:
        raw = bf16(x)
        val = (raw.astype(np.uint32) << 16).view(F)
    else:
        with np.errstate(over="ignore"):
            raw = x.astype(np.float16)
        val, raw = raw.astype(F), raw.view(np.uint16)
    wide = np.zeros(rows * ldx + offset, raw.dtype)
    np.lib.stride_tricks.as_strided(wide[offset:], (rows, n),
                                    (ldx * raw.itemsize, raw.itemsize))[:] = raw
    d_wide = to_dev(torch, wide.view(np.int16) if raw.dtype == np.uint16 else wide)
    d_q = torch.full((rows * ldq + offset,), 99, dtype=torch.int8, device="cuda")
    d_s = torch.empty(rows, device="cuda")
    with pz.Sampler(1, 16) as s:
        s.quant_rows_i8(d_wide.data_ptr() + offset * raw.itemsize, kind, ldx, rows, n,
                        d_q.data_ptr() + offset, ldq, d_s)
        s.sync()
    q, sc = quant(val)
    same(d_s.cpu().numpy(), sc, (label, "scale"))
    got = d_q.cpu().numpy()
    assert (got[:offset] == 99).all()
    full = np.full(rows * ldq, 99, np.int8)
    np.lib.stride_tricks.as_strided(full, (rows, n), (ldq, 1))[:] = q
    assert (got[offset:] == full).all(), (label, np.argwhere(got[offset:] != full)[:5])


@pytest.mark.parametrize("kind", [pz.PZ_F32, pz.PZ_BF16, pz.PZ_F16])
@pytest.mark.parametrize("n", [1, 3, 4, 5, 255, 1024, 1025, 2560, 4097, 8192, 8193, 20000])
def test_quantisation(torch_cuda, kind, n):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((7, n)) * np.logspace(-3, 3, 7)[:, None]).astype(F)
    run_quant(torch_cuda, x, kind, n, n, 0, (kind, n))
    run_quant(torch_cuda, x, kind, n + 3, n + 5, 1, (kind, n, "odd strides"))


@pytest.mark.parametrize("kind", [pz.PZ_F32, pz.PZ_BF16, pz.PZ_F16])
def test_quantisation_of_special_rows(torch_cuda, kind):
    n = 300
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, n)).astype(F)
    x[0] = 0.0
    x[1, 7] = np.inf
    x[2, 8] = -np.inf
    x[3, 9] = np.nan
    x[4] = -0.0
    x[5] = 1e-45      # the scale underflows to 0
    x[6] = np.where(np.arange(n) % 2, 2.5e-43, 1e-43)  # a subnormal scale
    x[7] = F(1.0)
    x[8] = np.arange(n) % 255 - 127            # scale 1: the integers themselves
    x[9] = (np.arange(n) % 254 - 127) + F(0.5)  # and halves, rounded to even
    x[9, 0] = 127
    x[10] = np.where(np.arange(n) % 2, 3e38, -3e38)
    x[11] = np.where(np.arange(n) == 5, 1e30, 1e-30)
    run_quant(torch_cuda, x, kind, n, n, 0, kind)


def run_product(torch, w, sw, xq, sx, ldx=None, ld=None, woff=0, xoff=0, label=""):
    (V, n), B = w.shape, xq.shape[0]
    ldx, ld = ldx or n, ld or V
    flat = np.full(V * n + woff, 77, np.int8)
    flat[woff:] = w.ravel()
    d_w = to_dev(torch, flat)
    xs = np.full(B * ldx + xoff, 55, np.int8)
    np.lib.stride_tricks.as_strided(xs[xoff:], (B, n), (ldx, 1))[:] = xq
    d_x = to_dev(torch, xs)
    d_sw, d_sx = to_dev(torch, sw), to_dev(torch, sx)
    d_y = torch.full((B, ld), -7.0, device="cuda")
    d_ids = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    with pz.Sampler(B, 16) as s:
        for _ in range(2):  # (the second call finds what the first left)
            s.lm_head_i8(d_w.data_ptr() + woff, d_sw, V, n, d_x.data_ptr() + xoff, d_sx, B, ldx,
                         d_y, ld)
            s.lm_head_argmax_i8(d_w.data_ptr() + woff, d_sw, V, n, d_x.data_ptr() + xoff, d_sx, B,
                                ldx, d_ids)
        s.sync()
    exp = product(w, sw, xq, sx)
    got = d_y.cpu().numpy()
    same(np.ascontiguousarray(got[:, :V]), exp, label)
    assert (got[:, V:] == -7.0).all(), (label, "past the rows")
    ids = [argmax(exp[b]) for b in range(B)]
    assert (d_ids.cpu().numpy() == ids).all(), (label, d_ids.cpu().numpy()[:8], ids[:8])


def operands(V, n, B, seed):
    rng = np.random.default_rng(seed)
    w = rng.integers(-127, 128, (V, n), dtype=np.int8)
    xq = rng.integers(-127, 128, (B, n), dtype=np.int8)
    sw = (rng.random(V) * 0.01 + 1e-4).astype(F)
    sx = (rng.random(B) + 0.1).astype(F)
    return w, sw, xq, sx


# a batch of each class of the tile rule, above and below five rows
I8_TILE_BATCHES = [1, 9, 30, 60, 100, 200, 300]
BATCHES = [1, 2, 3, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 256, 257, 300]


@pytest.mark.parametrize("B", BATCHES)
def test_every_batch(torch_cuda, B):
    for V, n in ((1000, 272), (515, 128)):
        run_product(torch_cuda, *operands(V, n, B, B), label=(V, n, B))


@pytest.mark.parametrize("n", [16, 32, 112, 128, 144, 256, 1008, 2560, 4096])
@pytest.mark.parametrize("B", [1, 20, 70])
def test_every_length(torch_cuda, n, B):
    run_product(torch_cuda, *operands(333, n, B, n + B), label=(n, B))


@pytest.mark.parametrize("n", [1, 2, 7, 15, 17, 127, 129, 1001, 2049])
@pytest.mark.parametrize("B", [1, 16, 40, 130])
def test_rows_off_16_bytes(torch_cuda, n, B):
    run_product(torch_cuda, *operands(130, n, B, n * B), label=(n, B))


def test_strides_and_offsets(torch_cuda):
    ops = operands(200, 256, 20, 6)
    run_product(torch_cuda, *ops, ldx=272, ld=204, label="fast strides")
    run_product(torch_cuda, *ops, ldx=259, ld=201, label="odd strides")
    run_product(torch_cuda, *ops, woff=1, label="W off")
    run_product(torch_cuda, *ops, xoff=3, label="x off")
    run_product(torch_cuda, *ops, woff=16, xoff=16, label="on 16")


@pytest.mark.parametrize("V", [1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 4097])
def test_every_vocabulary(torch_cuda, V):
    for B in (1, 33):
        run_product(torch_cuda, *operands(V, 160, B, V), label=(V, B))


I8_TILE_VOCABS = [3000, 9000, 13000, 20000, 33000, 40000, 60000, 90000]


@pytest.mark.parametrize("V", I8_TILE_VOCABS)
def test_every_tile(torch_cuda, V):
    """Each shape of pz_lmtile.h (test_lmhead_tiles.py shows that these reach
    them all), at lengths that end inside a stage, whole sizes on the device."""
    torch = torch_cuda
    g = torch.Generator(device="cuda")
    g.manual_seed(V)
    for B in I8_TILE_BATCHES:
        for n in (208, 400, 277):  # (277: rows off 16 bytes, shapes of their own)
            w = torch.randint(-128, 128, (V, n), generator=g, device="cuda", dtype=torch.int8)
            xq = torch.randint(-128, 128, (B, n), generator=g, device="cuda", dtype=torch.int8)
            sw = torch.rand(V, generator=g, device="cuda")
            sx = torch.rand(B, generator=g, device="cuda")
            y = torch.full((B, V), -7.0, device="cuda")
            ids = torch.empty(B, dtype=torch.int32, device="cuda")
            with pz.Sampler(B, 16) as s:
                s.lm_head_i8(w, sw, V, n, xq, sx, B, n, y, V)
                s.lm_head_argmax_i8(w, sw, V, n, xq, sx, B, n, ids)
                s.sync()
            acc = xq.float() @ w.float().t().contiguous()  # exact: 2^14 n < 2^24
            exp = (acc * sw[None]) * sx[:, None]
            assert torch.equal(y, exp), (V, B, n)
            first = torch.where(exp == exp.amax(1, keepdim=True),
                                torch.arange(V, device="cuda"), V).amin(1)
            assert torch.equal(ids.long(), first), (V, B, n)


def test_the_largest_sums(torch_cuda):
    """+-128 and +-127 throughout at the longest rows: the ends of int32, whose
    rounding to fp32 is part of the definition."""
    for n in (pz.PZ_I8_MAX_N, 131056):
        w = np.full((3, n), -128, np.int8)
        w[1] = 127
        w[2, ::2] = 127
        xq = np.stack([np.full(n, -128, np.int8), np.full(n, 127, np.int8)])
        run_product(torch_cuda, w, np.array([1, 0.37, 3], F), xq, np.array([1, 0.01], F), label=n)


def test_ties_nan_and_zero_scales(torch_cuda):
    """Equal channels tie to the lowest id; a NaN or zero scale of a token or a
    channel goes through both calls as through the formula."""
    w, sw, xq, sx = operands(700, 144, 37, 9)
    w[300:] = w[100]
    sw[300:] = sw[100]
    w[100:] = w[100]
    sx[3] = np.nan
    sx[5] = 0.0
    sx[7] = np.inf
    run_product(torch_cuda, w, sw, xq, sx, label="token scales")
    sw[0] = np.nan
    run_product(torch_cuda, w, sw, xq, sx, label="NaN logit 0")
    sw[0], sw[50], sw[101] = 0.0, np.nan, np.inf
    run_product(torch_cuda, w, sw, xq, sx, label="channel scales")


@pytest.mark.parametrize("V,n", [(128256, 2560), (2100, 131056)])
@pytest.mark.parametrize("B", [1, 9, 32, 60, 100, 256])
def test_large_weights(torch_cuda, V, n, B):
    """Weights past the Infinity Cache: quantised from fp32 on the device, product
    and ids."""
    torch = torch_cuda
    g = torch.Generator(device="cuda")
    g.manual_seed(B)
    w = torch.randint(-127, 128, (V, n), generator=g, device="cuda", dtype=torch.int8)
    sw = torch.rand(V, generator=g, device="cuda") * 1e-3
    x = torch.randn((B, n), generator=g, device="cuda")
    xq = torch.empty((B, n), dtype=torch.int8, device="cuda")
    sx = torch.empty(B, device="cuda")
    y = torch.empty((B, V), device="cuda")
    ids = torch.empty(B, dtype=torch.int32, device="cuda")
    with pz.Sampler(B, 16) as s:
        s.quant_rows_i8(x, pz.PZ_F32, n, B, n, xq, n, sx)
        s.lm_head_i8(w, sw, V, n, xq, sx, B, n, y, V)
        s.lm_head_argmax_i8(w, sw, V, n, xq, sx, B, n, ids)
        s.sync()
    q, sc = quant(x.cpu().numpy())
    assert (xq.cpu().numpy() == q).all()
    same(sx.cpu().numpy(), sc)
    acc = torch.empty((B, V), dtype=torch.float64, device="cuda")
    step = (1 << 26) // n
    for r in range(0, V, step):
        acc[:, r:r + step] = xq.double() @ w[r:r + step].double().t().contiguous()
    exp = (acc.float() * sw[None]) * sx[:, None]
    assert torch.equal(y, exp)
    first = torch.where(exp == exp.amax(1, keepdim=True),
                        torch.arange(V, device="cuda"), V).amin(1)
    assert torch.equal(ids.long(), first)


def test_refused_calls(torch_cuda):
    torch = torch_cuda
    w = torch.zeros((8, 16), dtype=torch.int8, device="cuda")
    f = torch.zeros(8, device="cuda")
    y = torch.zeros((8, 8), device="cuda")
    ids = torch.zeros(8, dtype=torch.int32, device="cuda")
    with pz.Sampler(4, 16) as s:
        for call, code in (
                (lambda: s.lm_head_i8(w, f, 8, 16, w, f, 5, 16, y, 8), pz.PZ_ERANGE),
                (lambda: s.lm_head_i8(w, f, 8, 16, w, f, 4, 16, y, 7), pz.PZ_EINVAL),
                (lambda: s.lm_head_i8(w, f, 8, 16, w, f, 4, 16, None, 8), pz.PZ_EINVAL),
                (lambda: s.lm_head_argmax_i8(w, f, 8, 16, w, f, 4, 16, None), pz.PZ_EINVAL),
                (lambda: s.lm_head_argmax_i8(w, f, 8, 131072, w, f, 4, 131072, ids),
                 pz.PZ_ERANGE),
                (lambda: s.quant_rows_i8(w, 9, 16, 8, 16, w, 16, f), pz.PZ_EINVAL)):
            with pytest.raises(pz.PzError) as e:
                call()
            assert e.value.code == code
        s.lm_head_i8(w, f, 8, 16, w, f, 0, 16, y, 8)  # no rows: nothing to do
        s.sync()


def test_captured_and_replayed(torch_cuda):
    """Quantisation, logits and greedy ids in one graph, replayed on new
    activations with eager calls between."""
    torch = torch_cuda
    V, n, B = 3000, 320, 6
    w, sw, _, _ = operands(V, n, B, 2)
    d_w, d_sw = to_dev(torch, w), to_dev(torch, sw)
    rng = np.random.default_rng(77)
    d_x = to_dev(torch, rng.standard_normal((B, n)).astype(F))
    xq = torch.empty((B, n), dtype=torch.int8, device="cuda")
    sx, y = torch.empty(B, device="cuda"), torch.empty((B, V), device="cuda")
    ids = torch.empty(B, dtype=torch.int32, device="cuda")

    def calls(s, sync):
        lib, h = s.lib, s.h
        p = [t.data_ptr() for t in (d_x, xq, sx, d_w, d_sw, y, ids)]
        assert lib.pz_quant_rows_i8(h, p[0], pz.PZ_F32, n, B, n, p[1], n, p[2]) == 0
        assert lib.pz_lm_head_i8(h, p[3], p[4], V, n, p[1], p[2], B, n, p[5], V) == 0
        assert lib.pz_lm_head_argmax_i8(h, p[3], p[4], V, n, p[1], p[2], B, n, p[6]) == 0
        if sync:
            s.sync()

    with pz.Sampler(B, 16) as s:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(s.stream)):
            calls(s, False)
        for i in range(4):
            x = rng.standard_normal((B, n)).astype(F)
            d_x.copy_(torch.from_numpy(x))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            q, sc = quant(x)
            exp = product(w, sw, q, sc)
            same(y.cpu().numpy(), exp, i)
            want = [argmax(exp[b]) for b in range(B)]
            assert (ids.cpu().numpy() == want).all(), i
            y.zero_()
            calls(s, True)
            same(y.cpu().numpy(), exp, (i, "eager"))
            assert (ids.cpu().numpy() == want).all(), i
