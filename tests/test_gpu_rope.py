"""Norms of queries' and keys' heads with their rotation (pz_qk_norm_rope).

Reference: 64 bits.  Bound per result, u = 2^-24, h = eps / 2 of the type:
  norm: the sum of D squares in fp32 is off by at most D u relative, its mean,
    square root and reciprocal add 3 u; y = x f w has two more roundings:
    |y error| <= |y| (D / 2 + 6) u
  cosine and sine: the angle in quarter turns is off by 3 2^-53 |t| and, rounded to
    fp32 within a quarter turn, by 2^-26; times pi / 2, with x rounded (u pi / 4), the
    series' missing terms (2e-9) and its last steps (2 u): at most 6 u + 2^-50 |angle|;
    amplitude adds one rounding
  a cos - b sin: two products and a sum, 3 u
  together with A = (|a| + |b|) |amplitude|:  A ((D / 2 + 6) + 7 + 3) u + A 2^-50 |angle|
  and the rounding to the type, h |y|, for fp16 at least 2^-25 (its smallest steps)."""
import numpy as np
import pytest

import pzsample as pz

pytestmark = pytest.mark.gpu

TYPES = {"fp32": (pz.PZ_F32, "float32", 2.0 ** -24), "bf16": (pz.PZ_BF16, "bfloat16", 2.0 ** -8),
         "fp16": (pz.PZ_F16, "float16", 2.0 ** -11)}
U = 2.0 ** -24


def reference(x, heads, D, rot, layout, freq, pos, w, eps, amp):
    """(results, bounds before the last rounding) of [n, heads * D] rows."""
    n = x.shape[0]
    y = x.astype(np.float64).reshape(n, heads, D)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + float(np.float32(eps))) * w.astype(
            np.float64)
    norm = np.abs(y) * (D / 2 + 6) * U if w is not None else np.zeros_like(y)
    out, tol = y.copy(), norm.copy()
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if layout == pz.PZ_ROPE_HALVES else (2 * i, 2 * i + 1)
    if rot:
        angle = pos.astype(np.float64)[:, None] * freq.astype(np.float64)
        c, s = np.cos(angle)[:, None] * amp, np.sin(angle)[:, None] * amp
        ya, yb = y[..., a], y[..., b]
        out[..., a] = ya * c - yb * s
        out[..., b] = yb * c + ya * s
        A = (np.abs(ya) + np.abs(yb)) * abs(amp)
        t = A * ((D / 2 + 16) * U + 2.0 ** -50 * np.abs(angle)[:, None])
        tol[..., a], tol[..., b] = t, t
    return out.reshape(n, -1), tol.reshape(n, -1)


def same_bits(torch, a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


class Case:
    def __init__(self, torch, kind, n, heads, kv, D, rot, layout, seed, norm=True, pad=0, off=0,
                 far=5000, amp=1.0, eps=1e-6, sigma=1.0):
        self.torch, self.kind, self.n, self.heads, self.kv, self.D = torch, kind, n, heads, kv, D
        self.rot, self.layout, self.amp, self.eps = rot, layout, amp, eps
        g = np.random.default_rng(seed)
        self.dt = getattr(torch, TYPES[kind][1])
        self.ld = (heads + 2 * kv) * D + pad  # queries, keys and values of a token in a row
        self.off = off
        x = torch.from_numpy(g.standard_normal((n, self.ld)).astype(np.float32) * sigma)
        self.x = x.to(self.dt)
        self.pos = g.integers(0, far, n).astype(np.int32)
        self.freq = (10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))).astype(np.float32)
        self.w = [(1 + 0.2 * g.standard_normal(D)).astype(np.float32) if norm else None
                  for _ in range(2)]

    def put(self, a):
        """On the device, `off` elements past an aligned address."""
        flat = self.torch.zeros(a.numel() + self.off, dtype=a.dtype, device="cuda")
        v = flat[self.off:].reshape(a.shape)
        v.copy_(a)
        return v

    def how(self):
        dev = lambda a: None if a is None else self.torch.from_numpy(a).cuda()  # noqa: E731
        return pz.qk_rope(type=TYPES[self.kind][0], n_heads=self.heads, n_kv_heads=self.kv,
                          head_dim=self.D, d_q_norm=dev(self.w[0]), d_k_norm=dev(self.w[1]),
                          eps=self.eps, rot_dim=self.rot, layout=self.layout,
                          d_freq=dev(self.freq), amplitude=self.amp)

    def run(self, s, in_place=False, label=""):
        torch, heads, kv, D = self.torch, self.heads, self.kv, self.D
        x = self.put(self.x)
        pos = torch.from_numpy(self.pos).cuda()
        size, q = x.element_size(), x.data_ptr()
        k = q + heads * D * size
        if in_place:
            qo, ko, ldq, ldk = q, k, self.ld, self.ld
        else:
            ldq, ldk = heads * D + self.off + 8, kv * D + self.off + 16
            oq = self.put(torch.full((self.n, ldq), 77.0, dtype=self.dt))
            ok = self.put(torch.full((self.n, ldk), 77.0, dtype=self.dt))
            qo, ko = oq.data_ptr(), ok.data_ptr()
        s.qk_norm_rope(self.how(), q, self.ld, k, self.ld, qo, ldq, ko, ldk, self.n, pos)
        s.sync()
        if in_place:
            oq, ok = x, x[:, heads * D:]
            assert same_bits(torch, x[:, (heads + kv) * D:].cpu(), self.x[:, (heads + kv) * D:]), \
                (label, "values")
        else:
            assert same_bits(torch, x.cpu(), self.x), (label, "the input")
            assert (oq[:, heads * D:].float() == 77).all() and (ok[:, kv * D:].float() == 77).all()
        return self.check(oq, ok, label)

    def check(self, oq, ok, label=""):
        heads, kv, D = self.heads, self.kv, self.D
        h = TYPES[self.kind][2]
        for part, got, m, at, w in (("q", oq, heads, 0, self.w[0]),
                                    ("k", ok, kv, heads * D, self.w[1])):
            if not m:
                continue
            x = self.x[:, at:at + m * D].double().numpy()
            with np.errstate(invalid="ignore", over="ignore"):
                want, tol = reference(x, m, D, self.rot, self.layout, self.freq, self.pos, w,
                                      self.eps, self.amp)
            got = got[:, :m * D].double().cpu().numpy()
            bad = ~np.isfinite(want)
            assert (np.isfinite(got) == ~bad).all(), (label, part, "not finite")
            t = h * np.abs(want) + tol * (1 + h) + (2.0 ** -25 if self.kind == "fp16" else 1e-37)
            off = (np.abs(got - want) - t)[~bad]
            assert off.size == 0 or off.max() <= 0, (label, part, off.max())
        return oq, ok


@pytest.fixture(scope="module")
def sampler(torch_cuda):
    with pz.Sampler(1, 16) as s:
        yield s


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", [pz.PZ_ROPE_HALVES, pz.PZ_ROPE_PAIRS])
@pytest.mark.parametrize("D", [8, 16, 64, 80, 96, 128, 192, 256, 512, 1024])
def test_heads(torch_cuda, sampler, kind, layout, D):
    for i, (n, heads, kv) in enumerate([(1, 32, 8), (7, 5, 1), (33, 3, 3)]):
        for rot in (D, D // 2, D // 4 // 2 * 2):
            c = Case(torch_cuda, kind, n, heads, kv, D, rot, layout, 10 * D + i, norm=i != 1)
            c.run(sampler, label=(n, heads, kv, rot))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", [pz.PZ_ROPE_HALVES, pz.PZ_ROPE_PAIRS])
@pytest.mark.parametrize("D,rot", [(1, 0), (2, 2), (7, 6), (50, 50), (128, 102), (130, 2), (40, 24),
                                   (24, 24), (1000, 998)])
def test_odd_sizes_strides_and_addresses(torch_cuda, sampler, kind, layout, D, rot):
    for off, pad in ((0, 0), (1, 3), (8, 0)):
        c = Case(torch_cuda, kind, 5, 3, 2, D, rot, layout, D + off, pad=pad, off=off)
        c.run(sampler, label=(off, pad))
        c.run(sampler, in_place=True, label=(off, pad, "in place"))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", [pz.PZ_ROPE_HALVES, pz.PZ_ROPE_PAIRS])
def test_in_place_and_many_tokens(torch_cuda, sampler, kind, layout):
    """More tokens than waves fit the device, so that waves take several heads."""
    c = Case(torch_cuda, kind, 3001, 20, 5, 128, 128, layout, 3)
    a = c.run(sampler)
    b = c.run(sampler, in_place=True)
    for x, y, m in zip(a, b, (20, 5)):
        assert torch_cuda.equal(x[:, :m * 128], y[:, :m * 128])


@pytest.mark.parametrize("layout", [pz.PZ_ROPE_HALVES, pz.PZ_ROPE_PAIRS])
def test_far_positions_amplitude_and_scaled_frequencies(torch_cuda, sampler, layout):
    for kind in TYPES:
        c = Case(torch_cuda, kind, 64, 4, 2, 128, 64, layout, 5, far=2 ** 31 - 1, amp=1.25)
        c.pos[:6] = [0, 1, -1, 2 ** 31 - 1, -(2 ** 31), 1 << 20]
        c.freq[:8] = [1.0, 0.5, 3.14159274, 1.57079637, 0.785398185, 0.0, -1.0, 6.28318548]
        c.run(sampler, label=kind)
        c.amp = -0.5
        c.run(sampler, label=kind)


def test_queries_or_keys_alone(torch_cuda, sampler):
    torch = torch_cuda
    for heads, kv in ((4, 0), (0, 3)):
        c = Case(torch, "bf16", 9, heads, kv, 64, 64, 0, 6)
        c.run(sampler, label=(heads, kv))
        x, pos = c.x.cuda(), torch.from_numpy(c.pos).cuda()
        out = torch.zeros_like(x)
        args = [x, c.ld] if heads else [None, 0]
        more = [None, 0] if heads else [x, c.ld]
        oargs = [out, c.ld] if heads else [None, 0]
        omore = [None, 0] if heads else [out, c.ld]
        sampler.qk_norm_rope(c.how(), *args, *more, *oargs, *omore, 9, pos)
        sampler.sync()
        c.check(out, out, (heads, kv))
    # a norm for the queries only
    c = Case(torch, "fp16", 9, 4, 2, 64, 32, 1, 7)
    c.w[1] = None
    c.run(sampler)
    c.w = [None, np.ones(64, np.float32)]
    c.run(sampler)


@pytest.mark.parametrize("layout", [pz.PZ_ROPE_HALVES, pz.PZ_ROPE_PAIRS])
@pytest.mark.parametrize("D", [64, 66])
def test_what_is_not_finite_stays_where_it_is(torch_cuda, sampler, layout, D):
    """Without a norm: NaN and infinities reach their pair and nothing else."""
    torch = torch_cuda
    c = Case(torch, "bf16", 4, 3, 2, D, 20, layout, 8, norm=False)
    clean = [t.clone() for t in c.run(sampler)]
    c.x[1, D + 25] = float("nan")       # not rotated
    c.x[2, 2 * D + 20] = float("inf")   # the first that is not rotated
    c.x[3, 3] = float("nan")            # rotated
    c.x[0, 3 * D + 19] = float("-inf")  # a key's, rotated (and the last one)
    q, k = c.run(sampler)
    pair = {pz.PZ_ROPE_HALVES: (3, 13), pz.PZ_ROPE_PAIRS: (2, 3)}[layout]
    kpair = {pz.PZ_ROPE_HALVES: (9, 19), pz.PZ_ROPE_PAIRS: (18, 19)}[layout]
    for got, was, odd in ((q, clean[0], [(1, D + 25), (2, 2 * D + 20), (3, pair[0]), (3, pair[1])]),
                          (k, clean[1], [(0, kpair[0]), (0, kpair[1])])):
        same = torch.ones_like(got, dtype=torch.bool)
        for r, i in odd:
            same[r, i] = False
            assert not torch.isfinite(got[r, i])
        assert torch.equal(got[same], was[same])


def test_zeros_and_large_rows(torch_cuda, sampler):
    """A head of zeros stays zero (eps > 0); squares near fp32's largest still sum."""
    c = Case(torch_cuda, "fp32", 3, 2, 1, 128, 128, 0, 9, sigma=1e18)
    c.x[1, :128] = 0.0
    q, _ = c.run(sampler)
    assert (q[1, :128] == 0).all()
    Case(torch_cuda, "bf16", 3, 2, 1, 128, 128, 0, 9, sigma=1e-12).run(sampler)


def test_replayed(torch_cuda, sampler):
    """Captured, then replayed on new rows and positions, eager calls between."""
    torch = torch_cuda
    c = Case(torch, "bf16", 50, 8, 2, 128, 128, 0, 10)
    how, x = c.how(), c.x.cuda()
    pos = torch.from_numpy(c.pos).cuda()
    q, k = (torch.zeros((50, m * 128), dtype=torch.bfloat16, device="cuda") for m in (8, 2))
    eq, ek = torch.zeros_like(q), torch.zeros_like(k)

    def call(a, b):
        p = x.data_ptr()
        assert sampler.lib.pz_qk_norm_rope(sampler.h, pz.ctypes.byref(how), p, c.ld, p + 2048, c.ld,
                                           a.data_ptr(), 1024, b.data_ptr(), 256, 50,
                                           pos.data_ptr()) == 0
    call(q, k)
    sampler.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(sampler.stream)):
        call(q, k)
    for i in range(4):
        x.normal_()
        pos += 3
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        call(eq, ek)
        sampler.sync()
        assert torch.equal(q, eq) and torch.equal(k, ek), i
        c.x, c.pos = x.cpu(), pos.cpu().numpy()
        c.check(q, k, i)


def test_refusals(torch_cuda, sampler):
    torch = torch_cuda
    c = Case(torch, "bf16", 2, 2, 1, 64, 64, 0, 11)
    x = c.x.cuda()
    pos = torch.from_numpy(c.pos).cuda()
    out = torch.zeros_like(x)
    c.rot = 65
    with pytest.raises(pz.PzError) as e:
        sampler.qk_norm_rope(c.how(), x, c.ld, x, c.ld, out, c.ld, out, c.ld, 2, pos)
    assert e.value.code == pz.PZ_EINVAL and "rot_dim" in str(e.value)
    c.rot = 64
    sampler.qk_norm_rope(c.how(), x, c.ld, x, c.ld, out, c.ld, out, c.ld, 0, pos)  # no tokens
    sampler.sync()
    assert (out == 0).all()
