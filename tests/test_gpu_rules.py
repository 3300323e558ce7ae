"""Logit rules (pz_rules_batch): penalties, biases and masks, bit for bit
against fp32 numpy operations in the header's order, and the penalties against
the samplers' own (the oracle's)."""
import ctypes

import numpy as np
import pytest

import pz_oracle as po
import pzsample as pz
from conftest import to_dev

pytestmark = pytest.mark.gpu

F = np.float32
SENTINEL = F(-12345.0)


def pack(on):
    """[n, V] truth values -> [n, words] uint32 masks."""
    n, V = on.shape
    pad = np.zeros((n, (V + 31) // 32 * 32), np.uint8)
    pad[:, :V] = on
    return np.packbits(pad, axis=1, bitorder="little").view(np.uint32)


def want(x, V, pen, hist=None, hist_len=None, bias_ids=None, bias=None, on=None, mask_row=None):
    """The rules in fp32, row by row; pen: (rep, presence, frequency) per row."""
    out = x[:, :V].copy()
    allowed = np.full(len(x), V, np.int32)
    with np.errstate(all="ignore"):
        for b in range(len(x)):
            rep, pres, freq = (F(v) for v in pen[b])
            if hist is not None:
                h = hist[b] if hist_len is None else hist[b][:max(hist_len[b], 0)]
                ids, c = np.unique(h[(h >= 0) & (h < V)], return_counts=True)
                y = out[b, ids]
                y = np.where(y > 0, y / rep, y * rep)
                out[b, ids] = y - (c.astype(F) * freq + pres)
            if bias_ids is not None:
                for e, i in enumerate(bias_ids[b]):
                    if 0 <= i < V:
                        out[b, i] = out[b, i] + bias[b, e]
            if on is not None:
                r = b if mask_row is None else mask_row[b]
                if 0 <= r < len(on):
                    out[b, ~on[r]] = -np.inf
                    allowed[b] = on[r].sum()
    return out, allowed


def same(got, exp, label):
    g, e = got.view(np.uint32), exp.view(np.uint32)
    ok = (g == e) | (np.isnan(got) & np.isnan(exp))
    assert ok.all(), (label, np.argwhere(~ok)[:4], got[~ok][:4], exp[~ok][:4])


def run(torch, x, V, pen=(1.0, 0.0, 0.0), per_row=None, hist=None, hist_len=None, bias_ids=None,
        bias=None, on=None, mask_row=None, inplace=True, ld_mask=None, offset=0, label=""):
    B, ld = x.shape
    flat = np.full(B * ld + offset, SENTINEL, F)
    flat[offset:] = x.ravel()
    d_flat = to_dev(torch, flat)
    d_x = d_flat[offset:]
    d_out = d_x if inplace else torch.full((B, ld), float(SENTINEL), device="cuda")
    kw, keep = {}, {}

    def put(name, a):
        if a is not None:
            keep[name] = to_dev(torch, np.ascontiguousarray(a))
            kw[name] = keep[name]

    put("d_penalties", None if per_row is None else np.asarray(per_row, F))
    put("d_hist", hist)
    put("d_hist_len", hist_len)
    put("d_bias_ids", bias_ids)
    put("d_bias", bias)
    if on is not None:
        words = pack(on)
        if ld_mask:
            wide = np.full((len(on), ld_mask), 0xFFFFFFFF, np.uint32)
            wide[:, :words.shape[1]] = words
            words = wide
        if V % 32:  # bits past V count for nothing
            words[:, (V - 1) // 32] |= np.uint32((0xFFFFFFFF << (V % 32)) & 0xFFFFFFFF)
        put("d_mask", words.view(np.int32))
        kw.update(n_masks=len(on), ld_mask=words.shape[1])
        put("d_mask_row", mask_row)
    d_allowed = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    rules = pz.logit_rules(*pen, H=0 if hist is None else hist.shape[1],
                           n_bias=0 if bias_ids is None else bias_ids.shape[1],
                           d_allowed=d_allowed, **kw)
    with pz.Sampler(1, 16) as s:
        s.rules(d_x, d_out, B, V, ld, ld, rules)
        s.sync()
    got = d_out.cpu().numpy().reshape(B, ld)
    exp, allowed = want(x, V, [pen] * B if per_row is None else per_row, hist, hist_len,
                        bias_ids, bias, on, mask_row)
    same(got[:, :V], exp, label)
    assert (got[:, V:] == (x[:, V:] if inplace else SENTINEL)).all(), (label, "past the rows")
    assert (d_allowed.cpu().numpy() == allowed).all(), label
    if not inplace:
        same(d_x.cpu().numpy().reshape(B, ld), x, (label, "input"))


def logits(B, ld, seed):
    return (np.random.default_rng(seed).standard_normal((B, ld)) * 3).astype(F)


PENS = [(1.0, 0.0, 0.0), (1.3, 0.0, 0.0), (1.0, 0.5, 0.0), (1.1, -0.25, 0.3)]


@pytest.mark.parametrize("V,pad", [(1, 0), (5, 3), (31, 0), (33, 0), (1000, 24), (8192, 0),
                                   (8193, 0), (50257, 0), (128256, 0)])
@pytest.mark.parametrize("inplace", [True, False])
def test_every_rule(torch_cuda, V, pad, inplace):
    B = 5
    rng = np.random.default_rng(V)
    x = logits(B, V + pad, V + 1)
    hist = rng.integers(-2, V + 2, (B, 70), dtype=np.int32)
    lens = np.array([0, 70, 35, -3, 999], np.int32)
    bias_ids = rng.integers(-1, V + 1, (B, 9), dtype=np.int32)
    bias = logits(B, 9, V + 2)
    on = rng.random((3, V)) < np.array([[0.5], [0.01], [0.98]])
    rows = np.array([2, -1, 0, 1, 3], np.int32)  # (-1 and 3: no mask)
    for pen in PENS:
        run(torch_cuda, x, V, pen, None, hist, lens, bias_ids, bias, on, rows, inplace,
            label=(V, pen))
    run(torch_cuda, x, V, (1.0, 0.0, 0.0), [PENS[b % 4] for b in range(B)], hist, None, None,
        None, None, None, inplace, label="penalties of each row")
    run(torch_cuda, x, V, PENS[3], inplace=inplace, label="no rule")


@pytest.mark.parametrize("H", [1, 3, 4, 1023, 2048, 2049, 20001])
@pytest.mark.parametrize("V", [700, 20000])
def test_long_histories(torch_cuda, H, V):
    rng = np.random.default_rng(H)
    x = logits(3, V, H)
    hist = rng.zipf(1.3, (3, H)).clip(max=V).astype(np.int32) - 1
    lens = np.array([H, H // 2 + 1, 1], np.int32)
    run(torch_cuda, x, V, PENS[3], None, hist, lens, label=H)
    on = rng.random((3, V)) < 0.5
    run(torch_cuda, x, V, PENS[3], None, hist, None, None, None, on, None, False, label=H)


def test_biases_of_one_id_add_up_in_order(torch_cuda):
    V, nb = 300, 2500  # (past what a hash table is made for, too)
    rng = np.random.default_rng(3)
    x = logits(2, V, 4)
    bias = (logits(2, nb, 5) * np.logspace(-6, 6, nb)).astype(F)
    for n in (2, 40, 1000, nb):
        ids = rng.integers(0, max(2, min(V, n // 3)), (2, n), dtype=np.int32)
        for inplace in (True, False):
            run(torch_cuda, x, V, PENS[3], None, ids[:, :n // 2].copy(), None, ids, bias[:, :n],
                None, None, inplace, label=n)


def test_masks_that_leave_nothing_or_everything(torch_cuda):
    for V in (31, 32, 8200):
        on = np.zeros((4, V), bool)
        on[1] = True
        on[2, V - 1] = True
        on[3, 0] = True
        x = logits(4, V, V)
        hist = np.tile(np.arange(8, dtype=np.int32), (4, 1))
        for inplace in (True, False):
            run(torch_cuda, x, V, PENS[3], None, hist, None, None, None, on, None, inplace)
            run(torch_cuda, x, V, on=on, inplace=inplace, ld_mask=(V + 31) // 32 + 3)


def test_special_values(torch_cuda):
    V = 4100
    x = logits(3, V, 9)
    vals = np.array([np.nan, np.inf, -np.inf, -0.0, 0.0, np.finfo(F).max, np.finfo(F).min, 1e-42],
                    F)
    x[:, :64] = np.tile(vals, 8)
    hist = np.tile(np.arange(40, dtype=np.int32), (3, 1))
    bias_ids = np.tile(np.arange(20, 60, dtype=np.int32), (3, 1))
    bias = np.tile(vals, (3, 5))
    on = np.ones((3, V), bool)
    on[:, 3:50:2] = False  # (NaN and infinities in masked places become -infinity)
    for inplace in (True, False):
        run(torch_cuda, x, V, PENS[3], None, hist, None, bias_ids, bias, on, None, inplace)


@pytest.mark.parametrize("offset,V,ld", [(1, 1001, 1001), (2, 4096, 4099), (3, 128256, 128256)])
def test_rows_off_16_bytes(torch_cuda, offset, V, ld):
    rng = np.random.default_rng(offset)
    x = logits(3, ld, offset)
    on = rng.random((3, V)) < 0.7
    hist = rng.integers(0, V, (3, 33), dtype=np.int32)
    for inplace in (True, False):
        run(torch_cuda, x, V, PENS[1], None, hist, None, None, None, on, None, inplace,
            offset=offset)


def test_many_rows(torch_cuda):
    B, V = 3000, 257
    rng = np.random.default_rng(8)
    on = rng.random((B, V)) < 0.4
    run(torch_cuda, logits(B, V, 8), V, PENS[3], None, rng.integers(0, V, (B, 12), dtype=np.int32),
        None, None, None, on)


def test_penalties_are_the_samplers_own(torch_cuda):
    """The rules and then a sampler without penalties give the ids and
    probabilities of the sampler with them (the oracle's)."""
    torch = torch_cuda
    B, V, H = 6, 32000, 64
    x = logits(B, V, 12)
    hist = np.random.default_rng(12).integers(0, V, (B, H), dtype=np.int32)
    hist[:, 10:] = hist[:, :H - 10]
    u = pz.synth_draws(B, 13)
    pen = dict(rep_penalty=1.2, presence_penalty=0.4, frequency_penalty=0.1)
    with pz.Sampler(B, V, max_hist=H) as s:
        for kw in (dict(temperature=0.0), dict(temperature=0.9),
                   dict(temperature=0.8, top_k=30, top_p=0.9), dict(temperature=0.7, top_p=0.9)):
            ids, p, _, _ = po.sample_batch(x, [po.params(**kw, **pen)], u=u, hist=hist)
            d_x, d_h = to_dev(torch, x), to_dev(torch, hist)
            s.rules(d_x, d_x, B, V, V, V, pz.logit_rules(**pen, d_hist=d_h, H=H))
            got, gp = s.sample(d_x, B, V, V, [pz.row_params(**kw)], u=u, want_p=True)
            assert (got == ids).all(), kw
            assert (gp == p).all(), kw


def test_a_constrained_row_is_sampled_inside_its_mask(torch_cuda):
    """Masked rows through every sampling mode: the id is one that the mask
    allows, as the oracle samples the same masked row; a row that allows
    nothing reads 0 in d_allowed."""
    torch = torch_cuda
    B, V = 4, 9001
    x = logits(B, V, 21)
    rng = np.random.default_rng(21)
    on = rng.random((B, V)) < np.array([[0.5], [0.02], [0.001], [0.999]])
    on[2, :] = False
    on[2, 4567] = True
    u = pz.synth_draws(B, 22)
    d_on = to_dev(torch, pack(on).view(np.int32))
    masked = np.where(on, x, F(-np.inf)).astype(F)
    with pz.Sampler(B, V) as s:
        for kw in (dict(temperature=0.0), dict(temperature=0.9),
                   dict(temperature=0.8, top_k=30, top_p=0.9), dict(temperature=0.7, top_p=0.9)):
            d_x = to_dev(torch, x)
            s.rules(d_x, d_x, B, V, V, V, pz.logit_rules(d_mask=d_on, ld_mask=d_on.shape[1],
                                                         n_masks=B))
            got, _ = s.sample(d_x, B, V, V, [pz.row_params(**kw)], u=u)
            ids, _, _, _ = po.sample_batch(masked, [po.params(**kw)], u=u)
            assert (got == ids).all(), kw
            assert on[np.arange(B), got].all(), kw


def test_refused_calls_change_nothing(torch_cuda):
    torch = torch_cuda
    x = to_dev(torch, logits(2, 100, 1))
    before = x.clone()
    with pz.Sampler(1, 16) as s:
        for r in (pz.logit_rules(H=3), pz.logit_rules(n_bias=2), pz.logit_rules(n_masks=2)):
            with pytest.raises(pz.PzError) as e:
                s.rules(x, x, 2, 100, 100, 100, r)
            assert e.value.code == pz.PZ_EINVAL and "needs" in str(e.value)
        rc = s.lib.pz_rules_batch(s.h, x.data_ptr(), 99, x.data_ptr(), 99, 2, 100,
                                  ctypes.byref(pz.logit_rules()))
        assert rc == pz.PZ_EINVAL
        s.sync()
    assert torch.equal(x, before)


def test_captured_and_replayed(torch_cuda):
    """One call captured on the sampler's stream, replayed on new inputs with
    eager work between; every replay against an eager call."""
    torch = torch_cuda
    B, V, H = 3, 5000, 40
    rng = np.random.default_rng(31)
    x0 = [logits(B, V, 40 + i) for i in range(4)]
    d_x = to_dev(torch, x0[0])
    d_h = to_dev(torch, rng.integers(0, V, (B, H), dtype=np.int32))
    on = rng.random((B, V)) < 0.6
    d_on = to_dev(torch, pack(on).view(np.int32))
    rules = pz.logit_rules(1.2, 0.3, 0.1, d_hist=d_h, H=H, d_mask=d_on, ld_mask=d_on.shape[1],
                           n_masks=B)
    with pz.Sampler(1, 16) as s:
        st = torch.cuda.ExternalStream(s.stream)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=st):
            assert s.lib.pz_rules_batch(s.h, d_x.data_ptr(), V, d_x.data_ptr(), V, B, V,
                                        ctypes.byref(rules)) == 0
        for i in range(4):
            d_x.copy_(torch.from_numpy(x0[i]))
            d_h.copy_(torch.from_numpy(rng.integers(0, V, (B, H), dtype=np.int32)))
            d_e = d_x.clone()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            s.rules(d_e, d_e, B, V, V, V, rules)
            s.sync()
            assert torch.equal(d_x, d_e), i
