"""Logit rules of long lists (pz_rules_batch): bias lists far past what a hash
table is made for, and rows, histories and masks that lie past 2^31 elements."""
import numpy as np
import pytest

import pzsample as pz
from conftest import to_dev
from test_gpu_rules import F, PENS, logits, pack, run, same, want

pytestmark = pytest.mark.gpu


def adding_up(x, ids, bias):
    """x[ids[e]] += bias[e] in the list's order, in fp32."""
    y = x.copy()
    order = np.argsort(ids, kind="stable")
    i, b = ids[order], bias[order]
    first = np.concatenate([[True], i[1:] != i[:-1]])
    nth = np.arange(len(i)) - np.maximum.accumulate(np.where(first, np.arange(len(i)), 0))
    for k in range(int(nth.max()) + 1):
        at = nth == k
        y[i[at]] = y[i[at]] + b[at]
    return y


@pytest.mark.parametrize("V,n,ids", [(128256, 1 << 18, 100000), (1000, 1 << 16, 1000),
                                     (40000, 6000, 3)])
def test_bias_lists_are_read_once(torch_cuda, V, n, ids):
    """Every id many times over: in order, and in a time that grows with the list,
    not with the list times its ids (150 ms at the first size)."""
    torch = torch_cuda
    rng = np.random.default_rng(n)
    x = logits(1, V, n)
    bid = rng.integers(0, ids, n, dtype=np.int32)
    bias = (logits(1, n, n + 1)[0] * np.logspace(-4, 4, n)).astype(F)
    exp = adding_up(x[0], bid, bias)
    d_x = to_dev(torch, x)
    out = torch.empty_like(d_x)
    rules = pz.logit_rules(d_bias_ids=to_dev(torch, bid), d_bias=to_dev(torch, bias), n_bias=n)
    ms = []
    with pz.Sampler(1, 16) as s:
        st = torch.cuda.ExternalStream(s.stream)
        for i in range(3):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record(st)
            s.rules(d_x, out, 1, V, V, V, rules)
            b.record(st)
            s.sync()
            ms.append(a.elapsed_time(b))
            same(out.cpu().numpy(), exp[None], i)
    assert min(ms) < 30.0, ms


def test_long_lists_of_repeated_ids_with_every_rule(torch_cuda):
    """Masked, unmasked, penalised and only biased ids, each named once, twice
    and often, in lists past a hash table's."""
    V, H, n = 9000, 5000, 700
    rng = np.random.default_rng(5)
    x = logits(3, V, 5)
    hist = rng.integers(-1, V, (3, H), dtype=np.int32)
    bid = rng.integers(-2, 500, (3, n), dtype=np.int32)
    bid[1] = rng.integers(0, V, n)
    bid[2, :600] = 17
    bid[0, :4] = [-2 ** 31, 2 ** 31 - 1, V, V - 1]
    bias = logits(3, n, 6)
    on = rng.random((3, V)) < 0.6
    for mask in (None, on):
        for inplace in (True, False):
            run(torch_cuda, x, V, PENS[3], None, hist, None, bid, bias, mask, None, inplace)


@pytest.mark.parametrize("H", [70, 1 << 30])
@pytest.mark.parametrize("inplace", [True, False])
def test_rows_past_32_bits(torch_cuda, H, inplace):
    """Three rows 2^30 elements apart, of logits, masks and (the longer ones)
    histories: the last lie past 2^31 elements."""
    torch = torch_cuda
    V, far = 4100, 1 << 30
    rng = np.random.default_rng(9)
    x = logits(3, V, 9)
    hist = rng.integers(-1, V, (3, 70), dtype=np.int32)
    lens = np.array([70, 40, 69], np.int32)
    bid = rng.integers(-1, V, (3, 9), dtype=np.int32)
    bias = logits(3, 9, 10)
    on = rng.random((3, V)) < 0.7

    def spread(a, ld):
        pool = torch.empty(2 * ld + a.shape[1], dtype=torch.from_numpy(a).dtype, device="cuda")
        pool.as_strided(a.shape, (ld, 1)).copy_(torch.from_numpy(a))
        return pool

    words = pack(on).view(np.int32)
    d_x, d_mask = spread(x, far), spread(words, far)
    d_hist = spread(hist, H) if H > 70 else to_dev(torch, hist)
    d_out = d_x if inplace else spread(np.zeros_like(x), far + 3)
    d_allowed = torch.empty(3, dtype=torch.int32, device="cuda")
    rules = pz.logit_rules(*PENS[3], d_hist=d_hist, H=H, d_hist_len=to_dev(torch, lens),
                           d_bias_ids=to_dev(torch, bid), d_bias=to_dev(torch, bias), n_bias=9,
                           d_mask=d_mask, ld_mask=far, n_masks=3, d_allowed=d_allowed)
    ld_out = far if inplace else far + 3
    with pz.Sampler(1, 16) as s:
        s.rules(d_x, d_out, 3, V, far, ld_out, rules)
        s.sync()
    exp, allowed = want(x, V, [PENS[3]] * 3, hist, lens, bid, bias, on)
    same(d_out.as_strided((3, V), (ld_out, 1)).cpu().numpy(), exp, (H, inplace))
    assert (d_allowed.cpu().numpy() == allowed).all()
