"""Logit rules of long lists (pz_rules_batch): bias lists far past what a hash
table is made for, and rows, histories and masks that lie past 2^31 elements."""
import numpy as np
import pytest

import pzsample as pz
from conftest import to_dev
from test_gpu_rules import F, PENS, logits, run, same

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
