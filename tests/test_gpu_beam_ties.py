"""Selection among beams whose best candidates lie as close as log sum exp is held
(pz_beam_select): the order of their scores is that of the 64-bit definition.

The rows of a group are random and different, so that nothing but their sums of exponentials
decides.  Bound: an exponential is off by at most 2^-43 of itself (test_beam_exp.py), the
factor that joins a row's segments as much, and the sums, of at most 2^5 terms in a thread,
2^8 in a workgroup and 2^8 segments in turns, by fewer than 64 2^-53: lse by 2^-42 + 2^-46,
and by 4 2^-53 of its value (log, the maximum that is added, exp(-m) where exponentials are
taken as they are).  The score takes two more roundings.  Two scores whose difference is more
than twice that are in order.  The reference is in long double (2^-63)."""
import numpy as np
import pytest

import pzsample as pz
from conftest import to_dev

pytestmark = pytest.mark.gpu

W = 3


def rows(rng, G, V, kind):
    """Logits whose largest of each row is its first candidate by 1 at least, and scores with
    which these candidates of a group are `gap` apart; their order, best first."""
    x = (rng.standard_normal((G, W, V)) * 3).astype(np.float32)
    x = np.clip(x, -30, 9)
    at = np.stack([rng.choice(V, 2, replace=False) for _ in range(G * W)]).reshape(G, W, 2)
    if kind == "mixed":  # the largest past 500 in one segment, the others' below it
        at[..., 0] = V - 1 - at[..., 0] % 100
        at[..., 1] = at[..., 1] % 1000
    top, free = at[..., 0], at[..., 1]
    g, w = np.ogrid[:G, :W]
    base = {"near": 0.0, "far": 1000.0, "below": -800.0, "mixed": 486.0}[kind]
    x = (x + np.float32(base)).astype(np.float32)
    peak = np.float32(base + 16.0)
    x[g, w, top] = peak
    # a second logit of each row is set so that lse is the same in every row of a group, as far
    # as it can be in 32 bits
    x[g, w, free] = -np.inf
    with np.errstate(divide="ignore"):
        e = np.exp(x.astype(np.longdouble) - np.longdouble(peak))
    rest = e.sum(2)
    want = rest.max(1, keepdims=True) * np.longdouble(1.02)
    x[g, w, free] = (np.log(want - rest) + np.longdouble(peak)).astype(np.float32)
    lse = np.log(np.exp(x.astype(np.longdouble) - np.longdouble(peak)).sum(2))  # less peak
    # what is left is in the scores, which are small: their last bits are 2^-40 and less
    order = np.argsort(rng.random((G, W)), axis=1)
    rank = np.argsort(order, axis=1)
    gap = np.where(np.arange(G) % 3 == 0, 2.0 ** -36, 2.0 ** -37 if kind != "near" else 2.0 ** -38)
    centre = lse[:, :1]
    score = ((lse - centre) - rank * gap[:, None].astype(np.longdouble)).astype(np.float32)
    total = score.astype(np.longdouble) + (x[g, w, top].astype(np.longdouble)
                                           - (lse + np.longdouble(peak)))
    return x, score, top, order, total


@pytest.mark.parametrize("kind", ["near", "far", "below", "mixed"])
@pytest.mark.parametrize("G,V", [(20, 3000), (60, 20000), (180, 8000)])  # (2, 3 segments, one)
def test_the_order_of_scores_that_lie_close(torch_cuda, kind, G, V):
    torch = torch_cuda
    if kind == "mixed" and V == 8000:
        V = 9000  # (so that it has two)
    rng = np.random.default_rng(V + len(kind))
    x, score, top, order, total = rows(rng, G, V, kind)
    # the cases are what they are made for: in order, by more than twice the bound, and by so
    # little that a sum off by 2^-34 decides otherwise
    best = np.take_along_axis(total, order, 1)
    apart = (best[:, :-1] - best[:, 1:]).min()
    value = np.abs(x[np.isfinite(x)]).max() + 20.0
    assert apart > 2 * (2.0 ** -42 + 2.0 ** -46 + 6 * 2.0 ** -53 * value)
    off = total + 2.0 ** -34 * rng.standard_normal(total.shape)
    assert (np.argsort(-off, axis=1) != order).any(1).mean() > 0.5
    if kind == "mixed":
        assert (x[:, :, :2048].max(2) <= 500).all() and (x.max(2) > 500).all()
    outs = [torch.zeros((G, W), dtype=d, device="cuda")
            for d in (torch.int32, torch.int32, torch.float32)]
    with pz.Sampler(1, 16) as s:
        s.beam_select(to_dev(torch, x.reshape(G * W, V)), V, G, W, V,
                      to_dev(torch, score.reshape(-1)), W, *outs)
        s.sync()
    parent, ids = (t.cpu().numpy() for t in outs[:2])
    assert (parent == order).all(), np.argwhere(parent != order)[:5]
    assert (ids == np.take_along_axis(top, order, 1)).all()
