"""Selections where many candidates reach the first bound: groups whose beams' scores lie far
apart, rows whose masked logits are low but finite, equal rows.  Results as in
test_gpu_beam.py; and their time stays near that of other values, since a search's scores
spread and masks are part of it."""
import time

import numpy as np
import pytest

import pzsample as pz
from test_gpu_beam import Selection

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampler(torch_cuda):
    with pz.Sampler(1, 16) as s:
        yield s


def spread(torch, G, W, V, seed, by):
    c = Selection(torch, G, W, V, seed)
    c.score = (np.random.default_rng(seed).standard_normal((G, W)) * by - 30).astype(np.float32)
    return c


def masked(torch, G, W, V, seed, keep, low):
    c = Selection(torch, G, W, V, seed)
    c.x[np.random.default_rng(seed).random(c.x.shape) >= keep] = low
    return c


@pytest.mark.parametrize("by", [2.0, 6.0, 40.0])
@pytest.mark.parametrize("G,W,V,K", [(1, 16, 128256, 128), (2, 64, 20000, 128), (3, 32, 40000, 64),
                                     (40, 16, 9000, 33), (1, 2, 300000, 128)])
def test_scores_far_apart(torch_cuda, sampler, G, W, V, K, by):
    c = spread(torch_cuda, G, W, V, V + W, by)
    c.run(sampler, K, eos=[3, 77], label=by)
    # some have ended, one of them far above the others
    c.done = (np.random.default_rng(5).random((G, W)) < 0.3).astype(np.uint8)
    c.done[0, W - 1], c.score[0, W - 1] = 1, -1.0
    c.score[0, 0] = -np.inf
    c.pad_id = 9
    c.run(sampler, K, eos=[3, 77], label=(by, "ended"))


@pytest.mark.parametrize("low", [-1e9, np.finfo(np.float32).min])
@pytest.mark.parametrize("G,W,V,K", [(1, 4, 20000, 8), (2, 4, 20000, 128), (8, 8, 40000, 16),
                                     (160, 4, 9000, 64), (1, 64, 9000, 128)])
def test_masked_ids_of_low_logits(torch_cuda, sampler, G, W, V, K, low):
    for keep in (0.01, 2e-4):
        masked(torch_cuda, G, W, V, V + K, keep, low).run(sampler, K, label=keep)


def test_equal_rows_of_many_beams(torch_cuda, sampler):
    """More candidates of one score than are counted against each other: by beam, then id."""
    for G, W, V, K in ((2, 64, 9000, 128), (1, 64, 3000, 7), (1, 16, 70000, 64)):
        c = Selection(torch_cuda, G, W, V, 11)
        c.x[:] = np.round(c.x[:, :1])
        c.score[:] = -2.5
        c.run(sampler, K, label=(W, V, "rounded"))
        c.x[:] = 0.5
        c.score[:, W // 2:] = -2.0
        c.run(sampler, K, label=(W, V, "one value"))
        c.done = np.zeros((G, W), np.uint8)
        c.done[:, 1::2] = 1
        c.score[:] = np.float32(-np.log(V))
        c.run(sampler, K, label=(W, V, "ended"))


def took(torch, s, c, K):
    """Seconds of a call, the fastest of some runs of ten."""
    x, score, _ = c.device()
    out = [torch.zeros((c.G, K), dtype=d, device="cuda")
           for d in (torch.int32, torch.int32, torch.float32)]
    torch.cuda.synchronize()
    args = [x.data_ptr(), c.ld, c.G, c.W, c.V, score.data_ptr(), None, 0, K,
            *(t.data_ptr() for t in out), None]
    best = 1e9
    for _ in range(8):
        s.sync()
        t0 = time.perf_counter()
        for _ in range(10):
            assert s.lib.pz_beam_select(s.h, *args) == 0
        s.sync()
        best = min(best, (time.perf_counter() - t0) / 10)
    return best


def test_times(torch_cuda, sampler):
    """11 and 46 us as a rule; the masked rows took 365, the scores far apart 9700, where too
    many were counted against each other or one by one looked at every candidate.  (16 and 85
    now: a fourth of the bound at most.)"""
    torch = torch_cuda
    rule = took(torch, sampler, Selection(torch, 1, 4, 128256, 1), 8)
    assert took(torch, sampler, masked(torch, 1, 4, 128256, 1, 0.001, -1e9), 8) < 8 * rule
    rule = took(torch, sampler, Selection(torch, 1, 16, 128256, 1), 128)
    assert took(torch, sampler, spread(torch, 1, 16, 128256, 1, 6.0), 128) < 8 * rule
