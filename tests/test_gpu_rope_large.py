"""The rotation of as many tokens as a call takes."""
import numpy as np
import pytest

import pzsample as pz
import test_gpu_rope as ro

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [2 ** 26 - 4, 2 ** 26 - 1])  # (one kernel's most, the other's)
def test_the_most_tokens(torch_cuda, n):
    """One head of 8 each, in rows that repeat: every repetition as the first, and the first
    within test_gpu_rope.py's bound."""
    torch = torch_cuda
    D, some = 8, 4093
    g = np.random.default_rng(n & 7)
    rows = torch.from_numpy(g.standard_normal((some, D)).astype(np.float32)).to(torch.bfloat16)
    pos = torch.from_numpy(g.integers(0, 5000, some).astype(np.int32))
    freq = (10000.0 ** (-np.arange(D // 2) / (D / 2))).astype(np.float32)
    w = (1 + 0.1 * g.standard_normal(D)).astype(np.float32)
    times = n // some + 1
    x = rows.cuda().repeat(times, 1)[:n].contiguous()
    p = pos.cuda().repeat(times)[:n].contiguous()
    rope = pz.qk_rope(type=pz.PZ_BF16, n_heads=1, n_kv_heads=0, head_dim=D,
                      d_q_norm=torch.from_numpy(w).cuda(), d_k_norm=None, eps=1e-6, rot_dim=D,
                      layout=pz.PZ_ROPE_HALVES, d_freq=torch.from_numpy(freq).cuda())
    with pz.Sampler(1, 16) as s:
        s.qk_norm_rope(rope, x, D, None, 0, x, D, None, 0, n, p)
        s.sync()
        with pytest.raises(pz.PzError) as e:
            s.qk_norm_rope(rope, x, D, None, 0, x, D, None, 0, 2 ** 26, p)
        assert e.value.code == pz.PZ_ERANGE
    first = x[:some]
    whole = x[:n // some * some].reshape(-1, some, D)
    assert (whole == first).all() and torch.equal(x[len(whole) * some:], first[:n % some])
    want, tol = ro.reference(rows.double().numpy(), 1, D, D, pz.PZ_ROPE_HALVES, freq, pos.numpy(),
                             w, 1e-6, 1.0)
    h = 2.0 ** -8
    assert (np.abs(first.cpu().double().numpy() - want) <= h * np.abs(want) + tol * (1 + h)).all()
