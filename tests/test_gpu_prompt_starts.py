"""Attention over packed prompts whose `starts` fall: no row belongs to two prompts, whatever the device holds."""
import random

import pytest
import torch

from conftest import pkg
from test_gpu_prompt import DEV, _attn_check, _randn

pytestmark = pytest.mark.gpu


def _falling(seed, n, tokens):
    """Starts that grow, but for some: in the middle, at the ends of 64 prompts, and outside the rows."""
    rng = random.Random(seed)
    s = sorted(rng.randrange(tokens + 1) for _ in range(n + 1))
    for i in [i for i in (1, n // 2, 63, 64, 65, 127, 128, n - 1, n) if i <= n]:
        if rng.random() < 0.6:
            s[i] = rng.choice((0, -7, tokens + 9, rng.randrange(tokens + 1), rng.randrange(tokens + 1)))
    return s


STARTS = [([0, 100, 50, 150], 150), ([0, 1000, 500, 1500], 1500), ([1200, 0, 700], 1200), ([0, 400, 400, 0, 800], 900), ([30, 20, 10, 0], 40), ([0, 2000, 0, 2000, 0, 2000, 0, 2000], 2000),
          *((_falling(s, n, t), t) for s, (n, t) in enumerate([(5, 300), (64, 500), (65, 700), (66, 2000), (129, 1500), (200, 900), (200, 6000)]))]


@pytest.mark.parametrize("h,hk,d", [(4, 2, 64), (2, 2, 128), (2, 1, 88), (2, 1, 192), (2, 2, 256)], ids=str)
@pytest.mark.parametrize("starts,T", STARTS, ids=lambda v: "%d" % len(v) if isinstance(v, list) else str(v))
def test_a_start_below_an_earlier_one_counts_as_that_one(starts, T, h, hk, d):
    pr = pkg("prompt")
    qkv = _randn(7, T, h + 2 * hk, d, size=1.3).bfloat16()
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    at = torch.tensor(starts, dtype=torch.int32, device=DEV)
    grown = at.cummax(0).values.int().clamp(0, T)
    bounds = grown.tolist()
    want = pr.attn(q, k, v, grown, d ** -0.5, out=torch.full((T, h, d), 7.0, dtype=torch.bfloat16, device=DEV))
    _attn_check(want, q, k, v, bounds, d ** -0.5, True)
    assert (want[:bounds[0]] == 7).all() and (want[bounds[-1]:] == 7).all()
    for _ in range(3):
        got = pr.attn(q, k, v, at, d ** -0.5, out=torch.full((T, h, d), 7.0, dtype=torch.bfloat16, device=DEV))
        assert torch.equal(got, want)
