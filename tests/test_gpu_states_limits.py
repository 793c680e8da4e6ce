"""Attention to stored states at the ends of what its calls take, against the formulas in 64 bits and the bounds of test_gpu_states.py."""
import pytest
import torch

from conftest import pkg
from test_gpu_states import DEV, _attn_check, _cross_check, _filled, _gen, _rows

pytestmark = pytest.mark.gpu


def test_mixed_batches_with_more_rows_than_a_join_takes():
    """300 sequences of which one has a piece of a prompt, counted as 2^26 rows: every sequence's are those of the formula."""
    kv = pkg("kvcache")
    new = [90] + [1 + i % 3 for i in range(299)]
    lens = [m + i % 40 for i, m in enumerate(new)]
    cache, table, model = _filled(lens, 8, 16, 16, 91)
    q = torch.randn(sum(new), 32, 16, device=DEV, generator=_gen(92)).bfloat16()
    rows = _rows(kv, new, lens, table)._replace(most=8192)      # a bound that a program knows beforehand
    assert 300 * 8 * 8192 * 4 > 2 ** 26
    for causal in (True, False):
        o = kv.attn(q, cache, rows, 0.25, causal)
        assert o.shape == q.shape
        _attn_check(o, q, model, new, lens, 0.25, causal)


def test_cross_attn_with_more_rows_than_a_join_takes():
    """4 x 524288 rows of 32 heads, queries alike: every row is the one that a short call gives."""
    ql = pkg("qlinear")
    g = _gen(93)
    one = torch.randn(4, 1, 32, 8, device=DEV, generator=g).bfloat16()
    k, v = (torch.randn(4, 20, 32, 8, device=DEV, generator=g).bfloat16() for _ in range(2))
    o = ql.cross_attn(one.expand(-1, 524288, -1, -1), k, v, 0.3)
    _cross_check(o[:, :1], one, k, v, 0.3)
    assert bool((o == o[:, :1]).all())
