"""Attention over packed prompts with keys that are infinite: their scores are, and the softmax of those is the output.  A score of +inf, or nothing but
-inf, makes a row NaN; -inf beside numbers weighs nothing.
"""
import math

import pytest
import torch

from conftest import pkg
from test_gpu_prompt import DEV, U, _randn, name
from test_gpu_states import _check, _reference

pytestmark = pytest.mark.gpu

# in the pipelined kernel with one, two and four waves to a row's keys, and in the other with one and two
LENS = [([900, 130], 4, 1, 64), ([1000, 900], 10, 10, 64), ([1000] * 4, 16, 16, 128), ([1000, 300, 1], 4, 2, 128), ([290, 70, 310, 1], 16, 16, 128), ([77, 40], 3, 3, 96), ([1000, 300], 2, 2, 192),
        ([1000, 300], 2, 2, 256)]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=name)
@pytest.mark.parametrize("lens,h,hk,d", LENS, ids=str)
def test_the_first_keys_of_prompts(lens, h, hk, d, dtype, sign):
    """The first key of every prompt is infinite in one channel: its first row sees nothing else."""
    pr = pkg("prompt")
    T, at = sum(lens), [sum(lens[:i]) for i in range(len(lens) + 1)]
    qkv = _randn(11, T, h + 2 * hk, d, size=1.3).to(dtype)
    q, k, v = qkv[:, :h].clone(), qkv[:, h:h + hk].clone(), qkv[:, h + hk:]
    q[..., 3] = torch.where(q[..., 3] == 0, torch.ones_like(q[..., 3]), q[..., 3])      # (0 times infinity)
    safe = k.clone()
    k[at[:-1], :, 3] = sign * math.inf
    o = pr.attn(q, k, v, torch.tensor(at, dtype=torch.int32, device=DEV), d ** -0.5)
    for b, e in zip(at[:-1], at[1:]):
        for j in sorted({0, h - 1}):
            x, y, z, got = q[b:e, j], safe[b:e, j * hk // h], v[b:e, j * hk // h], o[b:e, j]
            up = sign * x[:, 3] > 0
            nan = up.clone()
            nan[0] = True
            assert got[nan].isnan().all(), (b, j, got[nan].isnan().float().mean().item())
            keep = torch.ones(e - b, e - b, dtype=torch.bool, device=DEV).tril()
            keep[1:, 0] = False
            want, bound = _reference(x, y, z, d ** -0.5, keep, torch.zeros(e - b, dtype=torch.float64, device=DEV), U[dtype], U[dtype], z.double().abs().max() if dtype == torch.float16 else None)
            if not nan.all():
                _check(got[~nan], want[~nan], bound[~nan], "prompt at %d, head %d" % (b, j))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=name)
@pytest.mark.parametrize("lens,h,hk,d", [([1000] * 4, 16, 16, 56), ([900, 130], 4, 1, 40), ([1000, 900], 10, 10, 24), ([1000] * 4, 16, 16, 96), ([1000, 300, 1], 4, 2, 120), ([1000] * 4, 16, 16, 120),
                                         ([290, 70, 310, 1], 16, 16, 104), ([1000, 300], 2, 2, 160), ([1000, 300], 2, 2, 248)], ids=str)
def test_the_last_channel_of_head_dims_that_are_padded(lens, h, hk, d, dtype, sign):
    """A key that is infinite in a head's last channel: the padding behind it is none of its channels."""
    pr = pkg("prompt")
    T, at = sum(lens), [sum(lens[:i]) for i in range(len(lens) + 1)]
    qkv = _randn(13, T, h + 2 * hk, d, size=1.3).to(dtype)
    q, k, v = qkv[:, :h].clone(), qkv[:, h:h + hk].clone(), qkv[:, h + hk:]
    q[..., -1] = torch.where(q[..., -1] == 0, torch.ones_like(q[..., -1]), q[..., -1])
    starts = torch.tensor(at, dtype=torch.int32, device=DEV)
    holes = [b + n for b, e in zip(at[:-1], at[1:]) for n in (5, 70) if b + n < e]
    k[holes, :, -1] = sign * math.inf
    out = pr.attn(q, k, v, starts, d ** -0.5)
    for b, e in zip(at[:-1], at[1:]):
        row = torch.arange(e - b, device=DEV)
        seen = (row >= 5) if e - b > 5 else torch.zeros(e - b, dtype=torch.bool, device=DEV)
        for j in sorted({0, h - 1}):
            up = seen & (sign * q[b:e, j, -1] > 0)
            assert out[b:e, j][up].isnan().all() and not out[b:e, j][~up].isnan().any(), (b, j)


@pytest.mark.parametrize("T,h,d", [(300, 2, 128), (1000, 16, 128), (77, 2, 64), (300, 2, 192)])
def test_every_key_of_a_row_at_minus_infinity(T, h, d):
    """All keys infinite against the queries' sign, and finite ones whose products leave fp32 downwards."""
    pr = pkg("prompt")
    starts = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    v = _randn(12, T, h, d).bfloat16()
    q, k = torch.ones_like(v), torch.full_like(v, -math.inf)
    for causal in (True, False):
        assert pr.attn(q, k, v, starts, 0.1, causal).isnan().all()
        assert pr.attn(q * 1e20, torch.full_like(v, -1e20), v, starts, 0.1, causal).isnan().all()
