"""Attention over packed prompts: a row's denominator is the sum of the probabilities that multiply its values, as they are rounded.  What all of a
row's probabilities lose alike then leaves the output alone, which counts where few keys have most of the weight.
"""
import ctypes

import pytest
import torch

from conftest import pkg
from test_gpu_prompt import DEV, _randn, name

pytestmark = pytest.mark.gpu

# (rows of a workgroup, waves to a row's keys): head dims to 64 and to 128, prompts of up to 1000 tokens
FORMS = [((64, 4), [900, 130], 4, 1, 64), ((128, 2), [1000, 900], 10, 10, 64), ((256, 1), [1000] * 4, 16, 16, 64), ((256, 1), [1000] * 4, 16, 16, 56), ((128, 2), [1000, 300, 1], 4, 2, 128),
         ((256, 1), [1000] * 4, 16, 16, 128), ((128, 2), [700, 1000], 6, 3, 80), ((128, 0), [290, 70, 310] * 6, 16, 16, 128), ((128, 2), [1000, 300], 2, 2, 192), ((64, 2), [1000, 300], 2, 2, 256)]


def _case(form, lens, h, hk, d, dtype, ones):
    ffi, out = pkg("ffi"), (ctypes.c_int32 * 2)()
    T = sum(lens)
    ffi.k("gpu_internal_prompt_attn_form", T, len(lens), h, hk, d, ctypes.cast(out, ctypes.c_void_p))
    assert tuple(out) == form
    q, k = (_randn(i, T, n, d, size=6 ** 0.5).to(dtype) for i, n in ((1, h), (2, hk)))      # scores of deviation 6
    v = torch.ones_like(k) if ones else _randn(3, T, hk, d).to(dtype)
    starts = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    return q, k, v, starts


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=name)
@pytest.mark.parametrize("form,lens,h,hk,d", FORMS, ids=str)
def test_values_of_one_give_one(form, lens, h, hk, d, dtype):
    """Numerator and denominator are the same numbers, added in two orders: off by 1000 2^-23 (the products) and 300 2^-24 (four at a time) of themselves at most, 1.4e-4,
    where the next number below one is half a step of 2^-12 = 2.4e-4 (f16) or 2^-9 away."""
    q, k, v, starts = _case(form, lens, h, hk, d, dtype, True)
    for causal in (True, False):
        o = pkg("prompt").attn(q, k, v, starts, d ** -0.5, causal)
        far = (o.float() - 1).abs()
        assert far.max().item() == 0, (causal, far.max().item(), (far > 0).float().mean().item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=name)
@pytest.mark.parametrize("form,lens,h,hk,d", [f for f in FORMS if f[0][1] and f[4] <= 128], ids=str)
def test_the_pipelined_loop_is_as_exact_as_the_other(form, lens, h, hk, d, dtype):
    """Rows at odd addresses go through the loop that the pipelined one leaves the edges to.  Against 64 bits both are off by the same roundings of other
    numbers: the mean square over 2000 and more rows agrees to a few parts in a hundred."""
    q, k, v, starts = _case(form, lens, h, hk, d, dtype, False)
    odd = [torch.zeros(t.numel() + 1, dtype=dtype, device=DEV)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    pr = pkg("prompt")
    got, other = pr.attn(q, k, v, starts, d ** -0.5, False).double(), pr.attn(*odd, starts, d ** -0.5, False).double()
    off = [0.0, 0.0]
    at = starts.tolist()
    for b, e in zip(at[:-1], at[1:]):
        for j in range(h):
            x, y, z = q[b:e, j].double(), k[b:e, j * hk // h].double(), v[b:e, j * hk // h].double()
            s = (x @ y.t().contiguous()) * d ** -0.5
            want = torch.softmax(s, -1) @ z.contiguous()
            for i, o in enumerate((got, other)):
                off[i] += (o[b:e, j] - want).square().sum().item()
    assert off[0] <= 1.05 ** 2 * off[1], (off[0] / off[1]) ** 0.5
