"""A prompt model's layer without a GPU: refusals of the C ABI and of the Python side, and the tables of rotary positions."""
import math

import pytest
import torch

from conftest import pkg

ffi = pkg("ffi")
P = 1 << 20         # an address that is never followed: every call below is refused, or has nothing to do
INF, NAN = float("inf"), float("nan")


def _rows(dtype=2, pro=0, x=P, resid=0, total=0, w=0, eps=1e-6, q=P, scales=P, stride=4, M=4, K=256):
    return ffi.raw("gpu_fp8_quant_rows", dtype, pro, x, 512, resid, 512, total, 512, 256, w, eps, q, scales, stride, M, K, 0)


@pytest.mark.parametrize("args,code", [({"dtype": 3}, -4), ({"dtype": -1}, -4), ({"pro": 2}, -3), ({"pro": 99}, -3), ({"K": 0}, -1), ({"K": 24}, -1), ({"K": 32768 + 16}, -2), ({"M": -1}, -1),
                                       ({"stride": 3}, -1), ({"resid": P}, -1), ({"total": P}, -1), ({"pro": 3, "resid": P, "total": P}, -1), ({"pro": 1}, -1), ({"pro": 1, "w": P, "eps": -1.0}, -1),
                                       ({"pro": 1, "w": P, "eps": NAN}, -1), ({"pro": 1, "w": P, "eps": INF}, -1), ({"x": 0}, -1), ({"q": 0}, -1), ({"q": P + 4}, -1), ({"scales": 0}, -1), ({"scales": P + 2}, -1),
                                       ({"x": P + 1}, -1), ({"dtype": 0, "x": P + 2}, -1), ({"resid": P + 1, "total": P}, -1), ({"pro": 1, "w": P + 2}, -1), ({"M": 2 ** 31 - 1, "stride": 2 ** 31}, -1),
                                       ({"M": 0}, 0)])
def test_quant_rows_refusals(args, code):
    assert _rows(**args) == code


def _gemm(A=P, W=P, xs=P, stride=8, ws=P, bias=0, D=P, work=P, M=8, N=8, K=256, dt=2):
    return ffi.raw("gpu_fp8_gemm", A, W, xs, stride, ws, bias, D, work, M, N, K, dt, 0)


@pytest.mark.parametrize("args,code", [({"dt": 3}, -4), ({"dt": -1}, -4), ({"M": -1}, -1), ({"N": -1}, -1), ({"K": 0}, -1), ({"K": 8}, -1), ({"K": 40}, -1), ({"stride": 7}, -1), ({"A": 0}, -1), ({"W": 0}, -1),
                                       ({"xs": 0}, -1), ({"ws": 0}, -1), ({"D": 0}, -1), ({"A": P + 8}, -1), ({"W": P + 4}, -1), ({"xs": P + 2}, -1), ({"ws": P + 1}, -1), ({"D": P + 1}, -1),
                                       ({"D": P + 2, "dt": 0}, -1), ({"bias": P + 1}, -1), ({"M": 1 << 31, "stride": 1 << 31}, -1), ({"N": 1 << 31}, -1), ({"M": 1 << 30, "stride": 1 << 30, "N": 1 << 20}, -1),
                                       ({"K": 8192, "work": 0}, -1), ({"K": 8192, "work": P + 8}, -1), ({"M": 0}, 0), ({"N": 0}, 0)])
def test_gemm_refusals(args, code):
    assert _gemm(**args) == code


def _rope(dtype=2, q=P, qo=P, h=2, k=P, ko=P, hk=1, pos=P, freqs=P, rot=64, factor=1.0, qn=0, kn=0, eps=1e-6, T=3, d=64):
    return ffi.raw("gpu_rope", dtype, q, 64, 64, qo, 64, 64, h, k, 64, 64, ko, 64, 64, hk, pos, freqs, rot, 0, factor, qn, kn, eps, T, d, 0)


@pytest.mark.parametrize("args,code", [({"dtype": 3}, -4), ({"T": -1}, -1), ({"h": -1}, -1), ({"hk": -1}, -1), ({"h": 65537}, -1), ({"d": 66}, -1), ({"d": 0}, -1), ({"d": 260}, -1), ({"rot": 0}, -1), ({"rot": 68}, -1),
                                       ({"rot": 6}, -1), ({"factor": INF}, -1), ({"qn": P, "eps": -1.0}, -1), ({"kn": P, "eps": NAN}, -1), ({"kn": P + 2}, -1), ({"q": 0}, -1), ({"qo": 0}, -1), ({"k": 0}, -1),
                                       ({"ko": 0}, -1), ({"pos": 0}, -1), ({"pos": P + 2}, -1), ({"freqs": 0}, -1), ({"freqs": P + 4}, -1), ({"q": P + 1}, -1), ({"dtype": 0, "ko": P + 2}, -1),
                                       ({"T": 0}, 0), ({"h": 0, "hk": 0}, 0)])
def test_rope_refusals(args, code):
    assert _rope(**args) == code


def _attn(dtype=2, q=P, k=P, v=P, o=P, starts=P, n=2, T=5, h=4, hk=2, d=64, scale=1.0):
    return ffi.raw("gpu_prompt_attn", dtype, q, 256, 64, k, 128, 64, v, 128, 64, o, 256, 64, starts, n, T, h, hk, d, scale, 1, 0)


@pytest.mark.parametrize("args,code", [({"dtype": 0}, -4), ({"dtype": 3}, -4), ({"n": -1}, -1), ({"T": -1}, -1), ({"T": 2 ** 30 + 1}, -1), ({"h": 0}, -1), ({"hk": 0}, -1), ({"h": 3}, -1), ({"d": 0}, -1), ({"d": 12}, -1),
                                       ({"d": 264}, -1), ({"scale": INF}, -1), ({"scale": NAN}, -1), ({"q": 0}, -1), ({"k": 0}, -1), ({"v": 0}, -1), ({"o": 0}, -1), ({"starts": 0}, -1), ({"starts": P + 2}, -1),
                                       ({"q": P + 1}, -1), ({"T": 2 ** 30, "h": 8, "hk": 2}, -1), ({"T": 2 ** 30, "h": 64, "hk": 64}, -1), ({"n": 2 ** 31 - 1}, -1), ({"n": 0}, 0), ({"T": 0}, 0)])
def test_attn_refusals(args, code):
    assert _attn(**args) == code


def test_rope_freqs():
    pr = pkg("prompt")
    f = pr.rope_freqs(64, base=500000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1 and abs(f[16].item() * 500000.0 ** 0.5 - 1) < 1e-14
    assert torch.equal(pr.rope_freqs(64, 500000.0, 4.0, device="cpu"), f / 4)
    g = pr.rope_freqs(64, 500000.0, parts=(8.0, 8192, 1.0, 4.0), device="cpu")
    turns = f * 8192 / (2 * math.pi)
    share = (turns - 1) / 3
    mid = (share > 0) & (share < 1)
    assert mid.any() and torch.allclose(g[mid], f[mid] * (share + (1 - share) / 8)[mid], rtol=1e-13) and torch.equal(g[turns > 4], f[turns > 4])
    for bad in ((0,), (-4,), (6,)):
        with pytest.raises(ValueError):
            pr.rope_freqs(*bad, device="cpu")
    with pytest.raises(ValueError):
        pr.rope_freqs(64, parts=(8.0, 8192, 4.0, 4.0), device="cpu")


def test_python_calls_refuse_tensors_without_a_gpu():
    ql, pr = pkg("qlinear"), pkg("prompt")
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ql.fp8_quant_rows(x)
    e = torch.zeros(4, 256).to(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="CUDA"):
        ql.fp8_gemm(e, e, torch.zeros(2, 4), torch.zeros(1, 2))
    with pytest.raises(ValueError, match="CUDA"):
        pr.rope(x.view(4, 4, 64), None, torch.zeros(4, dtype=torch.int32), pr.rope_freqs(64, device="cpu"))
    with pytest.raises(ValueError, match="CUDA"):
        pr.attn(x.view(4, 4, 64), x.view(4, 4, 64), x.view(4, 4, 64), torch.zeros(2, dtype=torch.int32), 1.0)
