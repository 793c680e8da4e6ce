"""The prompt model's calls at the ends of what they document: tensors of more than 2^31 elements, outputs whose rows overlap, tensors of other ranks.

Bounds as in test_gpu_prompt.
"""
import ctypes
import math

import pytest
import torch

from conftest import pkg
from test_gpu_prompt import DEV, _attn_check, _codes, _operands, _product, _randn
from test_gpu_states import _check

pytestmark = pytest.mark.gpu


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _last_rows(n, last, *shape, seed=0, dtype=torch.bfloat16):
    """Zeros, and `last` rows of numbers behind them."""
    t = torch.zeros(n, *shape, dtype=dtype, device=DEV)
    t[n - last:] = _randn(seed, last, *shape).to(dtype)
    return t


def test_rows_past_32_bits():
    """A row's codes do not depend on where it lies."""
    ql = pkg("qlinear")
    M, K = 600000, 4096
    x, w = _last_rows(M, 5, K, seed=1), 1 + 0.1 * _randn(2, K)
    resid = _last_rows(M, 5, K, seed=3)
    want = ql.fp8_quant_rows(x[-5:].clone(), "rms", w, 1e-6, resid[-5:].clone())
    q, s, total = ql.fp8_quant_rows(x, "rms", w, 1e-6, resid, resid)
    assert total.data_ptr() == resid.data_ptr()
    for got, small in ((q[-5:], want[0]), (s[:, -5:], want[1]), (total[-5:], want[2])):
        assert torch.equal(_bits(got), _bits(small))
    assert not q[:M - 5:997].view(torch.uint8).any() and not total[:M - 5:997].any()


@pytest.mark.parametrize("M,N,K", [(150000, 40, 16384), (70000, 32768, 128), (40, 150000, 16384)])
def test_products_past_32_bits(M, N, K):
    ql = pkg("qlinear")
    G, last_m, last_n = K // 128, min(M, 20), min(N, 20)
    a, w = torch.zeros(M, K, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.zeros(N, K, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    a.view(torch.uint8)[M - last_m:] = _codes(1, last_m, K).view(torch.uint8)
    w.view(torch.uint8)[N - last_n:] = _codes(2, last_n, K).view(torch.uint8)
    xs, ws = torch.exp(_randn(3, G, M)) / 100, torch.exp(_randn(4, -(-N // 128), G)) / 100
    d = ql.fp8_gemm(a, w, xs, ws)
    first = N - last_n
    rows = ws.repeat_interleave(128, 0)[first:N]      # (of the last columns only)
    A = a[-last_m:].double() * xs[:, -last_m:].double().t().repeat_interleave(128, 1)
    W = w[-last_n:].double() * rows.double().repeat_interleave(128, 1)
    want, mass = A @ W.t().contiguous(), A.abs() @ W.abs().t().contiguous()
    cut = sum(7 * 2.0 ** -13 * (A[:, None, k:k + 8].abs() * W[None, :, k:k + 8].abs()).amax(-1) for k in range(0, K, 8))
    _check(d[-last_m:, -last_n:], want, (2.0 ** -8 * want.abs()).clamp(min=1e-38) + (128 + G + 4) * 2.0 ** -23 * mass + cut, "the last rows and columns")
    assert not d[:M - last_m:499].any() and not d[:, :N - last_n:499].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("M,N,K", [(1, 8, 128), (130, 260, 640), (300, 129, 1296), (257, 1000, 272), (128, 128, 8400)])
def test_products_two_workgroups_to_a_cu(M, N, K, dtype):
    ql, ffi = pkg("qlinear"), pkg("ffi")
    a, w, xs, ws, bias = _operands(M, N, K, dtype, seed=60)
    ffi.k("gpu_internal_fp8_gemm_force", 501)
    try:
        got = [ql.fp8_gemm(a, w, xs, ws, b, dtype) for b in (bias, None, None)]
        room = torch.zeros(M * N + 1, dtype=dtype, device=DEV)[1:].view(M, N)      # (an address that is no multiple of 16)
        ql.fp8_gemm(a, w, xs, ws, None, dtype, room)
    finally:
        ffi.k("gpu_internal_fp8_gemm_force", -1)
    for b, d in ((bias, got[0]), (None, got[1])):
        want, bound = _product(a, w, xs, ws, b, dtype)
        _check(d, want, bound, "bias" if b is not None else "no bias")
    assert torch.equal(got[1], got[2]) and torch.equal(room, got[1])


@pytest.mark.parametrize("M,N,K,dtype,form", [(2048, 4096, 256, torch.bfloat16, 5), (2048, 4096, 256, torch.float32, 2), (33, 256, 4096, torch.float32, 3), (200, 128, 64, torch.float32, 0)])
def test_sizes_take_the_forms_that_are_made_for_them(M, N, K, dtype, form):
    ql, ffi = pkg("qlinear"), pkg("ffi")
    out = (ctypes.c_int32 * 2)()
    ffi.k("gpu_internal_fp8_gemm_plan", M, N, K, ffi.DT_BF16 if dtype == torch.bfloat16 else ffi.DT_F32, ctypes.cast(out, ctypes.c_void_p))
    assert out[0] == form
    a, w, xs, ws, bias = _operands(M, N, K, dtype, seed=70)
    want, bound = _product(a[-40:], w, xs[:, -40:], ws, bias, dtype)
    _check(ql.fp8_gemm(a, w, xs, ws, bias, dtype)[-40:], want, bound, "the last rows")


def test_rope_past_32_bits():
    pr = pkg("prompt")
    T, h, hk, d = 500000, 32, 8, 128
    q, k = _last_rows(T, 5, h, d, seed=1), _last_rows(T, 5, hk, d, seed=2)
    p = torch.arange(T, dtype=torch.int32, device=DEV)
    f = pr.rope_freqs(d)
    want = pr.rope(q[-5:].clone(), k[-5:].clone(), p[-5:].clone(), f)
    got = pr.rope(q, k, p, f, out=(q, k))
    assert got[0] is q and torch.equal(q[-5:], want[0]) and torch.equal(k[-5:], want[1]) and not q[:T - 5:997].any()


def test_attention_past_32_bits():
    pr = pkg("prompt")
    n, each, h, d = 600, 1000, 32, 128
    T = n * each
    q, k, v = (_last_rows(T, each, h, d, seed=i) for i in (1, 2, 3))
    starts = torch.arange(0, T + 1, each, dtype=torch.int32, device=DEV)
    o = pr.attn(q, k, v, starts, d ** -0.5)
    heads = slice(h - 2, h)
    _attn_check(o[-each:, heads], q[-each:, heads], k[-each:, heads], v[-each:, heads], [0, each], d ** -0.5, True, "the last prompt")
    assert not o[:T - each:997].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("lens,h,hk,d,rows", [([20, 64, 1, 65, 0, 33, 77, 2] * 9, 16, 16, 64, 64), ([20, 64, 1, 65, 0, 33, 77, 2] * 9, 16, 16, 40, 64), ([20, 64, 1, 65, 0, 5] * 9, 12, 12, 80, 64),
                                              ([20, 64, 1, 65, 0, 5] * 9, 12, 12, 128, 64), ([20, 64, 1, 65, 0, 5] * 9, 12, 12, 256, 64), ([20, 64, 1, 65, 0, 5] * 9, 12, 12, 192, 128),
                                              ([150, 129, 1, 65, 0, 77] * 9, 16, 8, 104, 128), ([150, 129, 1, 65, 0, 77] * 18, 16, 16, 88, 128), ([520] * 12, 24, 24, 160, 256), ([520] * 12, 24, 24, 96, 128), ([77, 127, 64, 1], 12, 4, 80, 128),
                                              ([77, 127, 64, 1], 12, 4, 64, 128), ([77, 127, 128, 1], 4, 1, 128, 128),
                                              ([900, 130, 1], 4, 2, 160, (128, 2)), ([129, 127, 0, 300, 104], 6, 6, 192, (128, 2)), ([900, 130, 1], 4, 2, 256, (64, 2)), ([33, 500, 64, 1, 600], 6, 3, 200, (64, 2)),
                                              ([100, 33], 4, 2, 160, 128), ([199], 4, 2, 256, 128)])
def test_attention_forms_by_the_prompts_lengths(lens, h, hk, d, rows, dtype):
    """Prompts of a token, of a whole tile, of one more, and of none."""
    pr, ffi = pkg("prompt"), pkg("ffi")
    T, out = sum(lens), (ctypes.c_int32 * 2)()
    ffi.k("gpu_internal_prompt_attn_form", T, len(lens), h, hk, d, ctypes.cast(out, ctypes.c_void_p))
    assert tuple(out) == (rows if isinstance(rows, tuple) else (rows, 0))
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    qkv = _randn(80, T, h + 2 * hk, d, size=1.3).to(dtype)
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    at = torch.tensor(starts, dtype=torch.int32, device=DEV)
    heads = slice(h - 2 * h // hk, h), slice(hk - 2, hk)
    for causal in (True, False):
        o = pr.attn(q, k, v, at, d ** -0.5, causal)
        _attn_check(o[:, heads[0]], q[:, heads[0]], k[:, heads[1]], v[:, heads[1]], starts[:7], d ** -0.5, causal, "causal" if causal else "all keys")
        assert torch.equal(o, pr.attn(q, k, v, at, d ** -0.5, causal))
    # a NaN behind a row's keys does not reach it, one among them does
    n = next(i for i, l in enumerate(lens) if l > 4)
    hole, end = starts[n] + 3, starts[n + 1]
    v = v.clone()
    v[hole, :, 3] = math.nan
    o = pr.attn(q, k, v, at, d ** -0.5)
    assert o[hole:end, :, 3].isnan().all() and not o[:hole].isnan().any() and not o[end:].isnan().any() and not o[..., 4:].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("lens,h,hk,d,form", [([2050], 66, 33, 96, (256, 1)), ([1300, 3, 900, 1], 6, 3, 72, (128, 2)), ([200], 5, 5, 80, (128, 2)), ([129, 150], 4, 1, 88, (128, 2))])
def test_attention_of_72_to_96_channels_as_128(lens, h, hk, d, form, dtype):
    """Rows at other addresses than whole 16 bytes too, and numbers behind the channels that there are: not read as channels."""
    pr, ffi = pkg("prompt"), pkg("ffi")
    T, out = sum(lens), (ctypes.c_int32 * 2)()
    ffi.k("gpu_internal_prompt_attn_form", T, len(lens), h, hk, d, ctypes.cast(out, ctypes.c_void_p))
    assert tuple(out) == form
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    wide = torch.full((T, h + 2 * hk, 128), math.nan, dtype=dtype, device=DEV)
    wide[..., :d] = _randn(90, T, h + 2 * hk, d, size=1.3).to(dtype)
    qkv = wide[..., :d]
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    at = torch.tensor(starts, dtype=torch.int32, device=DEV)
    out = torch.full((T, h, 128), 7.0, dtype=dtype, device=DEV)
    o = pr.attn(q, k, v, at, d ** -0.5, out=out[..., :d])
    heads = slice(h - 2 * h // hk, h), slice(hk - 2, hk)
    if hk == 1:
        heads = slice(0, h), slice(0, 1)
    _attn_check(o[:, heads[0]], q[:, heads[0]], k[:, heads[1]], v[:, heads[1]], starts, d ** -0.5, True, "causal")
    assert (out[..., d:] == 7).all()
    room = [torch.zeros(t.numel() + 1, dtype=dtype, device=DEV)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    far = pr.attn(*room, at, d ** -0.5)
    _attn_check(far[:, heads[0]], q[:, heads[0]], k[:, heads[1]], v[:, heads[1]], starts, d ** -0.5, True, "odd addresses")


def test_outputs_with_rows_that_share_memory_and_other_ranks_are_refused():
    ql, pr = pkg("qlinear"), pkg("prompt")
    x = torch.ones(4, 256, device=DEV).bfloat16()
    q, k = torch.ones(4, 2, 64, device=DEV).bfloat16(), torch.ones(4, 1, 64, device=DEV).bfloat16()
    p, f, s = torch.arange(4, dtype=torch.int32, device=DEV), pr.rope_freqs(64), torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    one, wide = x[:1].expand(4, 256), torch.ones(4 * 256, device=DEV).bfloat16().as_strided((4, 256), (200, 1))
    heads = q[:, :1].expand(4, 2, 64)
    tokens = torch.ones(1024, device=DEV).bfloat16().as_strided((4, 2, 64), (64, 64, 1))
    for bad in (lambda: ql.fp8_quant_rows(x, resid=x, out=one), lambda: ql.fp8_quant_rows(x, resid=x, out=wide), lambda: pr.rope(q, k, p, f, out=(heads, k)), lambda: pr.rope(q, k, p, f, out=(tokens, k)),
                lambda: pr.rope(q, k, p, f, out=(torch.empty_like(q), k[:1].expand(4, 1, 64))), lambda: pr.attn(q, k, k, s, 1.0, out=heads), lambda: pr.attn(q, k, k, s, 1.0, out=tokens),
                lambda: pr.rope(q, k[0, 0], p, f), lambda: pr.rope(q, k[0], p, f), lambda: pr.rope(q[0], k, p, f), lambda: pr.attn(q, k[0, 0], k, s, 1.0), lambda: pr.attn(q, k, k[0], s, 1.0),
                lambda: pr.attn(q[0, 0], k, k, s, 1.0), lambda: ql.fp8_quant_rows(x[0, 0]), lambda: ql.fp8_quant_rows(x[None])):
        with pytest.raises(ValueError):
            bad()
    # inputs may share theirs, and outputs may lie heads first
    got = ql.fp8_quant_rows(one, resid=x)
    assert (got[2] == 2).all()
    out = torch.empty(2, 4, 64, device=DEV).bfloat16().transpose(0, 1)
    assert torch.equal(pr.attn(heads, k, k, s, 1.0, out=out), pr.attn(heads, k, k, s, 1.0))
    assert torch.equal(pr.rope(heads, None, p, f, out=(out, None))[0], pr.rope(heads, None, p, f)[0])
