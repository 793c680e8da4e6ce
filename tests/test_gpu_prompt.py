"""A prompt model's layer in 8-bit floating point on the GPU against the formulas in 64 bits: rows with norm, gate and codes, products with a scale
for each block of 128, rotary positions, attention over packed prompts, and a run of them together.

Bounds count roundings, each off by at most half a step u (bf16 2^-8, f16 2^-11, fp32 2^-24, e4m3 2^-4 relative to the value, 2^-10 below its ordinary
numbers); sums of n numbers in fp32 in any order by n 2^-23 of the sum of their magnitudes at most (2^-23, not 2^-24, where a matrix instruction
may cut off instead of rounding).
"""
import math

import pytest
import torch

from conftest import pkg
from test_gpu_states import U, _check, _reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4 = torch.float8_e4m3fn
TYPES = [torch.bfloat16, torch.float16, torch.float32]
name = lambda v: str(v).replace("torch.", "")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(seed, *shape, size=1.0):
    return size * torch.randn(*shape, device=DEV, generator=_gen(seed))


# ---- rows -> codes ---------------------------------------------------------------------------------------------------------------

def _rows_check(q, scales, n, off, what):
    """q [M, K], scales [G, M] against n in 64 bits, of which the kernel's is off by `off` of itself at most."""
    M, K = n.shape
    G = -(-K // 128)
    assert q.shape == (M, K) and q.dtype == E4 and scales.shape == (G, M) and scales.dtype == torch.float32, what
    pad = torch.nn.functional.pad(n, (0, 128 * G - K)).view(M, G, 128)
    A = pad.abs().amax(-1).clamp(min=2.0 ** -100)
    assert ((scales.t().double() - A / 448).abs() <= (off + 2.0 ** -23) * A / 448 + 2.0 ** -149).all(), what
    y = n * (448 / A).repeat_interleave(128, 1)[:, :K]
    far = (q.double() - y).abs() - ((2.0 ** -4 * y.abs()).clamp(min=2.0 ** -10) + (2 * off + 2.0 ** -21) * y.abs())
    assert far.max().item() <= 0, "%s: %.3g over the bound" % (what, far.max().item())


ROWS = [(1, 16), (3, 128), (2, 144), (5, 1040), (1, 4096), (65, 2048), (300, 512), (2100, 640), (4, 8192), (2, 12304), (3, 32768)]


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("M,K", ROWS)
def test_quant_rows(M, K, dtype):
    ql = pkg("qlinear")
    x = (_randn(1, M, 2 * K) * torch.exp(_randn(2, 2 * K))).to(dtype)
    if K % 2 == 0:
        q, s = ql.fp8_quant_rows(x, "swiglu")
        gate, up = x[:, :K].double(), x[:, K:].double()
        # e^-x by 2^(x log2 e): the product is off by |x| 2^-24 of a power, and four operations by a unit each
        _rows_check(q, s, torch.nn.functional.silu(gate) * up, (gate.abs().max().item() + 8) * 2.0 ** -23, "swiglu")
    x = x[:, :K]            # rows further apart than they are long
    q, s = ql.fp8_quant_rows(x)
    _rows_check(q, s, x.double(), 0.0, "plain")
    # the same operations elsewhere: equal (448 / A of a number and a tensor would be a product with the reciprocal)
    pad = torch.nn.functional.pad(x.float().cpu(), (0, -K % 128)).view(M, -1, 128)
    A = pad.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    assert torch.equal(q.cpu().view(torch.uint8), (pad * (torch.tensor(448.0) / A)).to(E4).view(M, -1)[:, :K].contiguous().view(torch.uint8)) and torch.equal(s.cpu(), (A[..., 0] / 448).t())
    w, resid = 1 + 0.2 * _randn(3, K), _randn(4, M, K, size=2.0).to(dtype)
    # a sum of K squares in fp32, half of whose error the root keeps, and six operations
    off = (0.5 * min(K, 64 * 8 + 16) + 8) * 2.0 ** -24
    for r, got in ((None, ql.fp8_quant_rows(x, "rms", w, 1e-6)), (resid, ql.fp8_quant_rows(x, "rms", w, 1e-6, resid))):
        total = x if r is None else (x.float() + r.float()).to(dtype)
        t = total.double()
        _rows_check(got[0], got[1], t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w.double(), off, "rms")
        if r is not None:
            assert torch.equal(got[2], total)
    q, s, total = ql.fp8_quant_rows(x, resid=resid)
    assert torch.equal(total, (x.float() + resid.float()).to(dtype))
    q2, s2 = ql.fp8_quant_rows(total)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


def test_quant_rows_in_place_unaligned_and_odd_values():
    ql = pkg("qlinear")
    M, K = 37, 400
    big = _randn(5, M, K + 3).bfloat16()
    x, resid, w = big[:, 3:], _randn(6, M, K + 1).bfloat16()[:, 1:], torch.ones(K + 1, device=DEV)[1:]
    want = ql.fp8_quant_rows(x.contiguous(), "rms", w, 1e-5, resid.contiguous())
    keep = resid.clone()
    got = ql.fp8_quant_rows(x, "rms", w, 1e-5, resid, out=resid)
    assert got[2].data_ptr() == resid.data_ptr() and torch.equal(resid, want[2]) and torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
    got = ql.fp8_quant_rows(x, "rms", w, 1e-5, keep, out=x)
    assert torch.equal(x, want[2]) and torch.equal(got[1], want[1]) and not torch.equal(big[:, :3], torch.zeros_like(big[:, :3]))
    # zeros, next to nothing, the largest, and what is no number
    x = torch.zeros(6, 256, device=DEV)
    x[1, :128], x[1, 200] = 1e-38, 2.0 ** -100
    x[2] = 3e38
    x[3, 5], x[3, 130] = math.nan, 1.0
    x[4, 250], x[4, 0] = -math.inf, 2.0
    x[5, 7] = 2.0 ** -149
    q, s = ql.fp8_quant_rows(x)
    v = q.float() * s.t().repeat_interleave(128, 1)
    assert not v[0].any() and v[1, 200] == 2.0 ** -100 and ((v[2] - 3e38).abs() <= 3e38 * 2.0 ** -4).all() and not v[5].any()
    assert v[3, :128].isnan().all() and v[3, 130] == 1 and not v[3, 131:].any()
    assert v[4, 128:].isnan().all() and v[4, 0] == 2
    g = torch.cat((x, torch.ones_like(x)), 1)
    q, s = ql.fp8_quant_rows(g, "swiglu")
    v = q.float() * s.t().repeat_interleave(128, 1)
    assert v[3, :128].isnan().all() and v[4, 128:].isnan().all() and abs(v[3, 130].item() - 0.7310586) < 0.05 and not v[0].any()
    # gates at both ends
    g = torch.zeros(1, 256, device=DEV)
    g[0, :6], g[0, 128:] = torch.tensor([-1e5, -200.0, -88.0, 90.0, 3e38, -3e38], device=DEV), 1.0
    q, s = ql.fp8_quant_rows(g, "swiglu")
    assert q.float().isfinite().all() and q[0, 4].float() == 448 and s[0, 0] == torch.tensor(3e38) / 448
    g[0, :6] = torch.tensor([-1e5, -200.0, -60.0, 20.0, -2.0, 0.5], device=DEV)
    q, s = ql.fp8_quant_rows(g, "swiglu")
    _rows_check(q, s, torch.nn.functional.silu(g[:, :128].double()), 70 * 2.0 ** -23, "gates")
    q, s = ql.fp8_quant_rows(torch.zeros(0, 64, device=DEV))
    assert q.shape == (0, 64) and s.shape == (1, 0)


# ---- products --------------------------------------------------------------------------------------------------------------------

def _codes(seed, n, k):
    c = torch.randint(0, 256, (n, k), dtype=torch.uint8, device=DEV, generator=_gen(seed))
    return torch.where(c & 127 == 127, c - 1, c).view(E4)


def _operands(M, N, K, dtype, seed=0):
    G = -(-K // 128)
    xs, ws = torch.exp(_randn(seed + 3, G, M)) / 100, torch.exp(_randn(seed + 4, -(-N // 128), G)) / 100
    return _codes(seed + 1, M, K), _codes(seed + 2, N, K), xs, ws, _randn(seed + 5, N).to(dtype)


def _product(a, w, xs, ws, bias, dtype):
    """In 64 bits, and the bound: sums of 128 in the matrix instruction, then over the groups, two operations on each.  For 16-bit outputs the
    instruction cuts seven of each eight products off at 2^-13 of the largest one's power of two."""
    (M, K), N = a.shape, w.shape[0]
    A = a.double() * xs.double().t().repeat_interleave(128, 1)[:, :K]
    W = w.double() * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    d = A @ W.t().contiguous()
    mass = A.abs() @ W.abs().t().contiguous()
    cut = 0.0
    if dtype != torch.float32:
        for k in range(0, K, 8):
            top = (A[:, None, k:k + 8].float().abs() * W[None, :, k:k + 8].float().abs()).amax(-1) if M * N <= 300000 else A[:, k:k + 8].abs().amax(1)[:, None] * W[:, k:k + 8].abs().amax(1)
            cut = cut + 7 * 2.0 ** -13 * top.double()
    if bias is not None:
        d = d + bias.double()
        mass = mass + bias.double().abs()
    low = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    return d, (U[dtype] * d.abs()).clamp(min=low) + (min(K, 128) + xs.shape[0] + 4) * 2.0 ** -23 * mass + cut


GEMM = [(1, 1, 16), (1, 128, 128), (3, 5, 144), (16, 128, 256), (17, 130, 400), (64, 256, 1024), (5, 1000, 4096), (128, 128, 128), (129, 127, 2640), (100, 520, 1152), (256, 512, 2048),
        (300, 264, 640), (1000, 1000, 384), (513, 777, 256), (700, 600, 1168), (512, 1040, 128), (769, 520, 4224)]


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("M,N,K", GEMM)
def test_fp8_gemm(M, N, K, dtype):
    ql = pkg("qlinear")
    a, w, xs, ws, bias = _operands(M, N, K, dtype)
    for b in (None, bias):
        want, bound = _product(a, w, xs, ws, b, dtype)
        _check(ql.fp8_gemm(a, w, xs, ws, b, dtype), want, bound, "bias" if b is not None else "plain")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=name)
@pytest.mark.parametrize("form,slices,sizes", [(0, 1, (40, 200, 1040)), (1, 1, (300, 260, 1040)), (1, 1, (20, 30, 128)), (2, 1, (130, 260, 640)), (2, 3, (200, 130, 1296)), (2, 7, (1, 1, 1024)),
                                               (3, 1, (65, 129, 640)), (3, 2, (64, 128, 400)), (3, 31, (50, 200, 4096)), (4, 1, (31, 70, 1040)), (4, 3, (16, 200, 4112)), (4, 2, (2, 4500, 144)),
                                               (4, 2, (17, 4500, 400))])
def test_every_form_of_fp8_gemm(form, slices, sizes, dtype):
    """Forced on sizes of any kind; where a form does not take a size, the one for any size runs."""
    ql, ffi = pkg("qlinear"), pkg("ffi")
    a, w, xs, ws, bias = _operands(*sizes, dtype, 70)
    want, bound = _product(a, w, xs, ws, bias, dtype)
    ffi.k("gpu_internal_fp8_gemm_force", 100 * form + slices)
    try:
        got = ql.fp8_gemm(a, w, xs, ws, bias, dtype)
        again = ql.fp8_gemm(a, w, xs, ws, bias, dtype)
    finally:
        ffi.k("gpu_internal_fp8_gemm_force", -1)
    _check(got, want, bound, "form %d" % form)
    assert torch.equal(got, again)


def test_fp8_gemm_layouts_and_odd_values():
    """Scales further apart than they are many, outputs at any address; codes and scales that are no numbers reach their rows and columns only."""
    ql = pkg("qlinear")
    M, N, K = 150, 200, 400
    a, w, xs, ws, bias = _operands(M, N, K, torch.bfloat16, 20)
    want = ql.fp8_gemm(a, w, xs, ws, bias)
    wide = torch.full((4, M + 7), math.nan, device=DEV)
    wide[:, 3:M + 3] = xs
    assert torch.equal(ql.fp8_gemm(a, w, wide[:, 3:M + 3], ws, bias), want)
    room = torch.zeros(M * N + 8, dtype=torch.bfloat16, device=DEV)
    D = room[1:M * N + 1].view(M, N)
    assert ql.fp8_gemm(a, w, xs, ws, bias, D=D) is D and torch.equal(D, want) and room[0] == 0 and not room[M * N + 1:].any()
    a.view(torch.uint8)[7, 130], w.view(torch.uint8)[11, 3], xs[2, 90] = 127, 255, math.nan
    got = ql.fp8_gemm(a, w, xs, ws, bias)
    bad = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    bad[7], bad[:, 11], bad[90] = True, True, True
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad])


# ---- rotary positions ------------------------------------------------------------------------------------------------------------

def _rope_want(x, positions, freqs, inter, factor, norm, eps):
    """In 64 bits, and how far 32-bit arithmetic and the output's rounding may be from it."""
    x = x.double()
    d, rel = x.shape[2], 2.0 ** -21      # sine and cosine by a few units, and two products and a sum
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * norm.double()
        rel += (d + 8) * 2.0 ** -24
    r = 2 * freqs.shape[0]
    at = positions.double()[:, None, None] * freqs
    cos, sin = torch.cos(at), torch.sin(at)
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., :r // 2], x[..., r // 2:r])
    u, v = factor * (a * cos - b * sin), factor * (a * sin + b * cos)
    mass = factor * (a.abs() + b.abs()) * (rel + at.abs() * 2.0 ** -50)
    both = lambda p, q: torch.stack((p, q), -1).flatten(-2) if inter else torch.cat((p, q), -1)
    rest = x[..., r:]
    return torch.cat((both(u, v), rest), -1), torch.cat((both(mass, mass), rest.abs() * rel), -1)


ROPE = [(1, 1, 1, 4, 4), (12, 32, 8, 128, 128), (3, 5, 2, 64, 32), (70, 4, 4, 80, 80), (5, 7, 7, 72, 72), (2, 3, 1, 256, 256), (9, 2, 1, 96, 40), (4, 3, 3, 40, 20), (1100, 2, 1, 128, 64), (7, 6, 0, 128, 96),
        (6, 1, 1, 252, 4)]


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "inter"])
@pytest.mark.parametrize("T,h,hk,d,rot", ROPE)
def test_rope(T, h, hk, d, rot, inter, dtype):
    pr = pkg("prompt")
    qkv = _randn(30, T, h + 2 * hk, d, size=2.0).to(dtype)
    q, k = qkv[:, :h], qkv[:, h:h + hk] if hk else None
    positions = torch.randint(-5, 1 << 21, (T,), dtype=torch.int32, device=DEV, generator=_gen(31))
    positions[0] = 0
    freqs = pr.rope_freqs(rot, stretch=4.0)
    qn, kn = 1 + 0.1 * _randn(32, d), 1 + 0.1 * _randn(33, d)
    for factor, norms in ((1.0, (None, None)), (1.25, (qn, kn)), (1.0, (None, kn))):
        got = pr.rope(q, k, positions, freqs, inter, factor, *norms, 1e-6)
        for x, y, norm in ((q, got[0], norms[0]), (k, got[1], norms[1])):
            if x is None:
                assert y is None
                continue
            want, bound = _rope_want(x, positions, freqs, inter, factor, norm, 1e-6)
            _check(y, want, bound + (U[dtype] * want.abs()).clamp(min=2.0 ** -25 if dtype == torch.float16 else 1e-38) * 1.001, "factor %g" % factor)
            if norm is None:
                assert torch.equal(y[..., rot:], x[..., rot:])
    # in place, and at an odd address
    q2, k2 = q.clone(), None if k is None else k.clone()
    pr.rope(q2, k2, positions, freqs, inter, 1.0, None, kn, 1e-6, out=(q2, k2))
    assert torch.equal(q2, got[0]) and (k is None or torch.equal(k2, got[1]))
    room = torch.zeros(q.numel() + 1, dtype=dtype, device=DEV)
    q3 = room[1:].view(q.shape)
    q3.copy_(q)
    assert torch.equal(pr.rope(q3, k, positions, freqs, inter, 1.0, None, kn, 1e-6)[0], got[0])


def test_rope_at_far_positions_and_long_contexts():
    """The largest positions turn as exactly as near ones; a position of an interpolated table is that of a nearer one."""
    pr = pkg("prompt")
    x = torch.ones(4, 1, 128, device=DEV)
    far = torch.tensor([2 ** 31 - 1, -2 ** 31, 1 << 30, 10 ** 9 + 7], dtype=torch.int32, device=DEV)
    freqs = pr.rope_freqs(128, base=500000.0)
    want, bound = _rope_want(x, far, freqs, False, 1.0, None, 0.0)
    _check(pr.rope(x, None, far, freqs)[0], want, bound + 2.0 ** -24, "far")
    p = torch.arange(4, dtype=torch.int32, device=DEV)
    assert torch.equal(pr.rope(x, None, 8 * p, pr.rope_freqs(128, stretch=8.0))[0], pr.rope(x, None, p, pr.rope_freqs(128))[0])
    f, by = pr.rope_freqs(128), pr.rope_freqs(128, parts=(32.0, 4096, 1.0, 32.0))
    turns = f * 4096 / (2 * math.pi)
    assert torch.equal(by[turns >= 32], f[turns >= 32]) and torch.allclose(by[turns <= 1], f[turns <= 1] / 32, rtol=1e-12) and (by <= f).all() and (by >= f / 32 * (1 - 1e-12)).all()


# ---- attention over packed prompts -----------------------------------------------------------------------------------------------

def _attn_check(o, q, k, v, starts, scale, causal, what=""):
    h, hk = q.shape[1], k.shape[1]
    for s, (b, e) in enumerate(zip(starts[:-1], starts[1:])):
        keep = torch.ones(e - b, e - b, dtype=torch.bool, device=DEV)
        if causal:
            keep = keep.tril()
        for j in range(h):
            x, y, z = q[b:e, j], k[b:e, j * hk // h], v[b:e, j * hk // h]
            if e > b:
                want, bound = _reference(x, y, z, scale, keep, torch.zeros(e - b, dtype=torch.float64, device=DEV), U[q.dtype], U[q.dtype], z.double().abs().max() if q.dtype == torch.float16 else None)
                _check(o[b:e, j], want, bound, "%s prompt %d head %d" % (what, s, j))


# (rows of a workgroup, waves to a row's keys): each form that there is
FORMS = {(64, 4): ([900, 130], 4, 1, 64), (128, 2): ([1000, 300, 1], 4, 2, 128), (256, 1): ([2100, 515, 1], 20, 20, 128), (128, 0): ([300, 5, 200, 150, 290, 70, 310, 64, 65] * 2, 16, 16, 128),
         (256, 0): ([420, 700, 63, 640, 450, 800], 24, 24, 64)}


def test_attn_forms_are_those_of_their_sizes():
    import ctypes
    ffi = pkg("ffi")
    out = (ctypes.c_int32 * 2)()
    for form, (lens, h, hk, d) in FORMS.items():
        ffi.k("gpu_internal_prompt_attn_form", sum(lens), len(lens), h, hk, d, ctypes.cast(out, ctypes.c_void_p))
        assert tuple(out) == form, (lens, tuple(out))


ATTN = [*FORMS.values(), ([700], 20, 20, 64), ([2500, 1800], 10, 10, 64), ([1200], 3, 3, 40), ([1300, 2], 2, 1, 104), ([1111], 24, 24, 56), ([900], 33, 33, 120), ([1] * 7 + [640, 128, 256], 2, 2, 128), ([1], 1, 1, 8), ([1, 2, 1], 4, 2, 64), ([0, 5, 0, 33, 0], 2, 2, 128), ([77, 64, 1, 200], 3, 1, 64), ([129, 31, 65], 8, 2, 128), ([300], 6, 6, 72), ([40, 513], 2, 1, 256), ([260], 7, 1, 160),
        ([128, 128], 2, 2, 96), ([1111], 4, 1, 128), ([700, 3, 1300], 4, 4, 80), ([2000, 47], 12, 4, 64), ([3, 2050], 5, 5, 48), ([1500, 900], 16, 16, 192), ([1000, 700, 300], 20, 20, 256),
        ([2600], 30, 15, 88), ([1700, 300], 24, 24, 128), ([1] * 130 + [70], 2, 1, 40)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=name)
@pytest.mark.parametrize("lens,h,hk,d", ATTN, ids=lambda v: str(v) if isinstance(v, int) else "x".join(map(str, v[-4:])))
def test_attn(lens, h, hk, d, dtype):
    pr = pkg("prompt")
    T = sum(lens)
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    qkv = _randn(40, T, h + 2 * hk, d, size=1.3).to(dtype)
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    at = torch.tensor(starts, dtype=torch.int32, device=DEV)
    scale = d ** -0.5
    _attn_check(pr.attn(q, k, v, at, scale), q, k, v, starts, scale, True, "causal")
    if T <= 1200:
        _attn_check(pr.attn(q, k, v, at, -scale, causal=False), q, k, v, starts, -scale, False, "all keys")


def test_attn_layouts_rows_of_no_prompt_and_bad_starts():
    pr = pkg("prompt")
    T, h, hk, d = 180, 4, 2, 64
    q, k, v = (_randn(50 + i, n, T, d).transpose(0, 1).bfloat16() for i, n in enumerate((h, hk, hk)))      # heads further apart than tokens
    starts = torch.tensor([20, 90, 90, 160], dtype=torch.int32, device=DEV)
    out = torch.full((T, h, d), 7.0, dtype=torch.bfloat16, device=DEV)
    got = pr.attn(q, k, v, starts, 0.125, out=out)
    assert got is out and (out[:20] == 7).all() and (out[160:] == 7).all()
    _attn_check(out, q, k, v, starts.tolist(), 0.125, True)
    # unaligned rows
    room = [torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    again = torch.full((T, h, d + 1), 7.0, dtype=torch.bfloat16, device=DEV)[:, :, 1:]
    pr.attn(*room, starts, 0.125, out=again)
    assert torch.equal(again, out)
    # starts outside the rows, and not growing: nothing outside is touched, and rows that one prompt alone has are right (10 .. 400 has some of the first)
    wild = torch.tensor([-50, 30, 10, 400, 400, 100], dtype=torch.int32, device=DEV)
    edge = torch.full((T + 64, h, d), 7.0, dtype=torch.bfloat16, device=DEV)
    pr.attn(q, k, v, wild, 0.125, out=edge[:T])
    assert (edge[T:] == 7).all()
    _attn_check(edge, q, k, v, [0, 10], 0.125, True)
    assert pr.attn(q[:0], k[:0], v[:0], starts, 1.0).shape == (0, h, d)
    assert (pr.attn(q, k, v, starts[:1], 1.0, out=torch.full_like(out, 3.0)) == 3).all()


def test_attn_large_scores_and_values_that_are_no_numbers():
    """Scores up to the ends of fp32; a key that holds no number reaches the rows that see it, and no others."""
    pr = pkg("prompt")
    T, d = 400, 128
    starts = torch.tensor([0, 150, 400], dtype=torch.int32, device=DEV)
    q, k, v = (_randn(60 + i, T, 2, d, size=s).bfloat16() for i, s in enumerate((30.0, 30.0, 1.0)))
    _attn_check(pr.attn(q, k, v, starts, 1.0), q, k, v, [0, 150, 400], 1.0, True, "large")
    want = pr.attn(q, k, v, starts, 0.05)
    k[200, 0, 3], v[60, 1, 5] = math.nan, math.inf
    got = pr.attn(q, k, v, starts, 0.05)
    assert torch.equal(got[:200, 0], want[:200, 0]) and got[200:, 0].isnan().all()
    assert torch.equal(got[:60, 1], want[:60, 1]) and torch.equal(got[150:, 1], want[150:, 1]) and not got[60:150, 1, 5].isfinite().any()
