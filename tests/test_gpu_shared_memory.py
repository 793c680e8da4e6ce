"""Outputs of a prompt model's calls that share memory with what they read: refused, but where they go in an input's place, which gives the same bits."""
import pytest
import torch

from conftest import pkg
from test_gpu_prompt import DEV, E4, _randn, name

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.fixture(params=[True, False], ids=["native", "python"])
def calls(request, monkeypatch):
    """The calls, made natively and in Python."""
    ql = pkg("qlinear")
    if not request.param:
        monkeypatch.setattr(ql, "_pycalls", None)
    return ql, pkg("prompt")


def test_outputs_over_inputs_are_refused(calls):
    ql, pr = calls
    x = torch.zeros(40, 256, device=DEV).bfloat16()
    a, b, w = x[:20], x[20:], torch.ones(256, device=DEV)
    both = torch.zeros(41, 256, device=DEV).bfloat16()
    t = torch.zeros(30, 8, 64, device=DEV).bfloat16()
    q, k, v = t[:, :4], t[:, 4:6], t[:, 6:]
    p, f, s = _i32(range(30)), pr.rope_freqs(64), _i32([0, 30])
    flat = torch.zeros(1 << 16, device=DEV).bfloat16()
    codes, W, xs, ws = torch.zeros(4, 256, device=DEV).to(E4), torch.zeros(512, 256, device=DEV).to(E4), torch.ones(2, 4, device=DEV), torch.ones(4, 2, device=DEV)
    for bad in (lambda: ql.fp8_quant_rows(a, resid=b, out=x[1:21]), lambda: ql.fp8_quant_rows(a, resid=b, out=x[10:30]), lambda: ql.fp8_quant_rows(both[:40], resid=x, out=both[1:]),
                lambda: ql.fp8_quant_rows(x, resid=both[1:], out=both[:40]), lambda: ql.fp8_quant_rows(flat[:800].view(20, 40)[:, :16], resid=a[:, :16], out=flat[:640].view(20, 32)[:, :16]),
                lambda: ql.fp8_quant_rows(a.float(), "rms", w, 0.1, resid=b.float(), out=w.expand(20, 256)), lambda: ql.fp8_gemm(codes, W, xs, ws, D=W.view(torch.bfloat16).view(-1)[:2048].view(4, 512)),
                lambda: ql.fp8_gemm(codes, W[:2], xs, ws[:1], None, torch.float32, xs.view(4, 2)), lambda: ql.fp8_gemm(codes, W[:8], xs, ws[:1], None, torch.float32, codes.view(torch.float32).view(-1)[:32].view(4, 8)),
                lambda: pr.rope(q, t[:, 4:], p, f, out=(t[:, 4:], q)), lambda: pr.rope(q, k, p, f, out=(t[:, 1:5], torch.empty_like(k))),
                lambda: pr.rope(q, k, p, f, out=(q, t[:, 3:5])), lambda: pr.rope(q, q, p, f, out=(q, torch.empty_like(q))), lambda: pr.rope(q, q, p, f, out=(q, q)),
                lambda: pr.rope(q[:29], None, p[:29], f, out=(q[1:], None)), lambda: pr.rope(q, k, p, f, out=(flat[:30 * 256].view(30, 4, 64), flat[128:128 + 30 * 128].view(30, 2, 64))),
                lambda: pr.attn(q, t[:, 4:], t[:, 4:], s, 1.0, out=t[:, 4:]), lambda: pr.attn(q, k, v, s, 1.0, out=t[:, 2:6]), lambda: pr.attn(q, k, v, s, 1.0, out=t[:, 3:7]),
                lambda: pr.attn(q, k, v, s, 1.0, out=t[:, 1:5]), lambda: pr.attn(q[:29], k[:29], v[:29], s, 1.0, out=q[1:]), lambda: pr.attn(v, v, v, s, 1.0, out=v)):
        with pytest.raises(ValueError, match="memory"):
            bad()


def test_outputs_beside_inputs_and_in_their_places_are_not(calls):
    ql, pr = calls
    fused = _randn(1, 60, 12, 64).bfloat16()
    q, k, v = fused[:, :8], fused[:, 8:10], fused[:, 10:]
    p, f, s = _i32(range(60)), pr.rope_freqs(64), _i32([0, 25, 60])
    turned = pr.rope(q, k, p, f)
    want = pr.attn(*turned, v, s, 0.125)
    assert torch.equal(pr.attn(*turned, v, s, 0.125, out=turned[0]), want)
    keep = v.clone()
    got = pr.rope(q, k, p, f, out=(q, k))
    assert got[0] is q and got[1] is k and torch.equal(k, turned[1])
    assert pr.attn(q, k, v, s, 0.125, out=q) is q and torch.equal(q, want) and torch.equal(v, keep)
    # columns of a buffer that the inputs are in, heads in turns, rows that interleave at other distances
    wide = torch.zeros(60, 20, 64, device=DEV).bfloat16()
    wide[:, :12] = fused
    assert torch.equal(pr.attn(wide[:, :8], wide[:, 8:10], wide[:, 10:12], s, 0.125, out=wide[:, 12:]), pr.attn(q, k, v, s, 0.125))
    turns = torch.zeros(60, 4, 3, 64, device=DEV).bfloat16()
    turns[:, :, 0], turns[:, :, 1] = q[:, :4], q[:, 4:]
    assert torch.equal(pr.attn(turns[:, :, 0], turns[:, :, 1], turns[:, :, 1], s, 0.125, out=turns[:, :, 2]), pr.attn(q[:, :4], q[:, 4:], q[:, 4:], s, 0.125))
    room = torch.zeros(4096, device=DEV).bfloat16()
    x, out = room.as_strided((20, 16), (96, 1)), room.as_strided((20, 16), (192, 1), 32)
    x.copy_(_randn(2, 20, 16))
    r = _randn(3, 20, 16).bfloat16()
    want = (x.float() + r.float()).bfloat16()
    assert torch.equal(ql.fp8_quant_rows(x, resid=r, out=out)[2], want) and torch.equal(ql.fp8_quant_rows(x, resid=r, out=x)[2], want) and torch.equal(x, want)


FORMS = [([900, 130], 4, 1, 64), ([1000, 900], 10, 10, 64), ([1000] * 4, 16, 16, 128), ([1000, 300, 1], 4, 2, 128), ([290, 70, 310, 1], 16, 16, 128), ([77, 40], 3, 3, 96), ([700, 1000], 6, 3, 80),
         ([1000, 300], 2, 2, 192), ([520] * 12, 24, 24, 160), ([1000, 300], 2, 2, 256), ([20, 64, 1, 65, 0, 33] * 9, 16, 16, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=name)
@pytest.mark.parametrize("lens,h,hk,d", FORMS, ids=lambda v: str(v) if isinstance(v, int) else "x".join(map(str, v[:4])))
def test_attention_in_the_queries_place(lens, h, hk, d, dtype):
    pr = pkg("prompt")
    T, at = sum(lens), _i32([sum(lens[:i]) for i in range(len(lens) + 1)])
    fused = _randn(5, T, h + 2 * hk, d, size=1.3).to(dtype)
    for causal in (True, False):
        t = fused.clone()
        q, k, v = t[:, :h], t[:, h:h + hk], t[:, h + hk:]
        want = pr.attn(q, k, v, at, d ** -0.5, causal)
        pr.attn(q, k, v, at, d ** -0.5, causal, out=q)
        assert torch.equal(q, want) and torch.equal(t[:, h:], fused[:, h:])


def test_outputs_are_taken_natively(monkeypatch):
    """The usual ones: tensors of their own, an input's place, columns of one buffer."""
    ql, pr = pkg("qlinear"), pkg("prompt")
    assert ql._pycalls is not None
    for module, what in ((ql, "_fp8_quant_rows"), (ql, "_fp8_gemm"), (pr, "_rope"), (pr, "_attn")):
        monkeypatch.setattr(module, what, lambda *a, **k: pytest.fail("left to the Python side"))
    fused = _randn(1, 60, 12, 64).bfloat16()
    q, k, v = fused[:, :8], fused[:, 8:10], fused[:, 10:]
    p, f, s = _i32(range(60)), pr.rope_freqs(64), _i32([0, 25, 60])
    pr.rope(q, k, p, f, out=(q, k)), pr.rope(q, k, p, f, out=(torch.empty(60, 8, 64, dtype=q.dtype, device=DEV), torch.empty(60, 2, 64, dtype=q.dtype, device=DEV))), pr.rope(q, None, p, f, out=(q, None))
    pr.attn(q, k, v, s, 1.0, out=q), pr.attn(q, k, v, s, 1.0, out=torch.empty_like(q)), pr.attn(q, k, v, s, 1.0, out=torch.empty(8, 60, 64, dtype=q.dtype, device=DEV).transpose(0, 1))
    x, r = _randn(2, 9, 256).bfloat16(), _randn(3, 9, 256).bfloat16()
    codes, xs, _ = ql.fp8_quant_rows(x, resid=r, out=r)
    ql.fp8_quant_rows(x, resid=r, out=x), ql.fp8_quant_rows(x, resid=r, out=torch.empty_like(x))
    ql.fp8_gemm(codes, torch.zeros(64, 256, device=DEV).to(E4), xs, torch.ones(1, 2, device=DEV), D=torch.empty(9, 64, device=DEV).bfloat16())
