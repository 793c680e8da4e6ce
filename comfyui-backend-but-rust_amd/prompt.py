"""What the layers of a prompt model (a text encoder, a model that writes prompts) need beside their linears: rotary positions, and attention
over whole prompts that lie one behind the other.  Single tokens behind stored ones go through kvcache.  What every call does with its tensors
stands in include/gpu_api.h.  Calls are queued on the current stream of the tensors' device and wait for nothing; there is no backward pass
and no forward mode: inputs that ask for gradients or carry tangents are refused.
"""
import math

import torch

from . import ffi, qlinear

_DT = {torch.float16: ffi.DT_F16, torch.bfloat16: ffi.DT_BF16}


def rope_freqs(rot, base=10000.0, stretch=1.0, parts=None, device="cuda:0"):
    """Radians that each of the rot / 2 pairs of channels turns per token, float64: base ** (-2 j / rot).  For contexts longer than a model was
    trained on: `stretch` divides all of them (positions interpolated); `parts` = (factor, trained length, slow, fast) divides by `factor` those
    that turn fewer than `slow` times over the trained length, leaves those that turn more than `fast` times, and blends in
    between, linearly in the turns.  (Models that blend linearly in the pair's number instead have other tables: the calls take any.)"""
    if rot <= 0 or rot % 4:
        raise ValueError("a multiple of four channels turns, not %d" % rot)
    f = torch.tensor([base ** (-2.0 * j / rot) for j in range(rot // 2)], dtype=torch.float64) / stretch
    if parts is not None:
        factor, length, slow, fast = parts
        if not fast > slow:
            raise ValueError("parts wants (factor, length, slow, fast) with fast above slow, got %r" % (parts,))
        keep = ((f * (length / (2 * math.pi)) - slow) / (fast - slow)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f.to(device)


def _heads(t, tokens, dim, what, like):
    if t.dim() != 3 or (tokens is not None and t.shape[0] != tokens) or (dim is not None and t.shape[2] != dim) or t.stride(2) != 1 or not t.is_cuda or t.device != like.device:
        raise ValueError("%s must be [%s, heads, %s] on q's CUDA device with a dense last axis, got %s with strides %s on %s"
                         % (what, "tokens" if tokens is None else tokens, "d" if dim is None else dim, tuple(t.shape), t.stride(), t.device))
    if t.dtype != like.dtype:
        raise ValueError("%s must be %s like q, got %s" % (what, like.dtype, t.dtype))
    qlinear._no_grad(t, what)


def rope(q, k, positions, freqs, interleaved=False, factor=1.0, q_norm=None, k_norm=None, eps=1e-6, out=None):
    """q [tokens, h, d] and k [tokens, hk, d] (bf16, f16 or f32, or k None) with their positions (int32 [tokens]) turned into them, as new tensors
    or into out = (q_out, k_out), which may be q and k, with their strides, and share no memory else.  The first 2 * len(freqs) channels of each head turn, in pairs of both halves or,
    interleaved, of neighbours; freqs float64: radians a token (rope_freqs).  factor scales what turns.  q_norm, k_norm (float32 [d]): each head
    is RMS-normed with that weight and eps first.  Returns (q_out, k_out)."""
    y = None if qlinear._pycalls is None else qlinear._pycalls.rope(q, k, positions, freqs, bool(interleaved), float(factor), q_norm, k_norm, float(eps), out)
    return _rope(q, k, positions, freqs, interleaved, factor, q_norm, k_norm, eps, out) if y is None else y


def _rope(q, k, positions, freqs, interleaved, factor, q_norm, k_norm, eps, out):
    """The call in Python, here and below: what the native one leaves to it, and every refusal."""
    if q.dtype not in qlinear._TORCH_DT:
        raise ValueError("q must be bfloat16, float16 or float32, got %s" % q.dtype)
    _heads(q, None, None, "q", q)
    T, h, d = q.shape
    if k is not None:
        _heads(k, T, d, "k", q)
    hk = 0 if k is None else k.shape[1]
    if positions.dtype != torch.int32 or positions.shape != (T,) or not positions.is_contiguous() or positions.device != q.device:
        raise ValueError("positions must be contiguous int32 [%d] on q's device, got %s %s on %s" % (T, positions.dtype, tuple(positions.shape), positions.device))
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous() or freqs.device != q.device:
        raise ValueError("freqs must be contiguous float64 [channels / 2] on q's device, got %s %s on %s" % (freqs.dtype, tuple(freqs.shape), freqs.device))
    qlinear._no_grad(freqs, "freqs")
    for t, what in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            if t.dtype != torch.float32 or t.shape != (d,) or not t.is_contiguous() or t.device != q.device:
                raise ValueError("%s must be contiguous float32 [%d] on q's device, got %s %s on %s" % (what, d, t.dtype, tuple(t.shape), t.device))
            qlinear._no_grad(t, what)
    if out is None:
        qo, ko = torch.empty((T, h, d), dtype=q.dtype, device=q.device), None if k is None else torch.empty((T, hk, d), dtype=q.dtype, device=q.device)
    else:
        qo, ko = out
        _heads(qo, T, d, "out[0]", q)
        qlinear._apart(qo, "out[0]")
        if qo.shape[1] != h or (ko is None) != (k is None):
            raise ValueError("out must be tensors of q's and k's shapes")
        if ko is not None:
            _heads(ko, T, d, "out[1]", q)
            qlinear._apart(ko, "out[1]")
            if ko.shape[1] != hk:
                raise ValueError("out must be tensors of q's and k's shapes")
            qlinear._separate(ko, "out[1]", (qo, q, positions, freqs, q_norm, k_norm), (k,))
        qlinear._separate(qo, "out[0]", (k, positions, freqs, q_norm, k_norm), (q,))
    side = lambda t, heads: (0, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1))
    with qlinear._on(q.device) as s:
        ffi.k("gpu_rope", qlinear._TORCH_DT[q.dtype], *side(q, h), *side(qo, h), h, *side(k, hk), *side(ko, hk), hk, positions.data_ptr(), freqs.data_ptr(), 2 * freqs.shape[0],
              1 if interleaved else 0, float(factor), qlinear._ptr(q_norm), qlinear._ptr(k_norm), float(eps), T, d, s)
    return qo, ko


def attn(q, k, v, starts, scale, causal=True, out=None):
    """softmax(scale * q k^T) v within each prompt: rows starts[s] .. starts[s + 1] (int32 [n + 1] on the device) of q [tokens, h, d] and k, v [tokens,
    hk, d] (bf16 or f16, any strides with a dense last axis, h a multiple of hk, d a multiple of 8 up to 256).  Causal: a row sees the keys up to
    its own.  A start below an earlier one counts as that one.  Returns o [tokens, h, d]; rows of no prompt are left as they are in `out`, which may be q,
    with its strides, and shares no memory with q, k and v else."""
    o = None if qlinear._pycalls is None else qlinear._pycalls.prompt_attn(q, k, v, starts, float(scale), bool(causal), out)
    return _attn(q, k, v, starts, scale, causal, out) if o is None else o


def _attn(q, k, v, starts, scale, causal, out):
    if q.dtype not in _DT:
        raise ValueError("q must be float16 or bfloat16, got %s" % q.dtype)
    _heads(q, None, None, "q", q)
    T, h, d = q.shape
    _heads(k, T, d, "k", q); _heads(v, T, d, "v", q)
    hk = k.shape[1]
    if v.shape != k.shape or hk == 0 or h == 0 or h % hk:
        raise ValueError("q [tokens, h, d] and k, v [tokens, hk, d] do not fit: %s, %s and %s" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if starts.dtype != torch.int32 or starts.dim() != 1 or starts.shape[0] == 0 or not starts.is_contiguous() or starts.device != q.device:
        raise ValueError("starts must be contiguous int32 [n + 1] on q's device, got %s %s on %s" % (starts.dtype, tuple(starts.shape), starts.device))
    o = torch.empty((T, h, d), dtype=q.dtype, device=q.device) if out is None else out
    if out is not None:
        _heads(o, T, d, "out", q)
        qlinear._apart(o, "out")
        if o.shape != q.shape:
            raise ValueError("out must be %s, got %s" % (tuple(q.shape), tuple(o.shape)))
        qlinear._separate(o, "out", (k, v, starts), (q,))
    with qlinear._on(q.device) as s:
        ffi.k("gpu_prompt_attn", _DT[q.dtype], q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), o.data_ptr(),
              o.stride(0), o.stride(1), starts.data_ptr(), starts.shape[0] - 1, T, h, hk, d, float(scale), 1 if causal else 0, s)
    return o
