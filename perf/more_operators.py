"""Timed cases of a prompt model's layer in 8-bit floating point: rows with their residual, norm and 8-bit codes, products with a scale for each
block of 128, rotary positions, and attention over packed prompts.

A case is a dict of plain values.  `kind` names the operator, the other keys its sizes and options.
"""
import importlib
import math

import torch

own = False

DEV = "cuda:0"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 128         # columns that share a scale
TOP = 448.0         # the largest e4m3 value
LEAST = 2.0 ** -100  # a group's largest magnitude counts as this at least
EPS = 1e-6


def listed():
    return [
        # one token between two blocks: the residual's addition, the norm and the codes for the next product; latency counts
        {"name": "norm_token", "kind": "rows", "what": "norm", "m": 1, "k": 4096, "dtype": "bf16"},
        # the same for a whole batch of prompts
        {"name": "norm_prompts", "kind": "rows", "what": "norm", "m": 8192, "k": 4096, "dtype": "bf16"},
        # gate and up halves of an MLP become the codes of its down product
        {"name": "gate_prompts", "kind": "rows", "what": "gate", "m": 4099, "k": 12288, "dtype": "f16"},
        # five tokens through the gate and up product: the weights' way in is all that counts
        {"name": "linear_tokens", "kind": "linear", "m": 5, "n": 24576, "k": 4096, "bias": False, "dtype": "bf16"},
        # one short prompt through the down product
        {"name": "linear_prompt", "kind": "linear", "m": 256, "n": 4096, "k": 12288, "bias": False, "dtype": "bf16"},
        # a head of odd sizes in 32 bits with a bias; the last group of columns is not a whole one
        {"name": "linear_ragged", "kind": "linear", "m": 1111, "n": 1000, "k": 2640, "bias": True, "dtype": "f32"},
        # the gate and up product of a batch of prompts
        {"name": "linear_prompts", "kind": "linear", "m": 8192, "n": 24576, "k": 4096, "bias": False, "dtype": "bf16"},
        # one token of each of twelve sequences, at far positions
        {"name": "rope_tokens", "kind": "rope", "t": 12, "h": 32, "hk": 8, "d": 128, "rot": 128, "inter": False, "stretch": 1.0, "far": 1 << 20, "dtype": "bf16"},
        # long prompts, half of each head rotated in neighbouring pairs, positions stretched by four
        {"name": "rope_prompts", "kind": "rope", "t": 16384, "h": 32, "hk": 8, "d": 128, "rot": 64, "inter": True, "stretch": 4.0, "far": 16384, "dtype": "bf16"},
        # 48 captions of a text encoder with small heads, from one token to 231
        {"name": "attn_captions", "kind": "attn", "n": 48, "len": 231, "h": 20, "hk": 20, "d": 64, "dtype": "f16"},
        # five prompts of 800 to 4000 tokens, four query heads to a key-value head
        {"name": "attn_prompts", "kind": "attn", "n": 5, "len": 4000, "h": 32, "hk": 8, "d": 128, "dtype": "bf16"},
        # one document of 16 thousand tokens
        {"name": "attn_document", "kind": "attn", "n": 1, "len": 16384, "h": 16, "hk": 4, "d": 128, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 1e15


def draw(rng):
    """One more case of the ranges above: any row counts and lengths, columns and head dims in the steps that the operators take."""
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("rows", "linear", "linear", "linear", "rope", "attn", "attn", "attn"))
        dt = rng.choice(("bf16", "bf16", "f16"))
        if kind == "rows":
            case = {"kind": kind, "what": rng.choice(("norm", "norm", "gate", "plain")), "m": _log(rng, 1, 16384), "k": 16 * _log(rng, 8, 1024), "dtype": dt}
        elif kind == "linear":
            k = rng.choice((128 * _log(rng, 2, 128), 128 * _log(rng, 2, 128), 16 * _log(rng, 16, 512)))
            case = {"kind": kind, "m": rng.choice((_log(rng, 1, 64), _log(rng, 1, 16384))), "n": rng.choice((128 * _log(rng, 4, 224), 8 * _log(rng, 16, 2048), _log(rng, 100, 9999))), "k": k,
                    "bias": rng.random() < 0.3, "dtype": rng.choice((dt, dt, dt, "f32"))}
        elif kind == "rope":
            hk, d = rng.randint(1, 16), rng.choice((64, 128, 128, 256, 8 * rng.randint(4, 32)))
            case = {"kind": kind, "t": _log(rng, 1, 32768), "h": hk * rng.choice((1, 2, 4, 4, 7, 8)), "hk": hk, "d": d, "rot": rng.choice((d, d, d // 2, 8 * rng.randint(1, d // 8))),
                    "inter": rng.random() < 0.5, "stretch": rng.choice((1.0, 1.0, 4.0, 32.0)), "far": _log(rng, 1000, 1 << 21), "dtype": dt}
            case["rot"] -= case["rot"] % 2
        else:
            hk = rng.choice((1, 2, 4, 8, 8, rng.randint(1, 24)))
            case = {"kind": kind, "n": _log(rng, 1, 64), "len": _log(rng, 1, 16384), "h": hk * rng.choice((1, 1, 2, 4, 4, 7, 8)), "hk": hk,
                    "d": rng.choice((64, 128, 128, 128, 256, 8 * rng.randint(5, 32))), "dtype": dt}
            if case["n"] * case["h"] * case["len"] ** 2 > 2 ** 32.1 or case["n"] * case["h"] * case["len"] * case["d"] > 2 ** 28:
                continue
        if _cost(case) <= most:
            return case


# ---- sizes that follow from a case -----------------------------------------------------------------------------------------------

def _groups(k):
    return -(-k // GROUP)


def _lens(case):
    """Tokens of every prompt: from the longest down to a fifth of it, the last of many a single token."""
    n, l = case["n"], case["len"]
    return [max(1, l - (4 * l * i // (5 * max(1, n - 1)))) if i < n - 1 or n < 8 else 1 for i in range(n)]


def work(case):
    if case["kind"] == "rows":
        a = {"norm": 7, "gate": 5, "plain": 3}[case["what"]]
        return {"bytes": case["m"] * (a * case["k"] + 4 * _groups(case["k"])) + (4 * case["k"] if case["what"] == "norm" else 0), "flops": 0}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": m * k + n * k + 4 * _groups(k) * (m + _groups(n)) + size * (m * n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    if case["kind"] == "rope":
        return {"bytes": 4 * case["t"] * (case["h"] + case["hk"]) * case["d"] + 4 * case["t"] + 4 * case["rot"], "flops": 0}
    lens = _lens(case)
    pairs = sum(l * (l + 1) // 2 for l in lens)
    return {"bytes": 4 * sum(lens) * (case["h"] + case["hk"]) * case["d"], "flops": 4 * pairs * case["h"] * case["d"]}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------

def _channels(g, *shape):
    """Rows with channels of their own sizes, a few of them large, as hidden states, keys and values of trained models have them."""
    x = torch.randn(*shape, device=DEV, generator=g)
    size = torch.exp(0.5 * torch.randn(shape[-1:], device=DEV, generator=g))
    return x * torch.where(torch.rand(shape[-1:], device=DEV, generator=g) < 0.02, 6 * size, size)


def _codes(x):
    """Codes and scales of x [m, k] in 32 bits, a scale for each group of columns of a row: [m, k] e4m3 and [groups, m]."""
    m, k = x.shape
    g = _groups(k)
    x = torch.nn.functional.pad(x, (0, g * GROUP - k)).view(m, g, GROUP)
    a = x.abs().amax(-1, keepdim=True).clamp(min=LEAST)
    q = (x * (TOP / a)).to(torch.float8_e4m3fn).view(m, g * GROUP)[:, :k].contiguous()
    return q, (a.squeeze(-1) / TOP).t().contiguous()


def _weights(g, n, k):
    """Codes and scales of a weight: a scale for each block of 128 x 128."""
    nb, kb = _groups(n), _groups(k)
    w = torch.randn(nb * GROUP, kb * GROUP, device=DEV, generator=g) * (k ** -0.5) * torch.exp(0.3 * torch.randn(nb * GROUP, 1, device=DEV, generator=g))
    w[n:], w[:, k:] = 0, 0
    b = w.view(nb, GROUP, kb, GROUP)
    a = b.abs().amax((1, 3), keepdim=True).clamp(min=LEAST)
    q = (b * (TOP / a)).to(torch.float8_e4m3fn).view(nb * GROUP, kb * GROUP)[:n, :k].contiguous()
    return q, (a / TOP).view(nb, kb).clone()


def _freqs(case):
    """Radians a token for every pair of channels, as a program keeps them: a base of 10000, positions stretched."""
    j = torch.arange(case["rot"] // 2, dtype=torch.float64, device=DEV)
    return 10000.0 ** (-2.0 * j / case["rot"]) / case["stretch"]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 % (1 << 62))
    kind, dt = case["kind"], _DT[case["dtype"]]
    if kind == "rows":
        m, k = case["m"], case["k"]
        s = {"case": case, "x": _channels(g, m, 2 * k if case["what"] == "gate" else k).to(dt)}
        if case["what"] == "norm":
            s["resid"] = (4 * _channels(g, m, k)).to(dt)
            s["w"] = 1 + 0.2 * torch.randn(k, device=DEV, generator=g)
        return s
    if kind == "linear":
        a, xs = _codes(_channels(g, case["m"], case["k"]))
        w, ws = _weights(g, case["n"], case["k"])
        return {"case": case, "a": a, "xs": xs, "w": w, "ws": ws, "bias": torch.randn(case["n"], device=DEV, generator=g).to(dt) if case["bias"] else None}
    h, hk, d = case["h"], case["hk"], case["d"]
    t = case["t"] if kind == "rope" else sum(_lens(case))
    # queries, keys and values as one projection leaves them
    qkv = _channels(g, t, (h + 2 * hk) * d).to(dt).view(t, h + 2 * hk, d)
    s = {"case": case, "q": qkv[:, :h], "k": qkv[:, h:h + hk], "v": qkv[:, h + hk:]}
    if kind == "rope":
        s["positions"] = torch.randint(0, case["far"], (t,), dtype=torch.int32, device=DEV, generator=g) if t < 64 else \
            torch.arange(t, dtype=torch.int32, device=DEV) % case["far"] + torch.randint(0, 64, (1,), dtype=torch.int32, device=DEV, generator=g)
        s["freqs"] = _freqs(case)
    else:
        lens = _lens(case)
        s["starts"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
        s["most"], s["scale"] = max(lens), 1.0 / math.sqrt(d)
    return s


# ---- the operators ---------------------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        pkg = "comfyui-backend-but-rust_amd"
        if kind in ("rows", "linear"):
            ql = importlib.import_module(pkg + ".qlinear")
            if kind == "linear":
                return ql.fp8_gemm(s["a"], s["w"], s["xs"], s["ws"], s["bias"], _DT[case["dtype"]])
            if case["what"] == "norm":
                return ql.fp8_quant_rows(s["x"], "rms", norm_w=s["w"], eps=EPS, resid=s["resid"])
            return ql.fp8_quant_rows(s["x"], "swiglu" if case["what"] == "gate" else "plain")
        prompt = importlib.import_module(pkg + ".prompt")
        if kind == "rope":
            return prompt.rope(s["q"], s["k"], s["positions"], s["freqs"], case["inter"])
        return prompt.attn(s["q"], s["k"], s["v"], s["starts"], s["scale"])
    if kind == "rows":
        return _rows(case, s["x"], s.get("resid"), s.get("w"))
    if kind == "linear":
        return _linear(s["a"], s["w"], s["xs"], s["ws"], s["bias"], _DT[case["dtype"]])
    if kind == "rope":
        return _rope(s["q"], s["k"], s["positions"], s["freqs"], case["inter"])
    return _attn(s["q"], s["k"], s["v"], s["starts"], s["most"], s["scale"])


def _rows(case, x, resid, w):
    if case["what"] == "norm":
        total = (x.float() + resid.float()).to(x.dtype)
        f = total.float()
        return _codes(f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * w) + (total,)
    if case["what"] == "gate":
        gate, up = x[:, :case["k"]].float(), x[:, case["k"]:].float()
        return _codes(gate / (1 + torch.exp(-gate)) * up)
    return _codes(x.float())


def _linear(a, w, xs, ws, bias, dtype):
    n, k = w.shape
    af = a.float() * xs.t().repeat_interleave(GROUP, 1)[:, :k]
    wf = w.float() * ws.repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    d = af @ wf.t()
    return (d if bias is None else d + bias.float()).to(dtype)


def _turned(x, cos, sin, inter):
    r = 2 * cos.shape[-1]
    f = x[..., :r].float()
    a, b = (f[..., 0::2], f[..., 1::2]) if inter else (f[..., :r // 2], f[..., r // 2:])
    a, b = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)
    return torch.cat((y.to(x.dtype), x[..., r:]), -1)


def _rope(q, k, positions, freqs, inter):
    angle = positions.double()[:, None, None] * freqs       # far positions need 64 bits
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    return _turned(q, cos, sin, inter), _turned(k, cos, sin, inter)


def _attn(q, k, v, starts, most, scale):
    n, h, d, hk = starts.shape[0] - 1, q.shape[1], q.shape[2], k.shape[1]
    starts = starts.long()
    i = torch.arange(most, device=q.device)
    there = i < (starts[1:] - starts[:-1])[:, None]
    at = torch.where(there, starts[:-1, None] + i, 0)
    qf = q[at].float().view(n, most, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, h // hk * most, d)
    kf, vf = k[at].float().transpose(1, 2), v[at].float().transpose(1, 2)
    s = ((qf @ kf.transpose(-1, -2)) * scale).view(n, hk, h // hk, most, most)
    s = torch.where(i <= i[:, None], s, -math.inf).view(n, hk, -1, most)    # (a row behind a prompt's end is not taken)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = (p @ vf) / p.sum(-1, keepdim=True)
    o = o.view(n, hk, h // hk, most, d).permute(0, 3, 1, 2, 4).reshape(n, most, h, d).to(q.dtype)
    return o[there]


# ---- the definitions in 64 bits, group by group and prompt by prompt -------------------------------------------------------------

def _e4m3(x):
    """x in 64 bits, rounded to the nearest value of 4 bits of exponent and 3 of fraction, ties to even."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rows":
        x, k, total = s["x"].double(), case["k"], None
        if case["what"] == "norm":
            total = (x + s["resid"].double()).to(s["x"].dtype).double()
            n = total / torch.sqrt((total * total).sum(1, keepdim=True) / k + EPS) * s["w"].double()
        elif case["what"] == "gate":
            n = torch.nn.functional.silu(x[:, :k]) * x[:, k:]
        else:
            n = x
        codes, scales = [], []
        for part in n.split(GROUP, 1):
            a = part.abs().max(1).values.clamp(min=LEAST)
            codes.append(_e4m3(part / a[:, None] * TOP))
            scales.append(a / TOP)
        out = (torch.cat(codes, 1), torch.stack(scales))
        return out if total is None else out + (total,)
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        d = torch.zeros(m, n, dtype=torch.float64, device=DEV)
        for g in range(_groups(k)):
            at = slice(g * GROUP, (g + 1) * GROUP)
            part = torch.mm(s["a"][:, at].double(), s["w"][:, at].double().t().contiguous())
            part *= s["xs"][g].double()[:, None]
            part *= s["ws"][:, g].double()[torch.arange(n, device=DEV) // GROUP]
            d += part
        return d if s["bias"] is None else d + s["bias"].double()
    if kind == "rope":
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["positions"].double()[:, None] * s["freqs"])[:, None]
        r, out = case["rot"], []
        for x in (s["q"].double(), s["k"].double()):
            first, second = (x[..., 0:r:2], x[..., 1:r:2]) if case["inter"] else (x[..., :r // 2], x[..., r // 2:r])
            z = torch.complex(first.contiguous(), second.contiguous()) * turn
            y = x.clone()
            if case["inter"]:
                y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
            else:
                y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
            out.append(y)
        return tuple(out)
    q, k, v, at = s["q"], s["k"], s["v"], s["starts"].tolist()
    o = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for b, e in zip(at[:-1], at[1:]):
        late = torch.ones(e - b, e - b, dtype=torch.bool, device=DEV).triu_(1)
        for i in range(case["h"]):
            j = i * case["hk"] // case["h"]
            x = torch.mm(q[b:e, i].double(), k[b:e, j].double().t().contiguous()) * s["scale"]
            o[b:e, i] = torch.mm(torch.softmax(x.masked_fill_(late, -math.inf), -1), v[b:e, j].double().contiguous())
    return o
