"""Timed cases of attention to stored states: cross attention to an encoder's states of another length, the paged cache of keys and
values in 8 bits (stored, read back, attended), and the moving of its pages.

A case is a dict of plain values.  `kind` names the operator, the other keys its sizes and options.
"""
import importlib
import math

import torch

own = False

DEV = "cuda:0"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 16      # tokens that share a scale


def listed():
    return [
        # SDXL transformer level at 1024x1024 with guidance: image tokens to two prompts of CLIP length, the empty one shorter
        {"name": "sdxl_prompt_keys", "kind": "cross", "b": 2, "lq": 4096, "lk": 77, "h": 10, "hk": 10, "d": 64, "mask": "lens", "dtype": "f16"},
        # video DiT, 8192 tokens of 5120 channels to 512 text states, padding named by a mask
        {"name": "video_text_states", "kind": "cross", "b": 1, "lq": 8192, "lk": 512, "h": 40, "hk": 40, "d": 128, "mask": "bool", "dtype": "bf16"},
        # a few latents of an editing branch to a whole reference image of 4608 tokens, weighted by a key bias
        {"name": "image_reference_states", "kind": "cross", "b": 2, "lq": 1111, "lk": 4608, "h": 24, "hk": 24, "d": 128, "mask": "bias", "dtype": "bf16"},
        # one pooled query per image over a vision tower's states: a single row, latency counts
        {"name": "pooled_query", "kind": "cross", "b": 4, "lq": 1, "lk": 1369, "h": 16, "hk": 16, "d": 72, "mask": "none", "dtype": "f16"},
        # one token of a prompt model, one short sequence: the smallest call of the cached attention
        {"name": "token_short", "kind": "attend", "n": 1, "new": 1, "len": 613, "h": 32, "hk": 8, "d": 128, "page": 64, "causal": True, "dtype": "bf16"},
        # a batch of 12 prompts, one token each, 16 to 32 thousand tokens stored in small pages
        {"name": "token_batch", "kind": "attend", "n": 12, "new": 1, "len": 32749, "h": 32, "hk": 8, "d": 128, "page": 16, "causal": True, "dtype": "bf16"},
        # a piece of a long prompt: two sequences of about 1000 new tokens behind 7000 stored ones
        {"name": "prompt_piece", "kind": "attend", "n": 2, "new": 1024, "len": 8192, "h": 32, "hk": 8, "d": 128, "page": 64, "causal": True, "dtype": "bf16"},
        # a frame's 2000 tokens to the frames kept so far, all of them visible, head dim 64
        {"name": "frame_window", "kind": "attend", "n": 1, "new": 2025, "len": 16200, "h": 16, "hk": 16, "d": 64, "page": 128, "causal": False, "dtype": "f16"},
        # keys and values of two whole prompts into the cache, and back in 16 bits
        {"name": "store_prompts", "kind": "store", "n": 2, "new": 4096, "len": 4099, "hk": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # one token each of 64 sequences into blocks that are begun already
        {"name": "store_tokens", "kind": "store", "n": 64, "new": 1, "len": 2041, "hk": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # compaction: 160 pages of all layers move down
        {"name": "pages_compact", "kind": "pages", "layers": 28, "pages": 512, "move": 160, "hk": 8, "d": 128, "page": 64},
        # a fork writes: the shared last pages of four sequences are copied
        {"name": "pages_fork", "kind": "pages", "layers": 12, "pages": 256, "move": 4, "hk": 4, "d": 128, "page": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 6e14


def draw(rng):
    """One more case of the ranges above: any lengths and row counts, head dims and pages in the steps that the operators take."""
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("cross", "cross", "attend", "attend", "attend", "store", "pages"))
        dt = rng.choice(("bf16", "bf16", "f16"))
        if kind == "cross":
            hk = rng.randint(1, 40)
            h = hk * rng.choice((1, 1, 1, 2, 4))
            case = {"kind": kind, "b": rng.choice((1, 1, 2, 3, 4)), "lq": _log(rng, 1, 16384), "lk": _log(rng, 1, 8192), "h": h, "hk": hk,
                    "d": rng.choice((64, 128, 128, 256, 8 * rng.randint(5, 32))), "mask": rng.choice(("none", "lens", "bool", "bias")), "dtype": dt}
        elif kind == "attend":
            hk = rng.choice((1, 2, 4, 8, 8, 16, rng.randint(1, 24)))
            case = {"kind": kind, "n": _log(rng, 1, 64), "new": rng.choice((1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 4096))), "len": _log(rng, 1, 262144), "h": hk * rng.choice((1, 2, 4, 4, 7, 8)),
                    "hk": hk, "d": rng.choice((64, 128, 128, 128, 256, 16 * rng.randint(3, 16))), "page": rng.choice((16, 32, 64, 64, 128, 256)),
                    "causal": rng.random() < 0.7, "dtype": dt}
            case["len"] = max(case["len"], case["new"])
        elif kind == "store":
            case = {"kind": kind, "n": _log(rng, 1, 64), "new": rng.choice((1, _log(rng, 2, 64), _log(rng, 64, 8192))), "len": _log(rng, 1, 16384), "hk": rng.randint(1, 16),
                    "d": rng.choice((64, 128, 128, 256, 16 * rng.randint(3, 16))), "page": rng.choice((16, 32, 64, 64, 128, 256)), "dtype": dt}
            case["len"] = max(case["len"], case["new"])
        else:
            pages = _log(rng, 16, 1024)
            case = {"kind": kind, "layers": rng.randint(1, 40), "pages": pages, "move": _log(rng, 1, max(1, pages // 3)), "hk": rng.randint(1, 16),
                    "d": rng.choice((64, 128, 128, 256, 16 * rng.randint(3, 16))), "page": rng.choice((16, 32, 64, 64, 128))}
        held = case["n"] * case["len"] * case["hk"] * case["d"] if kind in ("attend", "store") else case["layers"] * case["pages"] * case["hk"] * case["page"] * case["d"] if kind == "pages" else 0
        pairs = case["b"] * case["h"] * case["lq"] * case["lk"] if kind == "cross" else case["n"] * case["h"] * case["new"] * case["len"] if kind == "attend" else 0
        if held <= 2 ** 28.6 and pairs <= 2 ** 29.2 and (kind != "attend" or case["n"] * case["h"] * case["new"] * case["d"] <= 2 ** 25) and _cost(case) <= most:
            return case


# ---- sizes that follow from a case -----------------------------------------------------------------------------------------------

def _lens(case):
    """Tokens of every sequence: from the longest down to half of it, none shorter than its new tokens."""
    return [max(_new(case)[i], case["len"] - case["len"] * i // (2 * case["n"])) for i in range(case["n"])]


def _new(case):
    """New tokens of every sequence: a little fewer from one to the next."""
    return [max(1, case["new"] - 5 * i) for i in range(case["n"])]


def _k_lens(case):
    return [max(1, case["lk"] - case["lk"] * i // (2 * case["b"])) if case["mask"] == "lens" else case["lk"] for i in range(case["b"])]


def work(case):
    if case["kind"] == "cross":
        keys, row = sum(_k_lens(case)), case["h"] * case["d"]
        return {"bytes": 4 * case["b"] * case["lq"] * row + 4 * keys * case["hk"] * case["d"], "flops": 4 * case["lq"] * keys * row}
    if case["kind"] == "attend":
        lens, new, held = _lens(case), _new(case), 2 * case["hk"] * case["d"] + case["hk"] // 2
        pairs = sum(m * l - (m * (m - 1) // 2 if case["causal"] else 0) for m, l in zip(new, lens))
        return {"bytes": sum(lens) * held + 4 * sum(new) * case["h"] * case["d"], "flops": 4 * pairs * case["h"] * case["d"]}
    if case["kind"] == "store":     # 16-bit rows in, codes out; codes in, 16-bit rows out; keys and values
        return {"bytes": 2 * sum(_new(case)) * case["hk"] * case["d"] * (2 + 1 + 1 + 2), "flops": 0}
    return {"bytes": 2 * case["layers"] * case["move"] * case["hk"] * case["page"] * (2 * case["d"] + 8 / BLOCK), "flops": 0}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------

def _channels(g, *shape):
    """Rows with channels of their own sizes, a few of them large, as keys and values of trained models have them."""
    x = torch.randn(*shape, device=DEV, generator=g)
    size = torch.exp(0.5 * torch.randn(shape[-2:], device=DEV, generator=g))
    return x * torch.where(torch.rand(shape[-2:], device=DEV, generator=g) < 0.02, 4 * size, size)


def _cache(g, pages, hk, page, d):
    """Full pages in the cache's form: codes and the largest magnitude of every 16 tokens of a head."""
    out = []
    for _ in range(2):
        codes, scales = [], []
        for at in range(0, pages, 1024):
            x = _channels(g, min(1024, pages - at) * page, hk, d).bfloat16().float().view(-1, page, hk, d).transpose(1, 2)
            x = x.reshape(-1, hk, page // BLOCK, BLOCK * d)
            a = x.abs().amax(-1, keepdim=True)
            codes.append(torch.round(x * 127 / a).to(torch.int8).view(-1, hk, page, d))
            scales.append(a.squeeze(-1).clone())
        out += [torch.cat(codes), torch.cat(scales)]
    return [out[0], out[2], out[1], out[3]]      # k, v, k_scale, v_scale


def _rows(g, case):
    """starts, lens and page table of the case's sequences, pages in no order; and the number of pages, some of them unused."""
    lens, new, page = _lens(case), _new(case), case["page"]
    need = [-(-l // page) for l in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, device=DEV, generator=g).int()
    table = torch.zeros(case["n"], max(need), dtype=torch.int32, device=DEV)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    starts = torch.tensor([sum(new[:i]) for i in range(case["n"] + 1)], dtype=torch.int32, device=DEV)
    return {"starts": starts, "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "table": table, "most": max(new), "tokens": sum(new)}, pages


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 % (1 << 62))
    kind = case["kind"]
    if kind == "pages":
        shape = (case["layers"], case["pages"], case["hk"], case["page"], case["d"])
        scales = shape[:3] + (case["page"] // BLOCK,)
        order = torch.randperm(case["pages"], device=DEV, generator=g).int()
        cache = [torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=g) for _ in range(2)]
        cache += [torch.rand(scales, device=DEV, generator=g) + 0.5 for _ in range(2)]
        return {"case": case, "cache": cache, "src": order[:case["move"]].clone(), "dst": order[case["move"]:2 * case["move"]].clone()}
    dt = _DT[case["dtype"]]
    if kind == "cross":
        b, lk = case["b"], case["lk"]
        s = {"case": case, "scale": 1.0 / math.sqrt(case["d"]), "k_lens": None, "mask": None,
             "q": (1.5 * torch.randn(b, case["lq"], case["h"], case["d"], device=DEV, generator=g)).to(dt)}
        kv = _channels(g, b, lk, 2 * case["hk"], case["d"]).to(dt)      # keys and values as one projection leaves them
        s["k"], s["v"] = kv[:, :, :case["hk"]], kv[:, :, case["hk"]:]
        if case["mask"] == "lens":
            s["k_lens"] = torch.tensor(_k_lens(case), dtype=torch.int32, device=DEV)
        elif case["mask"] == "bool":
            s["mask"] = torch.rand(b, lk, device=DEV, generator=g) < 0.8
        elif case["mask"] == "bias":
            s["mask"] = torch.randn(b, lk, device=DEV, generator=g)
        return s
    rows, pages = _rows(g, case)
    s = {"case": case, "rows": rows, "cache": _cache(g, pages, case["hk"], case["page"], case["d"]), "scale": 1.0 / math.sqrt(case["d"])}
    if kind == "attend":
        s["q"] = (1.5 * torch.randn(rows["tokens"], case["h"], case["d"], device=DEV, generator=g)).to(dt)
    else:
        s["k"], s["v"] = (1.2 * _channels(g, rows["tokens"], case["hk"], case["d"]).to(dt) for _ in range(2))
        # what is read back: the new tokens and those before them in their first block, whose codes the call may have changed
        lens, new = _lens(case), _new(case)
        back = [m + (l - m) % BLOCK for l, m in zip(lens, new)]
        starts = torch.tensor([sum(back[:i]) for i in range(len(back) + 1)], dtype=torch.int32, device=DEV)
        s["back"] = {**rows, "starts": starts, "most": max(back), "tokens": sum(back)}
    return s


# ---- the operators ---------------------------------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        pkg = "comfyui-backend-but-rust_amd"
        if kind == "cross":
            return importlib.import_module(pkg + ".qlinear").cross_attn(s["q"], s["k"], s["v"], s["scale"], s["k_lens"], s["mask"])
        kv = importlib.import_module(pkg + ".kvcache")
        cache = kv.Cache(*s["cache"])
        if kind == "attend":
            return kv.attn(s["q"], cache, _own_rows(kv, s["rows"]), s["scale"], s["case"]["causal"])
        if kind == "store":
            kv.store(cache, _own_rows(kv, s["rows"]), s["k"], s["v"])
            return kv.read(cache, _own_rows(kv, s["back"]), s["back"]["tokens"], s["k"].dtype) + (cache.k_scale, cache.v_scale)
        kv.copy_pages(cache, s["src"], s["dst"])
        return [cache.k.view(torch.int32), cache.v.view(torch.int32), cache.k_scale, cache.v_scale]
    if kind == "cross":
        return _cross(s["q"], s["k"], s["v"], s["scale"], s["k_lens"], s["mask"])
    if kind == "attend":
        return _attend(s["q"], *s["cache"], s["rows"], s["scale"], s["case"]["causal"])
    if kind == "store":
        k, v, ks, vs = s["cache"]
        _store(k, ks, s["rows"], s["k"])
        _store(v, vs, s["rows"], s["v"])
        return _read(k, ks, s["back"], s["k"].dtype), _read(v, vs, s["back"], s["k"].dtype), ks, vs
    src, dst = s["src"].long(), s["dst"].long()
    k, v, ks, vs = s["cache"]
    k[:, dst], v[:, dst], ks[:, dst], vs[:, dst] = k[:, src], v[:, src], ks[:, src], vs[:, src]
    # pages move as they are: whole words, which have to be the same
    return [k.view(torch.int32), v.view(torch.int32), ks, vs]


def _own_rows(kv, r):
    return kv.Rows(r["starts"], r["lens"], r["table"], r["most"])


def _softmax_sum(s, v):
    """softmax(s) . v over the last axis of s; rows of nothing but -inf give 0."""
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(l == 0, 1.0, l)


def _cross(q, k, v, scale, k_lens, mask):
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    qf = q.float().transpose(1, 2).reshape(b, hk, h // hk * lq, d)
    kf, vf = k.float().transpose(1, 2), v.float().transpose(1, 2)
    s = (qf @ kf.transpose(-1, -2)) * scale
    if k_lens is not None:
        mask = torch.arange(lk, device=q.device) < k_lens[:, None]
    if mask is not None:
        mask = mask[:, None, None, :]
        s = s + mask if mask.is_floating_point() else torch.where(mask, s, -math.inf)
    return _softmax_sum(s, vf).view(b, h, lq, d).transpose(1, 2).to(q.dtype).contiguous()


def _padded(rows):
    """Row of the call's tensors for every (sequence, new token) of a padded batch, which of them exist, and their positions."""
    starts, lens, most = rows["starts"].long(), rows["lens"].long(), rows["most"]
    new = starts[1:] - starts[:-1]
    i = torch.arange(most, device=starts.device)
    there = i < new[:, None]
    return torch.where(there, starts[:-1, None] + i, 0), there, (lens - new)[:, None] + i


def _values(codes, scales, table):
    """All tokens of the table's pages, [n, hk, tokens, d] in 32 bits."""
    c, s = codes[table.long()], scales[table.long()]
    n, m, hk, page, d = c.shape
    x = c.view(n, m, hk, page // BLOCK, BLOCK, d).float() * (s / 127)[..., None, None]
    return x.view(n, m, hk, page, d).transpose(1, 2).reshape(n, hk, m * page, d)


def _attend(q, k, v, ks, vs, rows, scale, causal):
    at, there, pos = _padded(rows)
    n, most = at.shape
    h, d, hk = q.shape[1], q.shape[2], k.shape[1]
    g = h // hk
    kf, vf = _values(k, ks, rows["table"]), _values(v, vs, rows["table"])
    qf = q[at].float().view(n, most, hk, g, d).permute(0, 2, 3, 1, 4).reshape(n, hk, g * most, d)
    s = ((qf @ kf.transpose(-1, -2)) * scale).view(n, hk, g, most, -1)
    t = torch.arange(s.shape[-1], device=q.device)
    seen = t < rows["lens"][:, None, None]
    if causal:
        seen = seen & (t <= pos[:, :, None])
    s = torch.where(seen[:, None, None], s, -math.inf).view(n, hk, g * most, -1)
    o = _softmax_sum(s, vf).view(n, hk, g, most, d).permute(0, 3, 1, 2, 4).reshape(n, most, h, d).to(q.dtype)
    return o[0] if n == 1 else o[there]


def _token_places(rows, page):
    """Page, slot, position and sequence of every row of the call."""
    starts, lens = rows["starts"].long(), rows["lens"].long()
    i = torch.arange(rows["tokens"], device=starts.device)
    seq = torch.searchsorted(starts, i, right=True) - 1
    pos = lens[seq] - starts[seq + 1] + i
    return rows["table"].long()[seq, pos // page], pos % page, pos, seq


def _store(codes, scales, rows, x):
    pages, hk, page, d = codes.shape
    starts, lens = rows["starts"].long(), rows["lens"].long()
    first = lens - (starts[1:] - starts[:-1])
    at, slot, pos, seq = _token_places(rows, page)
    x = x.double()
    # largest magnitude of the new tokens in every block, and with it that of the earlier ones where a block was begun
    amax = torch.zeros(pages * (page // BLOCK), hk, dtype=torch.float64, device=x.device)
    block = at * (page // BLOCK) + slot // BLOCK
    amax.scatter_reduce_(0, block[:, None].expand(-1, hk), x.abs().amax(-1), "amax")
    fp = rows["table"].long().gather(1, (first // page)[:, None]).squeeze(1)
    fb = fp * (page // BLOCK) + first % page // BLOCK
    begun = first % BLOCK
    flat = scales.transpose(1, 2).reshape(-1, hk).double()
    old = torch.where(begun[:, None] > 0, flat[fb], 0.0)
    amax[fb] = torch.maximum(amax[fb], old)
    # earlier tokens of begun blocks: their codes by the grown scale
    j = torch.arange(BLOCK, device=x.device)
    place = (first % page // BLOCK * BLOCK)[:, None] + j
    c = codes[fp[:, None], :, place].double()                                       # [n, 16, hk, d]
    a = amax[fb]
    c2 = torch.round(c * old[:, None, :, None] / torch.where(a == 0, 1.0, a)[:, None, :, None])
    codes[fp[:, None], :, place] = torch.where((j < begun[:, None])[:, :, None, None], c2, c).to(torch.int8)
    a = amax[block][:, :, None]
    codes[at, :, slot] = torch.round(x * 127 / torch.where(a == 0, 1.0, a)).to(torch.int8)
    scales[at, :, slot // BLOCK] = amax[block].float()


def _read(codes, scales, rows, dtype):
    at, slot, _, _ = _token_places(rows, codes.shape[2])
    return (codes[at, :, slot].float() * (scales[at, :, slot // BLOCK] / 127)[:, :, None]).to(dtype)


# ---- the definitions in 64 bits, sequence by sequence ----------------------------------------------------------------------------

def _tokens(codes, scales, table, length):
    page = codes.shape[2]
    t = torch.arange(length, device=codes.device)
    p = table[t // page].long()
    return codes[p, :, t % page].double() * scales[p, :, t % page // BLOCK].double()[:, :, None] / 127


def _exact_heads(q, k, v, scale, bias):
    """q [m, h, d], k and v [l, hk, d] and bias [m or 1, l], all in 64 bits -> [m, h, d], a head at a time."""
    m, h, d = q.shape
    out = torch.zeros_like(q)
    for i in range(h):
        j = i * k.shape[1] // h
        s = torch.mm(q[:, i], k[:, j].t().contiguous()) * scale + bias
        p = torch.softmax(s, -1)
        out[:, i] = torch.mm(torch.where(torch.isneginf(s).all(-1, keepdim=True), 0.0, p), v[:, j].contiguous())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "cross":
        outs = []
        for i, l in enumerate(_k_lens(case)):
            bias = torch.zeros(1, case["lk"], dtype=torch.float64, device=DEV)
            if case["mask"] == "bool":
                bias[0, ~s["mask"][i]] = -math.inf
            elif case["mask"] == "bias":
                bias[0] = s["mask"][i].double()
            outs.append(_exact_heads(s["q"][i].double(), s["k"][i, :l].double(), s["v"][i, :l].double(), s["scale"], bias[:, :l]))
        return torch.stack(outs)
    if kind == "pages":
        whole = []
        for x in s["cache"]:
            y = x.clone()
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                y[:, b] = x[:, a]
            whole.append(y.view(torch.int32) if y.dtype == torch.int8 else y.double())
        return whole
    lens, starts, table = _lens(case), s["rows"]["starts"].tolist(), s["rows"]["table"]
    k, v, ks, vs = s["cache"]
    if kind == "attend":
        outs = []
        for i, l in enumerate(lens):
            q = s["q"][starts[i]:starts[i + 1]].double()
            m = q.shape[0]
            bias = torch.zeros(1, l, dtype=torch.float64, device=DEV)
            if case["causal"]:
                late = torch.arange(l, device=DEV) > torch.arange(l - m, l, device=DEV)[:, None]
                bias = torch.zeros(m, l, dtype=torch.float64, device=DEV).masked_fill_(late, -math.inf)
            outs.append(_exact_heads(q, _tokens(k, ks, table[i], l), _tokens(v, vs, table[i], l), s["scale"], bias))
        return torch.cat(outs)
    page, back = case["page"], [[], []]
    for which, (codes, scales, x) in enumerate(((k, ks, s["k"]), (v, vs, s["v"]))):
        for i, l in enumerate(lens):
            new = x[starts[i]:starts[i + 1]].double()
            first = l - new.shape[0]
            begun = first % BLOCK
            p, slot = int(table[i, first // page]), first % page
            # the block that was begun, then the new tokens, padded to whole blocks
            a_old = scales[p, :, slot // BLOCK].double()
            head = codes[p, :, slot - begun:slot].double().transpose(0, 1)            # [begun, hk, d]
            a_head = a_old if begun else torch.zeros_like(a_old)
            size = begun + new.shape[0]
            blocks = -(-size // BLOCK)
            t = torch.zeros(blocks * BLOCK, *new.shape[1:], dtype=torch.float64, device=DEV)
            t[begun:size] = new
            a = t.view(blocks, -1, *new.shape[1:]).abs().amax((1, 3))                 # [blocks, hk]
            a[0] = torch.maximum(a[0], a_head)
            div = torch.where(a == 0, 1.0, a).repeat_interleave(BLOCK, 0)[:, :, None]
            c = torch.round(t * 127 / div)
            c[:begun] = torch.round(head * a_head[None, :, None] / div[:1])
            back[which].append((c * a.repeat_interleave(BLOCK, 0)[:, :, None] / 127)[:size])
            for j in range(blocks):
                pos = first - begun + j * BLOCK
                scales[int(table[i, pos // page]), :, pos % page // BLOCK] = a[j].float()
    return torch.cat(back[0]), torch.cat(back[1]), ks.double(), vs.double()
