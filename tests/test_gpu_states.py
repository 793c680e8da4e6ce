"""Attention to stored states on the GPU against the formulas in 64 bits: cross attention, and the paged cache of 8-bit keys and values
(stored, read back, attended, its pages moved).

The cache's codes and scales are whole-number work and must be equal.  Attention outputs are held to bounds that count roundings, each off by at
most half a step u (bf16 2^-8, f16 2^-11, fp32 2^-24 relative to the value):
  the output's rounding                              u_out |o|, or half the type's smallest step (f16: 2^-25) where that is more
  probabilities, rounded for the product with V      u_p sum p |v| / sum p
  ... in f16, where they are subnormal               n 2^-34 max_j p_j A_j / sum p: they are held in units of 2^-9 times a base that is at most the
                                                     largest p_j A_j, A_j the magnitude that the kernel counts into p (1, or the block's), and
                                                     round by 2^-25 of a unit; the cache's sum takes them rounded where no A is below 1/16 of
                                                     the largest: n 2^-30 of the sum
  scores, fp32 sums of d products in any order       |dx| <= (d + 8) 2^-24 (scale max_j sum_i |q_i k_ji| + |bias|) in the exponent, in numerator
                                                     and denominator: 2 |dx| sum p |v| / sum p; exp2 itself 2^-22 likewise
  the sums over n keys                               (n + 8) 2^-23 sum p |v| / sum p
"""
import math

import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _reference(q, k, v, scale, keep, bias, u_p, u_out, tiny):
    """One head in 64 bits: q [m, d], k, v [l, d], keep bool [m, l], bias [l] -> (o, bound), both [m, d].  tiny: the
    A_j of f16 probabilities, or None."""
    q, k, v = q.double(), k.double(), v.double()
    keep = keep & ~torch.isneginf(bias)
    k, v = (torch.where(keep.any(0)[:, None], t, 0.0) for t in (k, v))     # a key that nobody sees may hold anything
    s = torch.where(keep, (q @ k.t().contiguous()) * scale + bias, -math.inf)
    m = s.amax(-1, keepdim=True) if k.shape[0] else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64, device=q.device)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    l = p.sum(-1, keepdim=True)
    some = l > 0
    l = torch.where(some, l, 1.0)
    o = (p @ v) / l
    mass = (p @ v.abs()) / l
    size = torch.where(keep, q.abs() @ k.abs().t().contiguous() * abs(scale), 0.0)
    if k.shape[0]:
        size = size.amax(-1, keepdim=True) + torch.where(torch.isinf(bias), 0.0, bias.abs().clamp(max=1e4)).max()
    d, n = q.shape[1], k.shape[0]
    dx = (d + 8) * 2.0 ** -24 * size + 2.0 ** -22 if n else 0.0
    low = n * (2.0 ** -34 * (p * tiny).amax(-1, keepdim=True) / l + 2.0 ** -30 * mass) if n and tiny is not None else 0.0
    return o, (u_out * o.abs()).clamp(min=2.0 ** -25 if u_out == U[torch.float16] else 0.0) + (u_p + 2 * dx + (n + 8) * 2.0 ** -23) * mass + low + 1e-30


def _check(got, want, bound, what):
    off = (got.double() - want).abs() / bound
    assert not torch.isnan(got).any(), what
    assert off.max().item() <= 1.0 if off.numel() else True, "%s: %.3g of the bound at %s" % (what, off.max().item(), off.argmax().item())


# ---- cross attention -------------------------------------------------------------------------------------------------------------

def _cross_inputs(b, lq, lk, h, hk, d, dtype, seed):
    g = _gen(seed)
    return [(f * torch.randn(b, n, m, d, device=DEV, generator=g)).to(dtype) for f, n, m in ((1.5, lq, h), (1.0, lk, hk), (1.0, lk, hk))]


def _cross_check(o, q, k, v, scale, k_lens=None, mask=None, what=""):
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    for i in range(b):
        keep = torch.ones(lq, lk, dtype=torch.bool, device=DEV)
        bias = torch.zeros(lk, dtype=torch.float64, device=DEV)
        if k_lens is not None:
            keep &= torch.arange(lk, device=DEV) < int(k_lens[i])
        if mask is not None:
            row = mask if mask.dim() == 1 else mask[i]
            if row.dtype == torch.bool:
                keep &= row
            else:
                bias = row.double()
        for j in range(h):
            want, bound = _reference(q[i, :, j], k[i, :, j * hk // h], v[i, :, j * hk // h], scale, keep, bias, U[q.dtype], U[q.dtype], v.double().nan_to_num(0, 0, 0).abs().max() if q.dtype == torch.float16 and lk else None)
            _check(o[i, :, j], want, bound, "%s item %d head %d" % (what, i, j))


CROSS = [(1, 1, 1, 1, 1, 8), (2, 1, 300, 4, 4, 64), (1, 3, 77, 6, 2, 128), (2, 33, 64, 2, 2, 72), (1, 130, 65, 3, 1, 128), (2, 200, 129, 4, 4, 64),
         (1, 257, 513, 2, 2, 256), (1, 7, 2000, 8, 1, 160), (3, 128, 1, 2, 1, 40), (1, 1, 5003, 2, 2, 128), (1, 300, 3000, 2, 1, 64), (2, 32, 95, 1, 1, 248),
         (1, 1, 4099, 5, 1, 200), (1, 45, 1030, 2, 2, 16), (1, 2, 31, 64, 2, 24), (1, 20, 60, 1, 1, 64),
         (1, 24, 3000, 1, 1, 64), (2, 20, 60, 1, 1, 128), (1, 24, 3000, 1, 1, 96), (1, 130, 3000, 1, 1, 128), (1, 200, 1010, 2, 2, 64), (1, 257, 1000, 1, 1, 128),
         (1, 150, 20000, 1, 1, 64), (1, 150, 20000, 1, 1, 128),
         (1, 60, 65, 1, 1, 96), (1, 70, 3000, 1, 1, 72), (2, 257, 1000, 1, 1, 88), (1, 150, 20000, 1, 1, 80), (1, 20, 60, 1, 1, 72), (1, 9, 60, 1, 1, 192), (1, 5, 3000, 2, 2, 136), (1, 60, 70, 2, 2, 168), (1, 60, 3000, 1, 1, 256), (1, 257, 1000, 1, 1, 144), (1, 150, 20000, 1, 1, 176),
         (1, 300, 70, 86, 86, 248), (1, 130, 2050, 65, 65, 240), (1, 33, 200, 260, 260, 16),
         (1, 1030, 2050, 86, 86, 64), (1, 130, 20000, 65, 65, 48), (1, 8200, 1030, 3, 3, 96), (1, 130, 4100, 86, 86, 128), (1, 130, 1030, 129, 129, 112),
         (1, 8200, 600, 3, 3, 192), (1, 130, 70, 1, 1, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("shape", CROSS, ids=lambda s: "x".join(map(str, s)))
def test_cross_attn(shape, dtype):
    ql = pkg("qlinear")
    q, k, v = _cross_inputs(*shape, dtype, 1)
    b, lk, d = shape[0], shape[2], shape[5]
    scale = d ** -0.5
    _cross_check(ql.cross_attn(q, k, v, scale), q, k, v, scale, what="plain")
    lens = torch.tensor([(lk * (i + 1)) // 2 for i in range(b)], dtype=torch.int32, device=DEV)
    _cross_check(ql.cross_attn(q, k, v, scale, lens), q, k, v, scale, lens, what="lengths")
    keep = torch.rand(b, lk, device=DEV, generator=_gen(2)) < 0.6
    _cross_check(ql.cross_attn(q, k, v, scale, None, keep), q, k, v, scale, None, keep, what="mask")
    bias = torch.where(torch.rand(b, lk, device=DEV, generator=_gen(3)) < 0.2, -math.inf, 2 * torch.randn(b, lk, device=DEV, generator=_gen(4)))
    _cross_check(ql.cross_attn(q, k, v, -scale, lens, bias), q, k, v, -scale, lens, bias, what="bias, lengths and a negative scale")
    _cross_check(ql.cross_attn(q, k, v, 0.0, lens, bias), q, k, v, 0.0, lens, bias, what="no scale")
    tiny = torch.randn(b, lk, device=DEV, generator=_gen(5))
    _cross_check(ql.cross_attn(q, k, v, 1e-36, None, tiny), q, k, v, 1e-36, None, tiny, what="next to no scale")
    _cross_check(ql.cross_attn(q, k, v, 1e-36), q, k, v, 1e-36, what="next to no scale, no bias")


@pytest.mark.parametrize("lq", [1, 40, 150])
def test_cross_attn_rows_without_keys_and_extreme_masks(lq):
    """Lengths of zero and beyond lk; masks that leave nothing; a bias of the type's lowest value is a logit like any other; what a key that is
    out holds does not matter."""
    ql = pkg("qlinear")
    q, k, v = _cross_inputs(4, lq, 130, 2, 1, 64, torch.bfloat16, 5)
    lens = torch.tensor([0, 1, 500, -3], dtype=torch.int32, device=DEV)
    o = ql.cross_attn(q, k, v, 0.125, lens)
    _cross_check(o, q, k, v, 0.125, lens.clamp(0, 130), what="lengths")
    assert not o[0].any() and not o[3].any()
    keep = torch.rand(4, 130, device=DEV, generator=_gen(6)) < 0.5
    keep[1] = False
    keep[2], keep[2, 129] = False, True
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[~keep], bad_v[~keep] = math.nan, math.inf
    o = ql.cross_attn(q, bad_k, bad_v, 0.125, None, keep)
    _cross_check(o, q, k, v, 0.125, None, keep, what="mask over NaN")
    assert not o[1].any()
    lens = torch.tensor([7, 64, 65, 0], dtype=torch.int32, device=DEV)
    for i, n in enumerate(lens.tolist()):
        bad_k[i], bad_v[i] = k[i], v[i]
        bad_k[i, n:], bad_v[i, n:] = math.inf, math.nan
    _cross_check(ql.cross_attn(q, bad_k, bad_v, 0.125, lens), q, k, v, 0.125, lens, what="lengths before NaN")
    low = torch.finfo(torch.float32).min
    bias = torch.zeros(4, 130, device=DEV)
    bias[0] = low
    bias[1], bias[1, 3] = low, 0.0
    bias[2, ::2] = low
    bias[3] = -math.inf
    o = ql.cross_attn(q, k, v, 0.125, None, bias)
    want = v[0].double().mean(0)     # |s| is lost beside the lowest value: all keys alike
    assert (o[0].double() - want).abs().max() <= 2 * U[torch.bfloat16] * v[0].double().abs().mean(0).max()
    _cross_check(o[1:2], q[1:2], k[1:2], v[1:2], 0.125, torch.tensor([130]), torch.arange(130, device=DEV) == 3, what="lowest value")
    _cross_check(o[2:3], q[2:3], k[2:3], v[2:3], 0.125, None, torch.arange(130, device=DEV) % 2 == 1, what="lowest value")
    assert not o[3].any()


def test_cross_attn_not_finite_where_the_formula_is_not():
    ql = pkg("qlinear")
    q, k, v = _cross_inputs(1, 40, 100, 2, 2, 64, torch.float16, 7)
    q[0, 3, 0, 5] = math.nan
    k[0, 50, 1, 0] = math.nan
    o = ql.cross_attn(q, k, v, 0.125)
    assert torch.isnan(o[0, 3, 0]).all() and torch.isnan(o[0, :, 1]).all()
    rest = torch.arange(40, device=DEV) != 3
    assert torch.isfinite(o[0, rest, 0]).all()


@pytest.mark.parametrize("lq,lk", [(1, 700), (5, 64), (200, 333)])
def test_cross_attn_strides(lq, lk):
    """Operands inside larger tensors, in other orders, off 16 bytes, one key-value item for all of the batch."""
    ql = pkg("qlinear")
    g = _gen(8)
    b, h, d = 2, 3, 64
    fused = torch.randn(b, lk, 2, h, d + 8, device=DEV, generator=g).half()
    k, v = fused[:, :, 0, :, 4:4 + d], fused[:, :, 1, :, 4:4 + d]
    q = torch.randn(b, h, lq, d, device=DEV, generator=g).half().transpose(1, 2)
    keep = (torch.rand(lk, 2 * b, device=DEV, generator=g) < 0.7).t().contiguous()[::2]
    _cross_check(ql.cross_attn(q, k, v, 0.1, None, keep), q, k, v, 0.1, None, keep, what="slices")
    odd = torch.randn(1 + b * lq * h * d, device=DEV, generator=g).half()[1:].view(b, lq, h, d)
    odd_k = torch.randn(b * lk * h * (d + 1), device=DEV, generator=g).half().view(b, lk, h, d + 1)[..., 1:]
    _cross_check(ql.cross_attn(odd, odd_k, v, 0.1), odd, odd_k, v, 0.1, what="off 16 bytes")
    one_k, one_v = (t[:1].expand(b, -1, -1, -1) for t in (k, v))
    bias = torch.randn(lk, device=DEV, generator=g)
    _cross_check(ql.cross_attn(q, one_k, one_v, 0.1, None, bias), q, one_k, one_v, 0.1, None, bias, what="shared keys")


def test_cross_attn_empty_sizes():
    ql = pkg("qlinear")
    for b, lq, lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = _cross_inputs(b, lq, lk, 2, 1, 64, torch.bfloat16, 9)
        o = ql.cross_attn(q, k, v, 0.125)
        assert o.shape == q.shape and not o.any()


# ---- the cache -------------------------------------------------------------------------------------------------------------------

class Model:
    """The cache in 64 bits, token by token: what it must hold."""

    def __init__(self, heads, dim, seqs):
        self.codes = [[torch.zeros(heads, 0, dim, dtype=torch.float64) for _ in range(2)] for _ in range(seqs)]
        self.amax = [[torch.zeros(heads, 0, dtype=torch.float64) for _ in range(2)] for _ in range(seqs)]

    def append(self, s, k, v):
        if not k.shape[0]:
            return
        for w, x in enumerate((k, v)):
            x = x.double().cpu().transpose(0, 1)               # [heads, new, dim]
            c, a = self.codes[s][w], self.amax[s][w]
            n0, n1 = c.shape[1], c.shape[1] + x.shape[1]
            c = torch.cat([c, torch.zeros_like(x)], 1)
            blocks = -(-n1 // 16)
            a = torch.cat([a, torch.zeros(a.shape[0], blocks - a.shape[1], dtype=torch.float64)], 1)
            for b in range(n0 // 16, blocks):
                lo, hi = max(n0, 16 * b), min(n1, 16 * b + 16)
                old = a[:, b] if lo > 16 * b else torch.zeros_like(a[:, b])
                new = torch.maximum(old, x[:, lo - n0:hi - n0].abs().amax((1, 2)))
                div = torch.where(new == 0, 1.0, new)[:, None, None]
                c[:, 16 * b:lo] = torch.round(c[:, 16 * b:lo] * old[:, None, None] / div)
                c[:, lo:hi] = torch.round(x[:, lo - n0:hi - n0] * 127 / div)
                a[:, b] = new
            self.codes[s][w], self.amax[s][w] = c, a

    def values(self, s, w):
        """[tokens, heads, dim]"""
        c, a = self.codes[s][w], self.amax[s][w]
        return (c * a.repeat_interleave(16, 1)[:, :c.shape[1], None] / 127).transpose(0, 1).to(DEV)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _table(lens, page, pages, seed, cols=None):
    """Pages of the sequences in no order, the rest of every row a page of somebody else's."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    need = [-(-l // page) for l in lens]
    assert sum(need) <= pages
    t = torch.full((len(lens), cols or max(need + [1])), order[-1], dtype=torch.int32)
    for i, m in enumerate(need):
        for j in range(m):
            t[i, j] = order.pop(0)
    return t.to(DEV)


def _rows(kv, new, lens, table):
    return kv.Rows(_i32([sum(new[:i]) for i in range(len(new) + 1)]), _i32(lens), table, max(new + [0]))


def _filled(lens, heads, dim, page, seed, dtype=torch.bfloat16, size=1.0):
    """A cache with the sequences stored in one call, and the model of it."""
    kv = pkg("kvcache")
    pages = sum(-(-l // page) for l in lens) + 2
    cache = kv.new_cache(pages, heads, dim, page)
    for t in cache:
        t.fill_(7)      # nothing may depend on what a page held
    table = _table(lens, page, pages, seed)
    g = _gen(seed)
    k, v = ((size * torch.randn(sum(lens), heads, dim, device=DEV, generator=g)).to(dtype) for _ in range(2))
    rows = _rows(kv, lens, lens, table)
    kv.store(cache, rows, k, v)
    model, at = Model(heads, dim, len(lens)), 0
    for s, l in enumerate(lens):
        model.append(s, k[at:at + l], v[at:at + l])
        at += l
    return cache, table, model


def _same_cache(kv, cache, table, lens, model):
    k, v = kv.read(cache, _rows(kv, lens, lens, table), sum(lens), torch.float32)
    at = 0
    for s, l in enumerate(lens):
        for w, got in enumerate((k, v)):
            want = model.values(s, w)
            off = (got[at:at + l].double() - want).abs()
            # code * fl(A / 127): three roundings of 2^-24; a code that differs by one is 2^17 times that off
            assert bool((off <= 4 * 2.0 ** -24 * want.abs()).all()), (s, "kv"[w], off.max().item())
        at += l


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("heads,dim,page", [(1, 16, 16), (3, 64, 32), (2, 80, 64), (8, 128, 64), (2, 256, 16), (5, 208, 128)])
def test_store_and_read(heads, dim, page, dtype):
    """Whole prompts, then pieces of many lengths behind them: codes and scales are those of the definition."""
    kv = pkg("kvcache")
    final = [page * 3 + 5, 16, 100, 1]
    pages = sum(-(-l // page) for l in final) + 2
    cache, table = kv.new_cache(pages, heads, dim, page), _table(final, page, pages, 3)
    model, held, g = Model(heads, dim, 4), [0, 0, 0, 0], _gen(4)
    for step, new in enumerate(([7, 16, 33, 0], [1, 0, 1, 1], [1, 0, 1, 0], [20, 0, 17, 0], [final[0] - 29, 0, 48, 0])):
        rows = [(torch.randn(n, heads, dim, device=DEV, generator=g) * 4.0 ** (step - 1)).to(dtype) for n in new for _ in range(2)]
        held = [a + b for a, b in zip(held, new)]
        kv.store(cache, _rows(kv, new, held, table), torch.cat(rows[::2]), torch.cat(rows[1::2]))
        for s in range(4):
            if new[s]:
                model.append(s, rows[2 * s], rows[2 * s + 1])
        _same_cache(kv, cache, table, held, model)
    assert held == final


def test_store_ties_and_ends_of_the_range():
    """Quotients that lie between two codes, blocks of zeros, the largest and the smallest values of the types."""
    kv = pkg("kvcache")
    for dtype, big in ((torch.bfloat16, 3.38e38), (torch.float16, 65504.0)):
        f = torch.finfo(dtype)
        x = torch.zeros(96, 1, 64, dtype=dtype)
        x[:16] = (torch.arange(16 * 64).view(16, 1, 64) % 257 - 128) / 128           # A = 1: x * 127 ends in .5 for half of them
        x[16:32] = torch.tensor([big, -big, big / 3, 1.0])[torch.arange(64) % 4]
        x[48:64] = torch.tensor([f.smallest_normal, -f.smallest_normal / 2, f.smallest_normal / 4, 0.0])[torch.arange(64) % 4]
        x[64:80] = torch.randn(16, 1, 64, generator=torch.Generator().manual_seed(1)) * f.smallest_normal / 4
        x[80:] = torch.tensor([127.0, 63.5, 0.5, 1.5, -2.5, -0.5, 126.5, -126.5])[torch.arange(64) % 8]
        x = x.to(DEV)
        cache = kv.new_cache(6, 1, 64, 16)
        table = _i32([[3, 1, 2, 0, 5, 4]])
        kv.store(cache, _rows(kv, [96], [96], table), x, -x)
        model = Model(1, 64, 1)
        model.append(0, x, -x)
        c = torch.stack([cache.k[p, 0] for p in table[0].tolist()]).view(96, 64).double().cpu()
        assert torch.equal(c, model.codes[0][0][0])
        assert torch.equal(torch.stack([cache.v[p, 0] for p in table[0].tolist()]).view(96, 64).double().cpu(), -c)
        assert torch.equal(cache.k_scale[table[0].long(), 0, 0].double().cpu(), model.amax[0][0][0])


def test_store_not_finite_poisons_its_block_alone_until_it_starts_anew():
    kv = pkg("kvcache")
    cache = kv.new_cache(4, 2, 64, 32)
    table = _i32([[2, 0]])
    x = torch.randn(40, 2, 64, device=DEV, generator=_gen(1)).bfloat16()
    bad = x.clone()
    bad[20, 1, 7], bad[3, 0, 0] = math.inf, math.nan
    kv.store(cache, _rows(kv, [40], [40], table), bad, x)
    k, v = kv.read(cache, _rows(kv, [40], [40], table), 40, torch.float32)
    nan = torch.isnan(k).all(2)
    want = torch.zeros(40, 2, dtype=torch.bool, device=DEV)
    want[16:32, 1] = True
    want[:16, 0] = True
    assert torch.equal(nan, want) and torch.equal(torch.isnan(k).any(2), want) and not torch.isnan(v).any()
    q = torch.randn(20, 2, 64, device=DEV, generator=_gen(2)).bfloat16()
    for which in range(2):      # attention: the rows that see the block, and no others
        c = kv.new_cache(4, 2, 64, 32)
        kv.store(c, _rows(kv, [40], [40], table), *((bad, x) if which == 0 else (x, bad)))
        for m in (20, 1):
            o = torch.isnan(kv.attn(q[:m], c, _rows(kv, [m], [15 + m], table), 0.125))
            assert bool(o[:, 0].all()) and not bool(o[:1, 1].any()) and bool(o[1:, 1].all())
    kv.store(cache, _rows(kv, [1], [17], table), x[:1], x[:1])     # cut back to 16 tokens, then one more: its block starts anew
    k, _ = kv.read(cache, _rows(kv, [1], [17], table), 1, torch.float32)
    assert torch.isfinite(k).all()


def test_rows_and_pages_outside_are_left_alone():
    """Entries that are no page, tokens beyond the table, row descriptors beyond the tensors: nothing else is written, what is read is NaN."""
    kv = pkg("kvcache")
    cache = kv.new_cache(6, 1, 64, 16)
    x = torch.ones(64, 1, 64, device=DEV, dtype=torch.bfloat16)
    for t in cache:
        t.fill_(5)
    before = [t.clone() for t in cache]
    # no sequence's rows are inside, or have a page
    kv.store(cache, kv.Rows(_i32([70, 90]), _i32([20]), _i32([[0, 1]]), 64), x, x)
    kv.store(cache, kv.Rows(_i32([40, 10]), _i32([20]), _i32([[0, 1]]), 64), x, x)
    kv.store(cache, kv.Rows(_i32([0, 32]), _i32([32]), _i32([[6, -1]]), 64), x, x)
    kv.store(cache, kv.Rows(_i32([0, 32]), _i32([2 ** 31 - 1]), _i32([[0, 1]]), 64), x, x)
    kv.store(cache, kv.Rows(_i32([0, 32]), _i32([-2 ** 31]), _i32([[0, 1]]), 64), x, x)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    # more rows than `most`: the first ones are stored, as the last tokens
    kv.store(cache, kv.Rows(_i32([0, 32]), _i32([8]), _i32([[2, 3]]), 8), x, x)
    assert bool((cache.k[2, 0, :8] == 127).all()) and torch.equal(cache.k[3], before[0][3])
    kv.store(cache, kv.Rows(_i32([0, 48]), _i32([48]), _i32([[0, 7, 1]]), 48), x, x)
    k, v = kv.read(cache, kv.Rows(_i32([0, 64]), _i32([64]), _i32([[0, 7, 1]]), 64), 64)
    assert torch.equal(torch.isnan(k[:, 0, 0]).cpu(), (torch.arange(64) // 16 % 2 == 1))
    q = torch.randn(3, 2, 64, device=DEV, generator=_gen(2)).bfloat16()
    for new, length, causal, nan in ((3, 18, True, [False, True, True]), (3, 18, False, [True] * 3), (3, 48, True, [True] * 3), (1, 16, True, [False]),
                                     (3, 2 ** 31 - 1, True, [True] * 3), (3, 0, True, [False] * 3), (3, 2, True, [False] * 3)):
        o = kv.attn(q[:new], cache, kv.Rows(_i32([0, new]), _i32([length]), _i32([[0, 7, 1]]), new), 0.1, causal)
        assert torch.isnan(o).flatten(1).all(1).tolist() == nan and torch.isnan(o).flatten(1).any(1).tolist() == nan, (new, length, causal)
    o = torch.full((3, 2, 64), 9.0, device=DEV, dtype=torch.bfloat16)
    kv.attn(q, cache, kv.Rows(_i32([1, 2]), _i32([16]), _i32([[0]]), 3), 0.1, True, out=o)
    assert bool((o[0] == 9).all()) and bool((o[2] == 9).all()) and not bool((o[1] == 9).any())


def _attn_check(o, q, model, new, lens, scale, causal, what=""):
    h, at = q.shape[1], 0
    heads = model.codes[0][0].shape[0]
    for s, (m, l) in enumerate(zip(new, lens)):
        k, v = model.values(s, 0)[:l], model.values(s, 1)[:l]
        pos = torch.arange(l - m, l, device=DEV) if causal else torch.full((m,), l, device=DEV)
        keep = torch.arange(l, device=DEV) <= pos[:, None]
        tiny = model.amax[s][1].repeat_interleave(16, 1)[:, :l].to(DEV)
        for j in range(h if m else 0):
            # q rows are scaled to f16: what lies 2^14 below the row's largest rounds by 2^-25 of it, less than the sums' own roundings
            want, bound = _reference(q[at:at + m, j], k[:, j * heads // h], v[:, j * heads // h], scale, keep, torch.zeros(l, dtype=torch.float64, device=DEV), U[torch.float16], U[q.dtype], tiny[j * heads // h])
            _check(o[at:at + m, j], want, bound, "%s sequence %d head %d" % (what, s, j))
        at += m


ATTN = [([1], [1], 1, 1, 16, 16), ([1, 1, 1], [5, 700, 64], 4, 2, 128, 64), ([3, 0, 1], [3, 20, 1], 2, 2, 64, 16), ([33, 1, 70], [33, 500, 90], 6, 2, 128, 32),
        ([200], [1333], 4, 1, 64, 128), ([1], [9001], 8, 1, 128, 16), ([40], [4000], 2, 2, 256, 256), ([5, 17], [900, 17], 7, 1, 80, 64), ([1], [3000], 3, 3, 208, 16),
        ([129], [129], 1, 1, 48, 16), ([1], [2000], 64, 1, 128, 64), ([1], [2000], 2, 2, 64, 32), ([20, 3], [50, 9], 1, 1, 64, 16), ([20], [3000], 1, 1, 64, 16),
        ([20], [50], 1, 1, 128, 16), ([20], [3000], 1, 1, 112, 16), ([1, 1], [60, 9], 2, 1, 128, 16), ([1], [40], 1, 1, 256, 16), ([40], [60], 1, 1, 240, 16),
        ([200, 9], [1008, 1], 1, 1, 64, 16), ([300], [1000], 1, 1, 128, 16), ([150], [20000], 1, 1, 64, 64), ([75], [20000], 2, 1, 128, 64),
        ([60, 3], [65, 9], 1, 1, 96, 16), ([70], [3000], 1, 1, 80, 32), ([257], [1000], 2, 2, 96, 16), ([150], [20000], 1, 1, 80, 64), ([9], [60], 1, 1, 192, 16), ([5], [3000], 2, 2, 144, 32), ([60, 2], [70, 33], 2, 2, 160, 16), ([60], [3000], 1, 1, 176, 16), ([257], [1000], 1, 1, 192, 16),
        ([150], [20000], 1, 1, 176, 64), ([300], [320], 86, 86, 240, 16), ([130], [2048], 65, 65, 256, 64),
        ([33], [208], 260, 260, 16, 16), ([40, 7], [120, 60], 1, 1, 128, 16), ([1030], [2050], 86, 86, 64, 64), ([130], [20000], 65, 65, 48, 64), ([130], [1030], 192, 3, 96, 64),
        ([130], [2050], 86, 86, 128, 64), ([130], [1030], 129, 129, 112, 16), ([130], [600], 192, 3, 192, 32), ([130], [130], 1, 1, 256, 16)]


def test_the_cases_reach_every_form():
    """Workgroups of 16, 32, 128 and 256 rows (of head dims up to 96 the last two alone, above 128 without the second), keys shared
    and not."""
    import ctypes
    ffi = pkg("ffi")
    out, dp = (ctypes.c_int32 * 3)(), lambda d, rows: 96 if 64 < d <= 96 and rows > 32 else -(-d // 64) * 64
    want = {(p, r, s) for p in (64, 96, 128, 192, 256) for r in (16, 32, 128, 256) for s in (False, True) if (p != 96 or r > 32) and (p < 192 or r != 32)}
    seen, blocks = {1: set(), 2: set()}, {(by, n) for by in (1, 2) for n in (1, 2)}
    for b, lq, lk, h, hk, d in CROSS:
        ffi.k("gpu_internal_states_plan", lq * (h // hk), b * hk, lk, d, 2, ctypes.cast(out, ctypes.c_void_p))
        blocks.discard((2, out[2]) if lk > 64 else None)
        seen[2].add((dp(d, lq * (h // hk)), out[0], out[1] > 1))
    for new, lens, h, heads, dim, page in ATTN:
        cols = max(-(-l // page) for l in lens)
        ffi.k("gpu_internal_states_plan", max(new) * (h // heads), len(lens) * heads, cols * page, dim, 1, ctypes.cast(out, ctypes.c_void_p))
        blocks.discard((1, out[2]) if max(lens) > 64 else None)
        seen[1].add((dp(dim, max(new) * (h // heads)), out[0], out[1] > 1))
    assert seen[2] >= want, sorted(want - seen[2])
    assert seen[1] >= want, sorted(want - seen[1])
    assert not blocks, blocks


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_cache_attn(case, dtype, causal):
    kv = pkg("kvcache")
    new, lens, h, heads, dim, page = case
    cache, table, model = _filled(lens, heads, dim, page, 11, dtype)
    q = (1.5 * torch.randn(sum(new), h, dim, device=DEV, generator=_gen(12))).to(dtype)
    scale = dim ** -0.5
    _attn_check(kv.attn(q, cache, _rows(kv, new, lens, table), scale, causal), q, model, new, lens, scale, causal)


@pytest.mark.parametrize("new", [1, 50])
def test_cache_attn_scales_of_all_sizes(new):
    """Values and queries at the ends of bf16, blocks whose scales differ by 2^20, blocks of zeros."""
    kv = pkg("kvcache")
    g, lens = _gen(13), [200]
    for q_size, k_size, v_size in ((1e-30, 1e30, 1e36), (3e30, 1e-30, 1e-20), (1.0, 1.0, 65504.0), (1e4, 1e-4, 1e-6)):
        cache, table = kv.new_cache(8, 1, 64, 32), _table(lens, 32, 8, 1)
        by = 2.0 ** torch.randint(-20, 1, (200, 1, 1), device=DEV, generator=g)
        by[32:64] = 0
        k = (k_size * torch.randn(200, 1, 64, device=DEV, generator=g)).bfloat16()
        v = (v_size * by * torch.randn(200, 1, 64, device=DEV, generator=g)).bfloat16()
        kv.store(cache, _rows(kv, lens, lens, table), k, v)
        model = Model(1, 64, 1)
        model.append(0, k, v)
        q = (q_size * torch.randn(new, 2, 64, device=DEV, generator=g)).bfloat16()
        _attn_check(kv.attn(q, cache, _rows(kv, [new], lens, table), 0.125, True), q, model, [new], lens, 0.125, True, "%g %g %g" % (q_size, k_size, v_size))


@pytest.mark.parametrize("new", [1, 50])
def test_cache_attn_small_values_with_most_of_the_probability(new):
    """Blocks whose values are 2^-30 of others' hold nearly all of the probability: their keys' p A is subnormal, their sum is not."""
    kv = pkg("kvcache")
    g, lens = _gen(14), [1600]
    cache, table = kv.new_cache(50, 1, 64, 32), _table(lens, 32, 50, 1)
    k = (0.05 * torch.randn(1600, 1, 64, device=DEV, generator=g)).bfloat16()
    v = torch.randn(1600, 1, 64, device=DEV, generator=g)
    v[16:] *= 2.0 ** -30
    v = v.bfloat16()
    kv.store(cache, _rows(kv, lens, lens, table), k, v)
    model = Model(1, 64, 1)
    model.append(0, k, v)
    q = torch.randn(new, 2, 64, device=DEV, generator=g).bfloat16()
    _attn_check(kv.attn(q, cache, _rows(kv, [new], lens, table), 0.125, True), q, model, [new], lens, 0.125, True)


def test_cache_attn_strided_rows():
    kv = pkg("kvcache")
    lens = [300, 40]
    cache, table, model = _filled(lens, 2, 64, 32, 21)
    for new in ([1, 1], [60, 20]):
        fused = torch.randn(sum(new), 3, 4, 66, device=DEV, generator=_gen(22)).bfloat16()
        for q in (fused[:, 1, :, :64], fused[:, 1, :, 1:65]):
            out = torch.zeros(sum(new), 4, 65, device=DEV, dtype=torch.bfloat16)[..., :64]
            kv.attn(q, cache, _rows(kv, new, lens, table), 0.125, True, out=out)
            _attn_check(out, q, model, new, lens, 0.125, True)


def test_cache_past_32_bit_offsets():
    """Pages of one cache whose codes lie beyond 4 GiB."""
    kv = pkg("kvcache")
    pages, page, heads, dim = 4200, 4096, 1, 256
    cache = kv.Cache(*(torch.empty(pages, heads, page, dim, dtype=torch.int8, device=DEV) for _ in range(2)),
                     *(torch.empty(pages, heads, page // 16, device=DEV) for _ in range(2)))
    assert cache.k.numel() > 2 ** 32
    lens, table = [5000], _i32([[pages - 1, pages - 2]])
    g = _gen(31)
    k, v = (torch.randn(5000, 1, 256, device=DEV, generator=g).bfloat16() for _ in range(2))
    kv.store(cache, _rows(kv, lens, lens, table), k, v)
    model = Model(1, 256, 1)
    model.append(0, k, v)
    _same_cache(kv, cache, table, lens, model)
    for m in (1, 40):
        q = torch.randn(m, 1, 256, device=DEV, generator=g).bfloat16()
        _attn_check(kv.attn(q, cache, _rows(kv, [m], lens, table), 0.0625), q, model, [m], lens, 0.0625, True)
    kv.copy_pages(cache, _i32([pages - 1, pages - 2]), _i32([3, pages - 3]))
    _same_cache(kv, cache, _i32([[3, pages - 3]]), lens, model)


@pytest.mark.parametrize("shape", [(None, 9, 1, 16, 16), (3, 20, 5, 64, 80), (2, 7, 8, 128, 128)])
def test_copy_pages(shape):
    kv = pkg("kvcache")
    layers, pages, heads, page, dim = shape
    cache = kv.new_cache(pages, heads, dim, page, layers)
    g = _gen(41)
    for t in cache:
        t.copy_(torch.randint(-127, 128, t.shape, device=DEV, generator=g))
    src, dst = [0, 4, 2, -1, pages, 5], [3, 1, 6, 0, 2, 5]     # two that are no pages, one onto itself
    want = [t.clone() for t in cache]
    axis = 0 if layers is None else 1
    for a, b in list(zip(src, dst))[:3]:
        for t, old in zip(want, cache):
            t.select(axis, b).copy_(old.select(axis, a))
    kv.copy_pages(cache, _i32(src), _i32(dst))
    assert all(torch.equal(a, b) for a, b in zip(cache, want))


# ---- as they are used ------------------------------------------------------------------------------------------------------------

def test_streams_and_graphs():
    """Calls on a side stream, and captured: replays with new inputs in place, the program's own work between them."""
    ql, kv = pkg("qlinear"), pkg("kvcache")
    lens = [1500, 70]
    cache, table, _ = _filled(lens, 2, 128, 32, 51)
    rows = _rows(kv, [1, 1], lens, table)
    g = _gen(52)
    q = torch.randn(2, 8, 128, device=DEV, generator=g).bfloat16()
    cq, ck, cv = _cross_inputs(2, 100, 2500, 2, 2, 64, torch.float16, 53)
    new_k, new_v = (torch.randn(2, 2, 128, device=DEV, generator=g).bfloat16() for _ in range(2))

    def step():
        kv.store(cache, rows, new_k, new_v)
        return kv.attn(q, cache, rows, 0.1), ql.cross_attn(cq, ck, cv, 0.125), *kv.read(cache, rows, 2)

    first = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, outs))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        q.normal_(generator=g); cq.normal_(generator=g); new_k.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_a_run_of_them_together():
    """Two prompts through two layers: stored, attended, forked, grown token by token, an encoder's states attended from the cache, one freed,
    pages moved: at every step what a plain implementation over each sequence's own tokens gives."""
    ql, kv = pkg("qlinear"), pkg("kvcache")
    layers, heads, h, dim, g = 2, 2, 4, 64, _gen(81)
    seqs = kv.Sequences(kv.new_cache(40, heads, dim, 16, layers))
    models = {}

    def step(ids, counts, causal=True):
        rows = seqs.extend(ids, counts)
        for layer in range(layers):
            cache = seqs.cache.layer(layer)
            k, v = (torch.randn(sum(counts), heads, dim, device=DEV, generator=g).bfloat16() for _ in range(2))
            q = torch.randn(sum(counts), h, dim, device=DEV, generator=g).bfloat16()
            kv.store(cache, rows, k, v)
            o = kv.attn(q, cache, rows, 0.125, causal)
            at = 0
            for s, c in zip(ids, counts):
                models[s][layer].append(0, k[at:at + c], v[at:at + c])
                _attn_check(o[at:at + c], q[at:at + c], models[s][layer], [c], [seqs.length(s)], 0.125, causal, "sequence %d layer %d" % (s, layer))
                at += c

    def copy_of(ms):
        out = [Model(heads, dim, 1) for _ in ms]
        for a, b in zip(out, ms):
            a.codes, a.amax = [[t.clone() for t in w] for w in b.codes], [[t.clone() for t in w] for w in b.amax]
        return out

    a, b = seqs.add(), seqs.add()
    for s in (a, b):
        models[s] = [Model(heads, dim, 1) for _ in range(layers)]
    step([a, b], [100, 37])
    step([b, a], [1, 1])
    c = seqs.fork(a)
    models[c] = copy_of(models[a])
    for _ in range(3):
        step([a, b, c], [1, 1, 1])
    step([c], [30])
    seqs.free(b)
    assert seqs.compact() > 0
    step([a, c], [2, 1])
    states = seqs.add()     # an encoder's states, attended by rows that are none of its tokens, and the same in 16 bits
    models[states] = [Model(heads, dim, 1) for _ in range(layers)]
    step([states], [77], causal=False)
    rows = seqs.rows([states, a], [200, 3])
    q = torch.randn(203, h, dim, device=DEV, generator=g).bfloat16()
    cache = seqs.cache.layer(1)
    o = kv.attn(q, cache, rows, 0.125, causal=False)
    _attn_check(o[:200], q[:200], models[states][1], [200], [77], 0.125, False, "states")
    _attn_check(o[200:], q[200:], models[a][1], [3], [seqs.length(a)], 0.125, False, "all of a")
    k, v = kv.read(cache, seqs.rows([states], [77]), 77)
    k16, v16 = (t.double()[None] for t in (k, v))
    x = ql.cross_attn(q[None, :200], k[None], v[None], 0.125)
    _cross_check(x, q[None, :200], k16, v16, 0.125, what="read back")


def test_native_calls_take_what_the_python_side_takes(monkeypatch):
    """The calls through csrc/py_states.hpp and the same calls in Python: the same bits, and none of them left to the other side."""
    ql, kv = pkg("qlinear"), pkg("kvcache")
    lens = [700, 33]
    cache, table, _ = _filled(lens, 2, 64, 32, 71)
    rows = _rows(kv, [3, 1], lens, table)
    g = _gen(72)
    q, x, y = (torch.randn(4, h, 64, device=DEV, generator=g).bfloat16() for h in (4, 2, 2))
    layered = kv.new_cache(6, 2, 64, 32, 3)
    for t in layered:
        t.copy_(torch.randint(-100, 100, t.shape, device=DEV, generator=g))
    cq, ck, cv = _cross_inputs(2, 5, 70, 2, 1, 64, torch.float16, 73)
    masks = [None, torch.rand(70, device=DEV, generator=g) < 0.5, torch.randn(2, 70, device=DEV, generator=g)]

    def calls():
        kv.store(cache, rows, x, y)
        kv.copy_pages(layered, _i32([1, 2]), _i32([4, 0]))
        return [kv.attn(q, cache, rows, 0.125), kv.attn(q, cache, rows, 1, False), *kv.read(cache, rows, 4), *kv.read(cache, rows, 4, torch.float32), *cache, *layered.layer(2),
                *(ql.cross_attn(cq, ck, cv, 0.125, _i32([70, 4]), m) for m in masks), ql.cross_attn(cq[:, ::2], ck, cv, 1)]

    assert ql._pycalls is not None
    with monkeypatch.context() as m:
        for module, name in ((kv, "_store"), (kv, "_read"), (kv, "_attn"), (kv, "_copy_pages"), (ql, "_cross_attn")):
            m.setattr(module, name, lambda *a, **k: pytest.fail("left to the Python side"))
        native = [t.clone() for t in calls()]
    monkeypatch.setattr(ql, "_pycalls", None)
    assert all(torch.equal(a, b) for a, b in zip(native, calls()))


def test_refusals_with_gpu_tensors():
    ql, kv = pkg("qlinear"), pkg("kvcache")
    q, k, v = _cross_inputs(1, 4, 6, 2, 2, 64, torch.bfloat16, 61)
    for bad in (lambda: ql.cross_attn(q.float(), k.float(), v.float(), 1.0), lambda: ql.cross_attn(q, k.half(), v, 1.0), lambda: ql.cross_attn(q, k[..., :32], v[..., :32], 1.0),
                lambda: ql.cross_attn(q[:, :, :1], k, v, 1.0), lambda: ql.cross_attn(q, k, v[:, :5], 1.0), lambda: ql.cross_attn(q, k, v, 1.0, _i32([1, 2])),
                lambda: ql.cross_attn(q, k, v, 1.0, torch.tensor([3], device=DEV)), lambda: ql.cross_attn(q, k, v, 1.0, None, torch.ones(1, 5, device=DEV)),
                lambda: ql.cross_attn(q, k, v, 1.0, None, torch.ones(6, device=DEV, dtype=torch.float16)), lambda: ql.cross_attn(q.cpu(), k, v, 1.0),
                lambda: ql.cross_attn(q.requires_grad_(), k, v, 1.0), lambda: ql.cross_attn(q.detach()[..., ::2], k[..., ::2], v[..., ::2], 1.0)):
        with pytest.raises(ValueError):
            bad()
    q = q.detach()
    for bad in (lambda: ql.cross_attn(q, k, v, math.inf), lambda: ql.cross_attn(q, k, v, math.nan), lambda: ql.cross_attn(q[..., :12], k[..., :12], v[..., :12], 1.0)):
        with pytest.raises(pkg("ffi").KernelError):
            bad()
    cache = kv.new_cache(4, 2, 64, 32)
    rows = kv.Rows(_i32([0, 1]), _i32([1]), _i32([[0]]), 1)
    x = torch.zeros(1, 2, 64, device=DEV, dtype=torch.bfloat16)
    wrong = [rows._replace(starts=_i32([0])), rows._replace(lens=torch.tensor([1], device=DEV)), rows._replace(table=_i32([[0], [1]])), rows._replace(table=_i32([[0]]).cpu())]
    for bad in [lambda r=r: kv.store(cache, r, x, x) for r in wrong] + [lambda r=r: kv.attn(x, cache, r, 1.0) for r in wrong] + [lambda r=r: kv.read(cache, r, 1) for r in wrong] + [
            lambda: kv.store(cache, rows, x[:, :1], x[:, :1]), lambda: kv.store(cache, rows, x.float(), x.float()), lambda: kv.store(cache, rows, x, x[:0]),
            lambda: kv.store(cache._replace(k=cache.k[:, :, :16]), rows, x, x), lambda: kv.store(cache._replace(k_scale=cache.k_scale[:2]), rows, x, x),
            lambda: kv.attn(x[..., :32], cache, rows, 1.0), lambda: kv.attn(torch.zeros(1, 3, 64, device=DEV).half(), cache, rows, 1.0),
            lambda: kv.attn(x, cache, rows, 1.0, True, torch.zeros(1, 2, 64, device=DEV)), lambda: kv.read(cache, rows, 1, torch.int8),
            lambda: kv.copy_pages(cache, _i32([0]), _i32([1, 2])), lambda: kv.copy_pages(cache, _i32([0]).long(), _i32([1]).long()),
            lambda: kv.new_cache(4, 2, 64, 24), lambda: kv.new_cache(4, 2, 60, 32)]:
        with pytest.raises(ValueError):
            bad()
