"""Attention to stored states at the ends of what its calls take, against the formulas in 64 bits and the bounds of test_gpu_states.py."""
import pytest
import torch

from conftest import pkg
from test_gpu_states import DEV, Model, U, _attn_check, _check, _cross_check, _cross_inputs, _filled, _gen, _reference, _rows, _table

pytestmark = pytest.mark.gpu


def test_mixed_batches_with_more_rows_than_a_join_takes():
    """300 sequences of which one has a piece of a prompt, counted as 2^26 rows: every sequence's are those of the formula."""
    kv = pkg("kvcache")
    new = [90] + [1 + i % 3 for i in range(299)]
    lens = [m + i % 40 for i, m in enumerate(new)]
    cache, table, model = _filled(lens, 8, 16, 16, 91)
    q = torch.randn(sum(new), 32, 16, device=DEV, generator=_gen(92)).bfloat16()
    rows = _rows(kv, new, lens, table)._replace(most=8192)      # a bound that a program knows beforehand
    assert 300 * 8 * 8192 * 4 > 2 ** 26
    for causal in (True, False):
        o = kv.attn(q, cache, rows, 0.25, causal)
        assert o.shape == q.shape
        _attn_check(o, q, model, new, lens, 0.25, causal)


def test_cross_attn_with_more_rows_than_a_join_takes():
    """4 x 524288 rows of 32 heads, queries alike: every row is the one that a short call gives."""
    ql = pkg("qlinear")
    g = _gen(93)
    one = torch.randn(4, 1, 32, 8, device=DEV, generator=g).bfloat16()
    k, v = (torch.randn(4, 20, 32, 8, device=DEV, generator=g).bfloat16() for _ in range(2))
    o = ql.cross_attn(one.expand(-1, 524288, -1, -1), k, v, 0.3)
    _cross_check(o[:, :1], one, k, v, 0.3)
    assert bool((o == o[:, :1]).all())


def _values_check(q, k, v, new, causal, unit, what):
    """Attention over one sequence of these keys and values, in units of `unit` (a power of two, of each row) against the formula.  Beside the
    roundings that test_gpu_states.py counts, p A is held in f16 in units of 2^-34 of the row's largest, in which an A below 2^-90 counts as that."""
    kv = pkg("kvcache")
    length, heads, dim = k.shape
    pages = -(-length // 64) + 1
    cache, table = kv.new_cache(pages, heads, dim, 64), _table([length], 64, pages, 1)
    kv.store(cache, _rows(kv, [length], [length], table), k, v)
    model = Model(heads, dim, 1)
    model.append(0, k, v)
    o = kv.attn(q, cache, _rows(kv, [new], [length], table), 0.125, causal).double() / unit[:, None, None]
    pos = torch.arange(length - new, length, device=DEV) if causal else torch.full((new,), length, device=DEV)
    values, keys = model.values(0, 1), model.values(0, 0)
    amax = model.amax[0][1].repeat_interleave(16, 1)[:, :length].to(DEV).clamp(min=2.0 ** -90)
    for j in range(q.shape[1]):
        i = j * heads // q.shape[1]
        for u in unit.unique().tolist():
            rows = unit == u
            keep = (torch.arange(length, device=DEV) <= pos[:, None])[rows]
            want, bound = _reference(q[rows, j], keys[:, i], values[:, i] / u, 0.125, keep, torch.zeros(length, dtype=torch.float64, device=DEV), U[torch.float16], U[q.dtype], amax[i] / u)
            _check(o[rows, j], want, bound, "%s head %d" % (what, j))


@pytest.mark.parametrize("dim", [64, 128, 240])
@pytest.mark.parametrize("new,length", [(1, 200), (1, 9000), (50, 200), (200, 300), (70, 9000)])
def test_cache_attn_values_far_below_and_above_each_other(new, length, dim):
    """Values near 1e-30; rows that see such values alone, before tokens whose values are 2^180 of theirs; values 2^-90 of others' that hold all
    but e^-60 of the probability; the largest of bf16 beside the smallest."""
    g = _gen(95)
    q = torch.randn(new, 2, dim, device=DEV, generator=g).bfloat16()
    k, v = (torch.randn(length, 1, dim, device=DEV, generator=g).bfloat16() for _ in range(2))
    one = torch.ones(new, dtype=torch.float64, device=DEV)
    for causal in (True, False):
        _values_check(q, k, (v.float() * 1e-30).bfloat16(), new, causal, one * 2.0 ** -100, "1e-30")
        some = torch.where(torch.arange(length, device=DEV) % 48 < 16, 0.0, 1e-28)[:, None, None]
        _values_check(q, k, (v.float() * some).bfloat16(), new, causal, one * 2.0 ** -93, "zeros beside 1e-28")
    first = length - (new + 1) // 2      # the later half of the rows' own tokens, or the last one's
    huge = torch.where(torch.arange(length, device=DEV) // 16 * 16 >= first, 1e30, 1e-25)[:, None, None]
    sees = torch.arange(length - new, length, device=DEV) >= (first + 15) // 16 * 16
    _values_check(q, k, (v.float() * huge).bfloat16(), new, True, torch.where(sees, 2.0 ** 100, 2.0 ** -83), "before 1e30")
    # one direction of the keys decides: the tokens of every third block have logits 60 above the others'
    q[..., 0], k[..., 0] = 16.0, 0.0
    third = torch.arange(length, device=DEV) // 16 % 3 == 0
    k[third, :, 0] = 30.0
    weak = torch.where(third, 1e-25, 100.0)[:, None, None]
    _values_check(q, k, (v.float() * weak).bfloat16(), new, False, one * 2.0 ** -83, "probable and small")
    k[third, :, 0] = 88.0
    weak = torch.where(third, 1e-38, 1e38)[:, None, None]
    _values_check(q, k, (v.float() * weak).clamp(-3.38e38, 3.38e38).bfloat16(), new, False, one * 2.0 ** -127, "ends of bf16")


@pytest.mark.parametrize("scale", [0.125, -2.0, 1e-3, 40.0, 1e-25])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("lq,lk", [(1, 130), (40, 70), (150, 300), (1, 3000)])
def test_cross_attn_very_large_biases_keep_their_order(lq, lk, dtype, scale):
    """A row whose biases are all far out, where q k^T is nothing beside them: the key with the largest has all of the probability, keys of
    the same bias share it, here and between ordinary keys and far ones."""
    ql = pkg("qlinear")
    q, k, v = _cross_inputs(1, lq, lk, 2, 1, 64, dtype, 94)
    low = torch.finfo(torch.float32).min
    best, second = lk // 3, lk - 1

    def winner(row, keys):
        o = ql.cross_attn(q, k, v, scale, None, torch.tensor(row, device=DEV, dtype=torch.float32))[0].double()
        want = v[0, keys, 0].double().mean(0)
        # probabilities alike, rounded once and summed as rounded: the sums' roundings and the output's
        assert ((o - want).abs() <= 2 * U[dtype] * v[0, keys, 0].double().abs().mean(0)).all(), (row[best], row[second], row[0])

    for rest, at_best in ((low, -1e38), (low, -3.3e38), (-3.4e38, -3.39e38), (-2.9e38, -2.2e38), (-1e38, -4e37), (3e37, 3e38), (1e38, -low), (low, -low), (low, -1e30), (-1e31, -1e30)):
        row = [rest] * lk
        row[best] = at_best
        winner(row, [best])
        row[second] = at_best
        winner(row, [best, second])
    # one of them after another, in steps of 1e-4
    steps = [-3.4e38 * (1 - 1e-4 * i) for i in range(lk)]
    winner(steps, [lk - 1])
    winner(steps[::-1], [0])
    winner([-x for x in steps], [0])
    row = [-x for x in steps[::-1]]
    row[second] = -3.4e38
    row[:2] = [-torch.inf, 0.0]
    winner(row, [lk - 2])


def test_cross_attn_as_many_keys_as_it_takes():
    """2^30 keys that are one key: sums of ones up to 2^22 a wave are exact, and so is what joins them."""
    ql = pkg("qlinear")
    one = torch.ones(1, 1, 1, 64, device=DEV, dtype=torch.bfloat16)
    many = one.expand(1, 1 << 30, 1, 64)
    assert bool((ql.cross_attn(one, many, many, 0.125) == 1).all())
    lens = torch.tensor([(1 << 30) - 5], dtype=torch.int32, device=DEV)
    assert bool((ql.cross_attn(one, many, many, 0.125, lens) == 1).all())


def test_dual_tensors_are_refused():
    """Forward mode has no rule here any more than reverse mode: a tangent is not dropped in silence, on neither side of the native calls."""
    ql, kv, ad = pkg("qlinear"), pkg("kvcache"), torch.autograd.forward_ad
    q, k, v = _cross_inputs(1, 4, 6, 2, 2, 64, torch.bfloat16, 61)
    bias = torch.zeros(6, device=DEV)
    cache, table, _ = _filled([20], 2, 64, 16, 62)
    rows = _rows(kv, [4], [20], table)
    x, out = q[0], torch.empty_like(q[0])
    ql.cross_attn(q, k, v, 0.125, None, bias)
    with ad.dual_level():
        dual = lambda t: ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: ql.cross_attn(dual(q), k, v, 0.125), lambda: ql.cross_attn(q, dual(k), v, 0.125), lambda: ql.cross_attn(q, k, dual(v), 0.125),
                     lambda: ql.cross_attn(q, k, v, 0.125, None, dual(bias)), lambda: kv.attn(dual(x), cache, rows, 0.125), lambda: kv.attn(x, cache, rows, 0.125, True, dual(out)),
                     lambda: kv.store(cache, rows, dual(x), x), lambda: kv.store(cache, rows, x, dual(x))):
            with pytest.raises(ValueError, match="carries a tangent"):
                call()
        want = ql.cross_attn(q, k, v, 0.125)
        assert torch.equal(ql.cross_attn(dual(q).detach(), k, v, 0.125), want)
        with torch.inference_mode():
            assert torch.equal(ql.cross_attn(dual(q), k, v, 0.125), want)


def test_scales_that_carry_derivatives_are_refused():
    """The cache's scales are numbers that a gradient could be asked for; the calls have none to give."""
    kv, ad = pkg("kvcache"), torch.autograd.forward_ad
    cache, table, _ = _filled([20], 2, 64, 16, 63)
    rows = _rows(kv, [4], [20], table)
    x = torch.randn(4, 2, 64, device=DEV, generator=_gen(64)).bfloat16()
    one, two = (torch.tensor([i], dtype=torch.int32, device=DEV) for i in (0, 1))
    with ad.dual_level():
        for name in ("k_scale", "v_scale"):
            scale = getattr(cache, name)
            for t, what in ((scale.clone().requires_grad_(), "asks for gradients"), (ad.make_dual(scale.clone(), scale), "carries a tangent")):
                bad = cache._replace(**{name: t})
                for call in (lambda: kv.store(bad, rows, x, x), lambda: kv.read(bad, rows, 4), lambda: kv.attn(x, bad, rows, 0.125), lambda: kv.copy_pages(bad, one, two)):
                    with pytest.raises(ValueError, match=name + " " + what):
                        call()
    trained = cache._replace(k_scale=cache.k_scale.clone().requires_grad_())
    with torch.no_grad():
        assert torch.equal(kv.attn(x, trained, rows, 0.125), kv.attn(x, cache, rows, 0.125))


def _attended_and_crossed(new, seed):
    """A cache call and a cross call whose keys are shared by workgroups, with what they read: both are functions of device data alone."""
    ql, kv = pkg("qlinear"), pkg("kvcache")
    lens = [2500, 900]
    cache, table, _ = _filled(lens, 2, 64, 32, seed)
    rows = _rows(kv, [new, new], lens, table)
    g = _gen(seed + 1)
    q = torch.randn(2 * new, 8, 64, device=DEV, generator=g).bfloat16()
    cq, ck, cv = _cross_inputs(2, new, 2500, 4, 2, 64, torch.float16, seed + 2)
    k_lens = torch.tensor([2500, 77], dtype=torch.int32, device=DEV)
    mask = torch.rand(2, 2500, device=DEV, generator=g) < 0.5
    return (q, cache, rows, cq, k_lens, mask), lambda: [kv.attn(q, cache, rows, 0.125), ql.cross_attn(cq, ck, cv, 0.125, k_lens, mask)]


@pytest.mark.parametrize("new", [1, 24, 60])
def test_two_graphs_follow_lengths_tables_and_masks(new):
    """What device data hold when a replay runs counts, not what they held at the capture; two graphs in turn, eager calls between them."""
    sets = [_attended_and_crossed(new, seed) for seed in (101, 111)]
    for _, call in sets:
        call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _, call in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for step, (lens, k_lens) in enumerate((([2500, 900], [2500, 77]), ([61, 2400], [0, 2500]), ([1700, 60], [3, 1300]), ([60, 60], [2500, 2499]))):
        for (q, cache, rows, cq, at, mask), _ in sets:
            q.normal_()
            cq.normal_()
            rows.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            rows.table.copy_(rows.table.flip(0) if step == 2 else rows.table)
            at.copy_(torch.tensor(k_lens, dtype=torch.int32))
            mask.logical_not_()
        for i in (1, 0, 1):
            graphs[i].replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        want = [call() for _, call in sets]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                # (tokens that a table does not hold are NaN)
                assert torch.equal(x.view(torch.int16), y.view(torch.int16)), (step, new)


@pytest.mark.parametrize("new", [1, 24, 60])
def test_two_streams_at_once(new):
    sets = [_attended_and_crossed(new, seed) for seed in (121, 131)]
    want = [call() for _, call in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(5):
        for i, (_, call) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(call())
    torch.cuda.synchronize()
    for many, once in zip(got, want):
        assert all(torch.equal(x, y) for o in many for x, y in zip(o, once))


@pytest.mark.parametrize("new", [1, 24, 70])
def test_pages_in_several_tables_and_outputs_in_the_queries_place(new):
    """Sequences that begin with the same pages; outputs written over the queries that they come from; a bound above the longest's rows."""
    kv = pkg("kvcache")
    cache, table, model = _filled([640], 2, 64, 32, 141)
    lens = [640, 300, 77]
    both = table.expand(3, -1).contiguous()
    q = torch.randn(3 * new, 8, 64, device=DEV, generator=_gen(142)).bfloat16()
    rows = _rows(kv, [new] * 3, lens, both)
    want = kv.attn(q, cache, rows, 0.125)
    for i, l in enumerate(lens):
        _attn_check(want[i * new:(i + 1) * new], q[i * new:(i + 1) * new], model, [new], [l], 0.125, True, "sequence %d" % i)
    place = q.clone()
    assert kv.attn(place, cache, rows, 0.125, out=place) is place and torch.equal(place, want)
    more = rows._replace(most=new + 200)
    for i, l in enumerate(lens):
        o = kv.attn(q, cache, more, 0.125)[i * new:(i + 1) * new]
        _attn_check(o, q[i * new:(i + 1) * new], model, [new], [l], 0.125, True, "bound, sequence %d" % i)
