"""Whether two tensors share memory (qlinear._meet), against the bytes they have, and what calls make of it."""
import random

import pytest
import torch

from conftest import pkg

ql = pkg("qlinear")


def _bytes(t):
    at = [t.data_ptr()]
    for n, s in zip(t.shape, t.stride()):
        at = [a + i * s * t.element_size() for a in at for i in range(n)]
    return {a + b for a in at for b in range(t.element_size())}


def _view(rng, room):
    """Any 1-, 2- or 3-D view with a dense last axis."""
    t = room.view(rng.choice((torch.uint8, torch.bfloat16, torch.float32)))
    have = t.numel()
    while True:
        dims = [rng.randrange(0 if rng.random() < 0.03 else 1, 7) for _ in range(rng.randrange(3))] + [rng.randrange(1, 9)]
        strides = [rng.choice((rng.randrange(1, 40), dims[-1], 8, 16, 24, 48)) for _ in dims[:-1]] + [1]
        if len(dims) == 3 and rng.random() < 0.5:
            strides[0] = strides[1] * rng.choice((dims[1], dims[1] + 1, 6)) if dims[1] else strides[0]
        reach = 1 + sum((n - 1) * s for n, s in zip(dims, strides))
        if reach <= have:
            return t.as_strided(dims, strides, rng.randrange(have - reach + 1))


def test_meet_is_exact():
    rng, room, seen = random.Random(4), torch.zeros(1024, dtype=torch.uint8), [0, 0]
    for _ in range(6000):
        a, b = _view(rng, room), _view(rng, room)
        want = bool(_bytes(a) & _bytes(b))
        assert ql._meet(a, b) == want and ql._meet(b, a) == want, (a.dtype, a.shape, a.stride(), a.storage_offset(), b.dtype, b.shape, b.stride(), b.storage_offset())
        seen[want] += 1
    assert min(seen) > 500


def test_views_of_one_buffer_that_programs_have():
    """Query, key and value columns of one product, heads of one tensor padded or turned around, rows behind rows."""
    qkv = torch.zeros(50, 12, 64, dtype=torch.bfloat16)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    assert not ql._meet(q, k) and not ql._meet(k, v) and ql._meet(q, qkv[:, 7:9]) and ql._meet(qkv, k)
    pad = qkv[..., :40]
    assert not ql._meet(pad[:, :8], pad[:, 8:10]) and not ql._meet(pad, qkv[..., 40:]) and ql._meet(pad, qkv[..., 39:])
    turned = torch.zeros(12, 50, 64, dtype=torch.bfloat16).transpose(0, 1)
    assert not ql._meet(turned[:, :8], turned[:, 8:]) and ql._meet(turned[:, :8], turned[:, 7:]) and not ql._meet(turned[:20], turned[20:]) and ql._meet(turned[:21], turned[20:])
    by_head = torch.zeros(50, 4, 3, 64, dtype=torch.bfloat16)
    assert not ql._meet(by_head[:, :, 0], by_head[:, :, 1]) and not ql._meet(by_head[:, :, 0], by_head[:, :, 2]) and ql._meet(by_head[:, :, 0], by_head[:, :, 0][1:])
    assert not ql._meet(qkv[:25], qkv[25:]) and ql._meet(qkv[:26], qkv[25:]) and not ql._meet(qkv[:0], qkv) and not ql._meet(qkv, qkv.clone())


def test_separate_takes_an_output_in_an_inputs_place_where_that_is_allowed():
    x = torch.zeros(6, 40)
    ql._separate(x, "out", [torch.zeros(3)], [x, x.view(6, 40)])
    ql._separate(x[:1], "out", [], [x.as_strided((1, 40), (99, 1))])      # (one row: its stride says nothing)
    ql._separate(x[:, :8], "out", [x[:, 8:], None], [x[:, :8]])
    for out, reads, places in ((x, [x], []), (x, [x], [x]), (x[:5], [], [x[1:]]), (x[:, :39], [], [x[:, 1:]]), (x[:, :20], [], [x.view(12, 20)[:6]]), (x, [x[:, 3:]], [x]), (x, [], [x, x.view(torch.int32)])):
        with pytest.raises(ValueError, match="out .* memory"):
            ql._separate(out, "out", reads, places)
