"""Attention to stored states without a GPU: the ends of what its calls take."""
import ctypes

import pytest
import torch

from conftest import pkg

ffi = pkg("ffi")
P = 1 << 20         # an address that is never followed: a call that passes the checks ends at a launch without a device
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="a launch would follow the addresses")


def _plan(rows, problems, keys, d, bytes):
    out = (ctypes.c_int32 * 3)()
    return ffi.raw("gpu_internal_states_plan", rows, problems, keys, d, bytes, ctypes.cast(out, ctypes.c_void_p)), tuple(out)[:2]


def _cross(b, lq, lk, h, hk, d=64, ws=P, lens=0):
    return ffi.raw("gpu_cross_attn", 2, P, P, P, P, ws, b, lq, lk, h, hk, d, *([64] * 12), 1.0, lens, 0, 0, 0, 0)


def _cache(n, most, h, hk, d=128, cols=64):
    return ffi.raw("gpu_kv8_attn", 2, P, h * d, d, P, h * d, d, P, P, P, P, P, 4, 64, P, P, P, cols, n, 9000, most, h, hk, d, 0.1, 1, 0)


@no_device
def test_calls_whose_rows_no_join_could_take():
    """2^26 rows, counted with the longest sequence's for each, in one part: tiles that return at once for the most part, and a launch
    like any other.  Beyond 8388607 workgroups a call is refused."""
    for n, most in ((255, 8192), (256, 8192), (64, 32768), (4096, 8192)):
        assert _cache(n, most, 32, 8) > 0, (n, most)
    for b, lq in ((4, 524287), (4, 524288), (16, 524288)):
        assert _cross(b, lq, 77, 32, 32) > 0, (b, lq)
    assert _cache(65536, 8192, 32, 8) == -1 and _cross(512, 1 << 20, 77, 32, 32) == -1


def test_plans_end_where_launches_do():
    most = 0xffffffff // 512
    assert _plan(1, most, 77, 64, 2) == (0, (16, 1)) and _plan(1, most + 1, 77, 64, 2)[0] == -1
    assert _plan(32768, 2048, 4096, 128, 1) == (0, (256, 1))
    rows = 1 << 24      # 65536 tiles of 256
    assert _plan(rows, most // 65536, 77, 64, 2)[0] == 0 and _plan(rows, most // 65536 + 1, 77, 64, 2)[0] == -1
    # (tiles of 128 rows would be too many)
    assert _plan(rows, 100, 77, 64, 2) == (0, (256, 1))
    # rows that no join could take are never shared
    for problems in (1, 2, 8):
        for keys in (1 << 12, 1 << 20, 1 << 29):
            for by in (1, 2):
                rc, (tile, parts) = _plan((1 << 26) // problems, problems, keys, 64, by)
                assert rc == 0 and parts == 1, (problems, keys, by)


def test_lengths_end_at_two_to_the_thirty():
    """Positions of keys, a few tiles past the last, and of rows behind them stay 32-bit numbers."""
    assert _cross(1, 64, (1 << 30) + 1, 1, 1, 8) == -1 and _cross(1, 64, (1 << 31) - 1, 1, 1, 8) == -1
    assert _cross(1, (1 << 30) + 1, 64, 1, 1, 8) == -1
    assert _plan(64, 1, (1 << 30) + 1, 8, 2)[0] == -1 and _plan(64, 1, 1 << 30, 8, 2)[0] == 0
    assert _cache(1, (1 << 30) + 1, 1, 1) == -1
    # a table may be wider than any sequence is long
    assert _plan(64, 1, 1 << 36, 64, 1)[0] == 0


@no_device
def test_lengths_up_to_two_to_the_thirty_pass():
    assert _cross(1, 64, 1 << 30, 1, 1, 8) > 0 and _cross(1, 1 << 30, 64, 1, 1, 8) > 0 and _cache(1, 1 << 30, 1, 1) > 0


def test_inputs_that_carry_derivatives_are_refused():
    ql, ad = pkg("qlinear"), torch.autograd.forward_ad
    x = torch.ones(3)
    ql._no_grad(x, "x")
    with pytest.raises(ValueError, match="x asks for gradients"):
        ql._no_grad(x.clone().requires_grad_(), "x")
    with ad.dual_level():
        dual = ad.make_dual(x, x)
        with pytest.raises(ValueError, match="x carries a tangent"):
            ql._no_grad(dual, "x")
        with torch.no_grad(), pytest.raises(ValueError, match="x carries a tangent"):      # which is reverse mode's alone
            ql._no_grad(dual, "x")
        with torch.inference_mode():
            ql._no_grad(dual, "x")
        ql._no_grad(dual.detach(), "x")
        ql._no_grad(x, "x")
    ql._no_grad(dual, "x")


def test_sequences_rows_want_a_count_for_each():
    """Too few counts made starts of some of the lengths, and lengths of the table."""
    kv = pkg("kvcache")
    seqs = kv.Sequences(kv.new_cache(4, 1, 16, 16, device="cpu"))
    a, b = seqs.add(), seqs.add()
    seqs.extend([a, b], [20, 3])
    for counts in ([1], [1, 2, 3], [], [1, -1]):
        with pytest.raises(ValueError, match="a count of rows"):
            seqs.rows([a, b], counts)
    rows = seqs.rows([a, b, a], [2, 0, 7])      # (a sequence may be attended twice)
    assert rows.starts.tolist() == [0, 2, 2, 9] and rows.lens.tolist() == [20, 3, 20] and rows.table.shape == (3, 2) and rows.most == 7
    rows = seqs.rows([], [])
    assert rows.starts.tolist() == [0] and rows.lens.shape == (0,) and rows.table.shape == (0, 1) and rows.most == 0
