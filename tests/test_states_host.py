"""Attention to stored states without a GPU: refusals of the C ABI and of the Python side, and the arithmetic that turns device data into
addresses, compiled for the host."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT, pkg

ffi = pkg("ffi")
P = 1 << 20         # an address that is never followed: every call below is refused, or has nothing to do


def _cross(dtype=2, q=P, k=P, v=P, o=P, ws=P, b=2, lq=3, lk=4, h=2, hk=2, d=64, scale=1.0, lens=0, mask=0, kind=0):
    return ffi.raw("gpu_cross_attn", dtype, q, k, v, o, ws, b, lq, lk, h, hk, d, *([64] * 12), scale, lens, mask, kind, 0, 0)


@pytest.mark.parametrize("args,code", [({"dtype": 0}, -4), ({"dtype": 3}, -4), ({"b": -1}, -1), ({"lq": -1}, -1), ({"lk": -1}, -1), ({"h": 3}, -1), ({"hk": 0}, -1), ({"h": 0}, -1),
                                       ({"d": 0}, -1), ({"d": 12}, -1), ({"d": 264}, -1), ({"scale": float("inf")}, -1), ({"scale": float("nan")}, -1), ({"kind": 3}, -1),
                                       ({"kind": 1}, -1), ({"q": 0}, -1), ({"k": 0}, -1), ({"o": 0}, -1), ({"b": 0}, 0), ({"lq": 0}, 0),
                                       ({"lq": 2 ** 31 - 1, "h": 4, "hk": 2}, -1), ({"lq": 1, "lk": 1 << 20, "ws": 0}, -1), ({"lq": 1, "lk": 1 << 20, "ws": P + 8}, -1)])
def test_cross_attn_refusals(args, code):
    assert _cross(**args) == code


def _attn(dtype=2, q=P, o=P, ws=P, k=P, v=P, ks=P, vs=P, pages=4, page=64, starts=P, lens=P, table=P, cols=4, n=2, rows=2, most=1, h=2, hk=2, d=64, scale=1.0):
    return ffi.raw("gpu_kv8_attn", dtype, q, 128, 64, o, 128, 64, ws, k, v, ks, vs, pages, page, starts, lens, table, cols, n, rows, most, h, hk, d, scale, 1, 0)


def _move(name, dtype=2, a=P, b=P, s=128, k=P, v=P, ks=P, vs=P, pages=4, page=64, starts=P, lens=P, table=P, cols=4, n=2, rows=2, most=1, hk=2, d=64):
    return ffi.raw(name, dtype, a, s, 64, b, s, 64, k, v, ks, vs, pages, page, starts, lens, table, cols, n, rows, most, hk, d, 0)


CACHE = [({"k": 0}, -1), ({"v": P + 8}, -1), ({"ks": 0}, -1), ({"vs": P + 2}, -1), ({"pages": 0}, -1), ({"page": 48}, -1), ({"page": 8}, -1), ({"page": 8192}, -1), ({"hk": 0}, -1),
         ({"d": 72}, -1), ({"d": 272}, -1), ({"d": 0}, -1), ({"starts": 0}, -1), ({"lens": 0}, -1), ({"table": 0}, -1), ({"cols": 0}, -1), ({"n": -1}, -1), ({"rows": -1}, -1), ({"most": -1}, -1),
         ({"n": 0}, 0), ({"n": 0, "cols": 0, "table": 0}, 0), ({"rows": 0}, 0), ({"most": 0}, 0)]


@pytest.mark.parametrize("args,code", CACHE + [({"dtype": 0}, -4), ({"h": 3}, -1), ({"scale": float("nan")}, -1), ({"q": 0}, -1), ({"o": 0}, -1), ({"cols": 1 << 16, "ws": 0}, -1)])
def test_cache_attn_refusals(args, code):
    assert _attn(**args) == code


@pytest.mark.parametrize("name", ["gpu_kv8_store", "gpu_kv8_read"])
@pytest.mark.parametrize("args,code", CACHE + [({"dtype": 5}, -4), ({"a": 0}, -1), ({"b": 0}, -1), ({"n": 65536}, -1)])
def test_store_and_read_refusals(name, args, code):
    assert _move(name, **args) == code


def test_store_takes_no_32_bit_rows_and_read_wants_aligned_ones():
    assert _move("gpu_kv8_store", dtype=0) == -4
    assert _move("gpu_kv8_read", a=P + 4) == -1 and _move("gpu_kv8_read", s=130) == -1 and _move("gpu_kv8_read", dtype=0, a=P + 8) == -1


def test_copy_pages_refusals():
    c = lambda k=P, layers=1, pages=4, page=64, hk=2, d=64, src=P, dst=P, n=1: ffi.raw("gpu_kv8_copy_pages", k, P, P, P, layers, pages, page, hk, d, src, dst, n, 0)
    for bad in ({"k": 0}, {"layers": -1}, {"pages": 0}, {"page": 24}, {"hk": 0}, {"d": 8}, {"src": 0}, {"dst": 0}, {"n": -1}, {"n": 65536}, {"layers": 65536}):
        assert c(**bad) == -1, bad
    assert c(n=0) == 0 and c(layers=0) == 0


def test_workspaces():
    """Bytes are asked for where a row's keys are shared by workgroups, and only there."""
    w = ffi.lib.gpu_cross_attn_workspace
    assert w(2, 4096, 77, 10, 10, 64) == 0 and w(0, 1, 1, 1, 1, 64) == 0 and w(1, 1, 100, 3, 2, 64) == 0
    assert w(1, 1, 1 << 16, 8, 8, 128) % 16 == 0 and w(1, 1, 1 << 16, 8, 8, 128) > 0
    assert ffi.lib.gpu_kv8_attn_workspace(1, 1, 32, 8, 128, 64, 1024) > 0 and ffi.lib.gpu_kv8_attn_workspace(1, 1, 32, 8, 128, 64, 1) == 0


def _plan(rows, problems, keys, d, bytes):
    out = (ctypes.c_int32 * 3)()
    ffi.k("gpu_internal_states_plan", rows, problems, keys, d, bytes, ctypes.cast(out, ctypes.c_void_p))
    return tuple(out)[:2]


@pytest.mark.parametrize("case,plan", [
    ((4096, 20, 77, 64, 2), (128, 1)),          # SDXL's prompt keys: short, many rows
    ((8192, 40, 512, 128, 2), (128, 1)),        # 142 us against 149 with tiles of 256 rows
    ((1111, 48, 4608, 128, 2), (256, 1)),       # 175 against 191; in two parts 217 to 230
    ((4096, 16, 8192, 128, 1), (256, 1)),       # 284 against 324; in two parts 336
    ((2025, 16, 16256, 64, 1), (256, 4)),       # 200 against 218 in two parts, 357 in one
    ((4, 96, 32752, 128, 1), (16, 8)),          # one full round: 130 against 138 and 154 in 5 and 6 parts
    ((1, 64, 1369, 72, 2), (16, 6)), ((20, 8, 4096, 128, 1), (32, 32)), ((33, 1, 64, 256, 2), (128, 1)), ((1, 1, 0, 8, 2), (16, 1)), ((1, 2000, 100000, 128, 1), (16, 8)), ((200, 1, 1010, 128, 2), (128, 6)), ((96, 24, 4608, 128, 2), (128, 9)),
    ((1024, 16, 1000, 192, 2), (128, 4)), ((83, 80, 524, 168, 2), (128, 3)), ((962, 20, 773, 256, 2), (128, 1)), ((2004, 132, 225, 256, 2), (256, 1)), ((4096, 16, 1024, 72, 2), (256, 1))])
def test_attention_forms_where_they_were_measured(case, plan):
    """For 256 CUs, which is what a host without a device is taken for."""
    assert _plan(*case) == plan


def test_python_side_refuses_host_tensors():
    ql, kv = pkg("qlinear"), pkg("kvcache")
    x = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ql.cross_attn(x, x, x, 1.0)
    cache = kv.new_cache(2, 2, 64, 32, device="cpu")
    i = torch.zeros(2, dtype=torch.int32)
    rows = kv.Rows(i, i[:1], i[:1, None], 1)
    for call in (lambda: kv.store(cache, rows, x[0], x[0]), lambda: kv.read(cache, rows, 1), lambda: kv.attn(x[0], cache, rows, 1.0), lambda: kv.copy_pages(cache, i, i)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    layered = kv.new_cache(2, 2, 64, 32, layers=3, device="cpu")
    assert layered.k.shape == (3, 2, 2, 32, 64) and layered.layer(1).k_scale.shape == (2, 2, 2)


PLACES = r"""
#include "kv8.hpp"
#include <cstdio>
#include <vector>
int main() {
    // every table entry, block and descriptor that device data may hold ends inside the arrays, or nowhere
    const int odd[] = {0, 1, 2, 3, 4, 5, 63, -1, -2147483647 - 1, 2147483647, 1 << 30, (1 << 30) + 1};
    for (int shift = 4; shift <= 12; ++shift)
        for (int cols = 1; cols <= 3; ++cols)
            for (int x : odd) for (int y : odd) for (int n_pages : {1, 4}) {
                std::vector<int32_t> table(cols, x);
                const int page = page_of(table.data(), cols, n_pages, shift, y);
                const bool inside = y >= 0 && (y >> (shift - 4)) < cols && x >= 0 && x < n_pages;
                if ((page >= 0) != inside || (inside && page != x)) return 1;
                if (!inside) continue;
                for (int hk : {1, 3}) for (int head = 0; head < hk; ++head) {
                    const int64_t scale = scale_at(page, hk, head, shift, y), code = codes_at(page, hk, head, shift, y, 48);
                    const int64_t tokens = (int64_t)n_pages * hk << shift;
                    if (scale < 0 || scale >= tokens / kBlock || code != scale * kBlock * 48 || code + kBlock * 48 > tokens * 48) return 2;
                }
            }
    for (int a : odd) for (int b : odd) for (int l : odd) for (int rows : {0, 5, 2147483647}) for (int most : {0, 3, 2147483647}) {
        const int32_t starts[2] = {a, b}, lens[1] = {l};
        const Span s = span(starts, lens, 0, rows, most);
        if (s.first < 0 || s.count < 0 || s.count > most || (int64_t)s.first + s.count > rows || s.len < 0 || s.len > kMostTokens) return 3;
        if (a >= 0 && b >= a && b <= rows && b - a <= most && (s.first != a || s.count != b - a)) return 4;
        if (l >= 0 && l <= kMostTokens && s.len != l) return 5;
    }
    // offsets that pass 32 bits
    if (codes_at(2000000, 8, 7, 6, 3, 128) != ((2000000LL * 8 + 7) * 64 + 48) * 128) return 6;
    std::puts("ok");
    return 0;
}
"""


def test_device_data_becomes_addresses_inside_the_cache(tmp_path):
    src = tmp_path / "places.cpp"
    src.write_text(PLACES)
    exe = str(tmp_path / "places")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-ftrapv", "-I",
                           os.path.join(ROOT, "comfyui-backend-but-rust_amd", "csrc"), str(src), "-o", exe])
    assert subprocess.check_output([exe], text=True) == "ok\n"


def _host_copy(cache, src, dst):
    src, dst = src.tolist(), dst.tolist()
    assert not set(src) & set(dst) and len(set(dst)) == len(dst)
    axis = cache.k.dim() - 4
    for t in cache:
        t.index_copy_(axis, torch.tensor(dst), t.index_select(axis, torch.tensor(src)))


def _write(seqs, rows, ids, held, first):
    """Marks every new token in its place, as a store would."""
    k = seqs.cache.k
    for i, s in enumerate(ids):
        n = int(rows.starts[i + 1] - rows.starts[i])
        for j in range(n):
            t = int(rows.lens[i]) - n + j
            held[s].append((first + j) % 120 + 1)
            k[..., int(rows.table[i, t // seqs.page]), 0, t % seqs.page, 0] = held[s][-1]
        first += n
    return first


def _holds(seqs, s, held):
    k = seqs.cache.k.flatten(0, -5)[0] if seqs.cache.k.dim() == 5 else seqs.cache.k
    return [int(k[seqs.pages(s)[t // seqs.page], 0, t % seqs.page, 0]) for t in range(seqs.length(s))] == held[s]


@pytest.mark.parametrize("layers", [None, 2])
def test_sequences_share_copy_and_move_pages(layers, monkeypatch):
    """Forks, cuts, ends, growth and compaction in any order: every sequence keeps its own tokens, and no page is lost."""
    import random
    kv = pkg("kvcache")
    monkeypatch.setattr(kv, "copy_pages", _host_copy)
    for seed in range(6):
        rng = random.Random(seed)
        seqs = kv.Sequences(kv.new_cache(24, 1, 16, 16, layers, device="cpu"))
        held, first = {}, 0
        for _ in range(150):
            what = rng.choice(("add", "extend", "extend", "extend", "fork", "fork", "truncate", "free", "compact"))
            ids = sorted(held)
            if what == "add" or not ids:
                held[seqs.add()] = []
            elif what == "fork":
                s = rng.choice(ids)
                held[seqs.fork(s)] = list(held[s])
            elif what == "truncate":
                s = rng.choice(ids)
                held[s] = held[s][:rng.randint(0, len(held[s]))]
                seqs.truncate(s, len(held[s]))
            elif what == "free":
                s = rng.choice(ids)
                seqs.free(s)
                del held[s]
            elif what == "compact":
                seqs.compact()
                used = {p for s in held for p in seqs.pages(s)}
                assert used == set(range(len(used)))
            else:
                some = rng.sample(ids, rng.randint(1, min(4, len(ids))))
                counts = [rng.choice((0, 1, 1, 5, 16, 40)) for _ in some]
                before = (seqs.unused, [seqs.pages(s) for s in ids], [seqs.length(s) for s in ids])
                try:
                    rows = seqs.extend(some, counts)
                except kv.CacheFull:
                    assert before == (seqs.unused, [seqs.pages(s) for s in ids], [seqs.length(s) for s in ids])
                    continue
                assert rows.most == max(counts) and rows.starts.tolist()[-1] == sum(counts)
                first = _write(seqs, rows, some, held, first)
            assert all(seqs.length(s) == len(h) and _holds(seqs, s, held) for s, h in held.items()), (seed, what)
            assert seqs.unused == 24 - len({p for s in held for p in seqs.pages(s)})
        for s in list(held):
            seqs.free(s)
        assert seqs.unused == 24


def test_sequences_refuse():
    kv = pkg("kvcache")
    seqs = kv.Sequences(kv.new_cache(2, 1, 16, 16, device="cpu"))
    a = seqs.add()
    for bad in (lambda: seqs.extend([a, a], [1, 1]), lambda: seqs.extend([a], [1, 2]), lambda: seqs.extend([a], [-1]), lambda: seqs.truncate(a, 1), lambda: seqs.truncate(a, -1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(kv.CacheFull):
        seqs.extend([a], [33])
    with pytest.raises(KeyError):
        seqs.free(a + 1)
    rows = seqs.rows([a], [0])
    assert rows.table.shape == (1, 1) and rows.table.item() == -1 and rows.most == 0
