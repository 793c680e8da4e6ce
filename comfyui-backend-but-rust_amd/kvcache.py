"""Keys and values that are made once and attended many times, in pages of 8-bit codes with a scale for each 16 tokens of a head:
an encoder's states over all steps of a sampler, the frames of a stream, the tokens of a prompt model.

`Cache` names the device arrays, `Rows` which rows of a call belong to which sequence and where its tokens lie; both are plain tuples, so a
program may keep the tensors as it likes.  The formats and what every call does with them stand in include/gpu_api.h.  Nothing here waits for
the GPU; calls are queued on the current stream of the tensors' device.  There is no backward pass and no forward mode: inputs that ask for
gradients or carry tangents are refused.
"""
from typing import NamedTuple

import torch

from . import ffi, qlinear

BLOCK = 16          # tokens that share a scale
_DT = {torch.float16: ffi.DT_F16, torch.bfloat16: ffi.DT_BF16}


class Cache(NamedTuple):
    k: torch.Tensor             # int8 [pages, heads, page, d], or [layers, pages, heads, page, d]
    v: torch.Tensor
    k_scale: torch.Tensor       # float32 [(layers,) pages, heads, page // 16]: the largest magnitude A; a code c stands for c * A / 127
    v_scale: torch.Tensor

    def layer(self, i):
        return Cache(self.k[i], self.v[i], self.k_scale[i], self.v_scale[i])


class Rows(NamedTuple):
    starts: torch.Tensor        # int32 [n + 1]: rows starts[s] .. starts[s + 1] of a call are the last tokens of sequence s
    lens: torch.Tensor          # int32 [n]: tokens that the sequence holds, the new ones among them
    table: torch.Tensor         # int32 [n, pages of a sequence]: token t lies in page table[s, t // page]
    most: int                   # rows of the sequence that has the most in this call, or a bound; one below that misplaces the rows above it


def new_cache(pages, heads, dim, page=64, layers=None, device="cuda:0"):
    """An empty cache: of one layer, or with an axis of layers in front."""
    if page < BLOCK or page > 4096 or page & (page - 1):
        raise ValueError("a page holds a power of two tokens from 16 to 4096, got %d" % page)
    if dim % 16 or not 16 <= dim <= 256:
        raise ValueError("head dims are multiples of 16 up to 256, got %d" % dim)
    shape = ((layers,) if layers is not None else ()) + (pages, heads, page, dim)
    codes = [torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2)]
    return Cache(*codes, *(torch.zeros(shape[:-2] + (page // BLOCK,), dtype=torch.float32, device=device) for _ in range(2)))


def _cache(cache, dims):
    k = cache.k
    if k.dtype != torch.int8 or k.dim() != dims or not k.is_cuda or not k.is_contiguous():
        raise ValueError("cache.k must be a contiguous int8 CUDA tensor of %d axes, got %s %s" % (dims, k.dtype, tuple(k.shape)))
    v = cache.v
    if v.dtype != torch.int8 or v.shape != k.shape or v.device != k.device or not v.is_contiguous():
        raise ValueError("cache.v must be like cache.k, got %s %s" % (v.dtype, tuple(v.shape)))
    want = k.shape[:-2] + (k.shape[-2] // BLOCK,)
    for t, what in ((cache.k_scale, "cache.k_scale"), (cache.v_scale, "cache.v_scale")):
        if t.dtype != torch.float32 or t.shape != want or t.device != k.device or not t.is_contiguous():
            raise ValueError("the cache's scales must be contiguous float32 %s on its device, got %s %s" % (tuple(want), t.dtype, tuple(t.shape)))
        qlinear._no_grad(t, what)
    return k.shape


def _row_args(rows, device):
    n = rows.lens.shape[0] if rows.lens.dim() == 1 else -1
    for t, shape in ((rows.starts, (n + 1,)), (rows.lens, (n,)), (rows.table, (n, rows.table.shape[-1]))):
        if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != device or not t.is_contiguous():
            raise ValueError("rows.starts [n + 1], lens [n] and table [n, m] must be contiguous int32 on the cache's device, got %s %s on %s"
                             % (t.dtype, tuple(t.shape), t.device))
    return rows.starts.data_ptr(), rows.lens.data_ptr(), rows.table.data_ptr(), rows.table.shape[1], n


def _heads(t, heads, dim, what, device):
    if t.dim() != 3 or t.shape[1] != heads and heads is not None or t.shape[2] != dim or t.stride(2) != 1 or t.device != device:
        raise ValueError("%s must be [rows, %s, %d] on the cache's device with a dense last axis, got %s with strides %s on %s"
                         % (what, "heads" if heads is None else heads, dim, tuple(t.shape), t.stride(), t.device))
    if t.dtype not in _DT:
        raise ValueError("%s must be float16 or bfloat16, got %s" % (what, t.dtype))
    qlinear._no_grad(t, what)


def store(cache, rows, k, v):
    """The rows of k and v ([rows, heads, d], bf16 or f16) become the last tokens of their sequences."""
    if qlinear._pycalls is None or qlinear._pycalls.kv8_store(k, v, *cache, *rows) is None:
        _store(cache, rows, k, v)


def _store(cache, rows, k, v):
    """The calls in Python, here and below: what the native ones leave to them, and every refusal."""
    pages, heads, page, dim = _cache(cache, 4)
    dev = cache.k.device
    _heads(k, heads, dim, "k", dev); _heads(v, heads, dim, "v", dev)
    if v.shape[0] != k.shape[0] or v.dtype != k.dtype:
        raise ValueError("k and v must have the same rows and type, got %s %s and %s %s" % (tuple(k.shape), k.dtype, tuple(v.shape), v.dtype))
    args = _row_args(rows, dev)
    with qlinear._on(dev) as s:
        ffi.k("gpu_kv8_store", _DT[k.dtype], k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), cache.k.data_ptr(),
              cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), pages, page, *args, k.shape[0], rows.most, heads, dim, s)


def read(cache, rows, tokens, dtype=torch.bfloat16):
    """The last tokens of the sequences as (k, v), each [tokens, heads, d]; tokens: all rows of the call, rows.starts[-1].  Rows of no
    sequence are left uninitialised."""
    kv = None if qlinear._pycalls is None else qlinear._pycalls.kv8_read(*cache, *rows, tokens, dtype)
    return _read(cache, rows, tokens, dtype) if kv is None else kv


def _read(cache, rows, tokens, dtype):
    pages, heads, page, dim = _cache(cache, 4)
    dev = cache.k.device
    if dtype not in qlinear._TORCH_DT:
        raise ValueError("tokens are read back as float32, float16 or bfloat16, not %s" % dtype)
    args = _row_args(rows, dev)
    k, v = (torch.empty((tokens, heads, dim), dtype=dtype, device=dev) for _ in range(2))
    with qlinear._on(dev) as s:
        ffi.k("gpu_kv8_read", qlinear._TORCH_DT[dtype], k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
              cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), pages, page, *args, tokens, rows.most,
              heads, dim, s)
    return k, v


def attn(q, cache, rows, scale, causal=True, out=None):
    """softmax(scale * q k^T) v over the stored tokens: q [rows, h, d] (bf16 or f16), h a multiple of the cache's heads.  Causal: a row sees the
    tokens up to its own place; otherwise all that its sequence holds.  Rows of no sequence are left as they are in `out`.  rows.most decides how
    all of the call runs: single tokens and long pieces of prompts are better two calls."""
    o = None if out is not None or qlinear._pycalls is None else qlinear._pycalls.kv8_attn(q, *cache, *rows, float(scale), bool(causal))
    return _attn(q, cache, rows, scale, causal, out) if o is None else o


def _attn(q, cache, rows, scale, causal, out):
    pages, heads, page, dim = _cache(cache, 4)
    dev = cache.k.device
    _heads(q, None, dim, "q", dev)
    h = q.shape[1]
    if h == 0 or h % heads:
        raise ValueError("q has %d heads, which is no multiple of the cache's %d" % (h, heads))
    o = torch.empty(q.shape, dtype=q.dtype, device=dev) if out is None else out
    if out is not None:
        _heads(o, h, dim, "out", dev)
        if o.dtype != q.dtype or o.shape != q.shape:
            raise ValueError("out must be %s %s, got %s %s" % (q.dtype, tuple(q.shape), o.dtype, tuple(o.shape)))
    args = _row_args(rows, dev)
    with qlinear._on(dev) as s:
        need = ffi.lib.gpu_kv8_attn_workspace(args[4], rows.most, h, heads, dim, page, args[3])
        ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
        ffi.k("gpu_kv8_attn", _DT[q.dtype], q.data_ptr(), q.stride(0), q.stride(1), o.data_ptr(), o.stride(0), o.stride(1), qlinear._ptr(ws),
              cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), pages, page, *args, q.shape[0], rows.most,
              h, heads, dim, float(scale), 1 if causal else 0, s)
    return o


def copy_pages(cache, src, dst):
    """Pages src[i] -> dst[i] (int32 tensors on the cache's device), scales and all layers included.  No page may be named twice in dst, or in
    both: the copies run side by side."""
    if qlinear._pycalls is None or qlinear._pycalls.kv8_copy_pages(*cache, src, dst) is None:
        _copy_pages(cache, src, dst)


def _copy_pages(cache, src, dst):
    layered = cache.k.dim() == 5
    shape = _cache(cache, 5 if layered else 4)
    pages, heads, page, dim = shape[-4:]
    dev = cache.k.device
    for t in (src, dst):
        if t.dtype != torch.int32 or t.dim() != 1 or t.device != dev or not t.is_contiguous() or t.shape != src.shape:
            raise ValueError("src and dst must be contiguous int32 [n] on the cache's device, got %s %s on %s" % (t.dtype, tuple(t.shape), t.device))
    with qlinear._on(dev) as s:
        ffi.k("gpu_kv8_copy_pages", cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
              shape[0] if layered else 1, pages, page, heads, dim, src.data_ptr(), dst.data_ptr(), src.shape[0], s)


class CacheFull(RuntimeError):
    pass


class Sequences:
    """Which pages hold which sequence: taken as sequences grow, shared by forks, copied before a shared one is written, given back, moved down.

    The book is kept on the host; what a call needs of it goes to the device with the call, and pages are moved by queued copies.  All calls on
    the cache are made on one stream, or ordered by the caller.  Pages' contents stay when they are given back: nothing reads them before they are
    written again.  Nothing here can be captured into a graph (a captured call's Rows are tensors that the program fills itself)."""

    def __init__(self, cache):
        self.cache = cache
        self.page = cache.k.shape[-2]
        self._users = [0] * cache.k.shape[-4]
        self._unused = list(range(len(self._users)))[::-1]      # the lowest is taken first
        self._seqs = {}                                         # id -> [pages, length]
        self._ids = 0

    def add(self):
        """A new, empty sequence."""
        self._ids += 1
        self._seqs[self._ids] = [[], 0]
        return self._ids

    def length(self, seq):
        return self._seqs[seq][1]

    def pages(self, seq):
        return list(self._seqs[seq][0])

    @property
    def unused(self):
        """Pages that nobody holds."""
        return len(self._unused)

    def fork(self, seq):
        """A new sequence of the same tokens, in the same pages until one of the two writes."""
        pages, length = self._seqs[seq]
        new = self.add()
        self._seqs[new] = [list(pages), length]
        for p in pages:
            self._users[p] += 1
        return new

    def truncate(self, seq, length):
        """Drops the tokens from `length` on."""
        s = self._seqs[seq]
        if not 0 <= length <= s[1]:
            raise ValueError("sequence %d has %d tokens, not %d" % (seq, s[1], length))
        keep = -(-length // self.page)
        self._give_back(s[0][keep:])
        del s[0][keep:]
        s[1] = length

    def free(self, seq):
        self._give_back(self._seqs.pop(seq)[0])

    def extend(self, seqs, counts):
        """Room for counts[i] more tokens at the end of seqs[i]; returns the Rows that store them, and that attend as them.  Raises CacheFull,
        and changes nothing, where the pages do not suffice."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("extend wants every sequence once, and a count of tokens for each")
        need, users = 0, dict()
        for s, c in zip(seqs, counts):
            pages, length = self._seqs[s]
            need += -(-(length + c) // self.page) - len(pages)
            if c and length % self.page:
                last = pages[-1]
                users[last] = users.get(last, self._users[last]) - 1
                need += users[last] > 0     # somebody else has it still: this one writes into a copy
        if need > len(self._unused):
            raise CacheFull("%d pages wanted, %d unused" % (need, len(self._unused)))
        src, dst = [], []
        for s, c in zip(seqs, counts):
            entry = self._seqs[s]
            pages, length = entry
            if c and length % self.page and self._users[pages[-1]] > 1:
                self._users[pages[-1]] -= 1
                src.append(pages[-1])
                pages[-1] = self._take()
                dst.append(pages[-1])
            while len(pages) * self.page < length + c:
                pages.append(self._take())
            entry[1] = length + c
        self._copy(src, dst)
        return self.rows(seqs, counts)

    def rows(self, seqs, counts):
        """Rows of counts[i] queries each to what seqs[i] hold: their last tokens (causal), or rows of something else (not causal)."""
        if len(seqs) != len(counts) or any(c < 0 for c in counts):
            raise ValueError("rows wants a count of rows for every sequence, got %d sequences and counts %s" % (len(seqs), list(counts)))
        n, cols = len(seqs), max([len(self._seqs[s][0]) for s in seqs] + [1])
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        flat = starts + [self._seqs[s][1] for s in seqs]
        for s in seqs:
            pages = self._seqs[s][0]
            flat += pages + [-1] * (cols - len(pages))
        t = self._upload(flat)
        return Rows(t[:n + 1], t[n + 1:2 * n + 1], t[2 * n + 1:].view(n, cols), max([0, *counts]))

    def compact(self):
        """Moves pages down into unused ones until the used ones are the lowest; returns how many moved.  Rows made before name the old places."""
        used = [p for p, u in enumerate(self._users) if u]
        dst = [p for p in range(len(used)) if not self._users[p]]
        src = used[len(used) - len(dst):]
        where = dict(zip(src, dst))
        self._copy(src, dst)
        for a, b in where.items():
            self._users[a], self._users[b] = 0, self._users[a]
        for entry in self._seqs.values():
            entry[0] = [where.get(p, p) for p in entry[0]]
        self._unused = list(range(len(used), len(self._users)))[::-1]
        return len(src)

    def _take(self):
        p = self._unused.pop()
        self._users[p] = 1
        return p

    def _give_back(self, pages):
        for p in pages:
            self._users[p] -= 1
            if not self._users[p]:
                self._unused.append(p)

    def _copy(self, src, dst):
        for i in range(0, len(src), 32768):
            t = self._upload(src[i:i + 32768] + dst[i:i + 32768])
            n = t.shape[0] // 2
            copy_pages(self.cache, t[:n], t[n:])

    def _upload(self, numbers):
        dev = self.cache.k.device
        return torch.tensor(numbers, dtype=torch.int32, pin_memory=dev.type == "cuda").to(dev, non_blocking=True)
