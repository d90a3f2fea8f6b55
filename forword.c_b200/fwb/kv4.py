"""Several sequences served from one paged cache of 4-bit keys and values: the
operators of include/forword_b200.h on torch CUDA tensors.

``empty``         memory for a cache
``append``        new tokens: queries and keys rotated, keys and values quantised into their pages
``Attention``     attention of the newest tokens over their sequences' pages
``read``          what the cache holds, as values
``check_status``  whether every call so far stayed inside its tables

A cache is a uint8 tensor [n_page, n_head_kv, page bytes]; the page size
follows from it and head_dim.  Page tables are int32 [n_seq, max_pages],
lengths int32 [n_seq] and count a sequence's new tokens; a padded batch says
with n_new how many of a sequence's n_query tokens there are.

Thin plumbing over the CUDA library (no CPU fallback), on the current stream
of torch and the current device.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import native
from .beam import TYPE_IDS, _capturing, _Plan, _raw_stream, _refuse
from .model import FwbError, _err

_u32, _u64, _vp = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_void_p


def _strides(what: str):
    return [(f"{what}_{n}_stride", _u64) for n in ("seq", "token", "head")]


class AppendArgs(ctypes.Structure):
    """fwb_kv4_append_t."""
    _fields_ = ([(n, _u32) for n in ("type", "n_seq", "n_query", "n_head", "n_head_kv", "head_dim", "page_size", "n_page",
                                     "max_pages", "n_pos", "halves")]
                + [("q", _vp)] + _strides("q") + [("k", _vp), ("v", _vp)] + _strides("k") + _strides("v")
                + [("q_out", _vp)] + _strides("q_out") + [("cache", _vp), ("pages", _vp), ("pages_stride", _u64)]
                + [(n, _vp) for n in ("lengths", "n_new", "cos", "sin")])


class ReadArgs(ctypes.Structure):
    """fwb_kv4_read_t."""
    _fields_ = ([(n, _u32) for n in ("type", "n_seq", "n", "n_head_kv", "head_dim", "page_size", "n_page", "max_pages")]
                + [("cache", _vp), ("pages", _vp), ("pages_stride", _u64)]
                + [(n, _vp) for n in ("start", "lengths", "k", "v")])


class AttnArgs(ctypes.Structure):
    """fwb_kv4_attn_t."""
    _fields_ = ([(n, _u32) for n in ("type", "n_seq", "n_query", "n_head", "n_head_kv", "head_dim", "page_size", "n_page",
                                     "max_pages")]
                + [("scale", ctypes.c_float), ("q", _vp)] + _strides("q")
                + [("cache", _vp), ("pages", _vp), ("pages_stride", _u64)]
                + [(n, _vp) for n in ("lengths", "n_new", "out", "lse")])


@functools.lru_cache(maxsize=256)
def page_bytes(head_dim: int, page_size: int) -> int:
    """Bytes of a page for one head (fwb_kv4_page_bytes)."""
    if not 0 <= head_dim < 1 << 32 or not 0 <= page_size < 1 << 32:
        raise ValueError("size out of range")
    lib = native.product()
    n = int(lib.fwb_kv4_page_bytes(head_dim, page_size))
    if not n:
        raise FwbError(_err(lib))
    return n


def empty(n_page: int, n_head_kv: int, head_dim: int, page_size: int, device=None) -> torch.Tensor:
    """Memory for a cache of n_page pages of page_size positions."""
    return torch.empty(n_page, n_head_kv, page_bytes(head_dim, page_size), dtype=torch.uint8,
                       device="cuda" if device is None else device)


@functools.lru_cache(maxsize=256)
def _page_size(head_dim: int, line: int) -> int:
    for n in (16, 32, 64, 128, 256):
        if page_bytes(head_dim, n) == line:
            return n
    raise ValueError(f"cache: a line of {line} bytes is no page of head_dim {head_dim}")


def _refuse_cache(cache, heads: int, dev: int):
    if cache is None:
        raise ValueError("cache is missing")
    raise ValueError(f"cache: expected contiguous torch.uint8 [n_page, {heads}, page bytes] on cuda:{dev}, "
                     f"got {cache.dtype} {tuple(cache.shape)} on {cache.device}")


def _refuse_pages(pages, n: int, dev: int):
    if pages is None:
        raise ValueError("pages is missing")
    raise ValueError(f"pages: expected torch.int32 [{n}, max_pages] on cuda:{dev}, the last dimension contiguous, "
                     f"got {pages.dtype} {tuple(pages.shape)} on {pages.device}")


def _tables(a, cache, pages, n: int, heads: int, head_dim: int, dev: int) -> None:
    """The arguments of a cache and its page table."""
    if (cache is None or cache.dtype is not torch.uint8 or cache.dim() != 3 or (cs := cache.shape)[1] != heads
            or cache.get_device() != dev or not cache.is_contiguous()):
        _refuse_cache(cache, heads, dev)
    a.page_size, a.n_page, a.cache = _page_size(head_dim, cs[2]), cs[0], cache.data_ptr()
    if (pages is None or pages.dtype is not torch.int32 or pages.dim() != 2 or (ps := pages.shape)[0] != n
            or pages.get_device() != dev or ((st := pages.stride())[1] != 1 and ps[1] > 1)):
        _refuse_pages(pages, n, dev)
    a.max_pages, a.pages_stride, a.pages = ps[1], st[0], pages.data_ptr()


def _ints(t, what: str, shape, dev: int) -> int:
    if t is None or t.dtype is not torch.int32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        _refuse(t, what, shape, torch.int32, dev)
    return t.data_ptr()


def _meet(levels, off: int, run: int) -> bool:
    """Whether runs share a byte with ones of the same layout `off` bytes on; levels: (count, stride) of them, the widest
    stride first, each level not reaching past the stride before it."""
    if not levels:
        return -run < off < run
    (n, stride), *inner = levels
    i = off // stride
    return any(-n < j < n and _meet(inner, off - j * stride, run) for j in (i, i + 1))


def _overlap(a, b) -> bool:
    """Whether rows of two tensors of one shape share memory without being the same rows."""
    off, size = b.data_ptr() - a.data_ptr(), a.element_size()
    if a.is_contiguous() and b.is_contiguous():
        return off != 0 and abs(off) < a.numel() * size
    run = a.shape[3] * size
    one, other = ([(n, s * size) for n, s in zip(t.shape[:3], t.stride()) if n > 1] for t in (a, b))
    if one == other:
        levels = sorted(one, key=lambda level: -level[1])
        return off != 0 and all(s for _, s in levels) and _meet(levels, off, run)
    return -sum((n - 1) * s for n, s in other) - run < off < sum((n - 1) * s for n, s in one) + run


def append(q, k, v, cache, pages, lengths, cos=None, sin=None, halves: bool = False, n_new=None, q_out=None):
    """New tokens into the cache (fwb_kv4_append_dev) -> q_out, the rotated queries.

    q [n_seq, n_query, n_head, head_dim] or None, k and v [n_seq, n_query,
    n_head_kv, head_dim]: views with a contiguous last dimension, addresses
    and strides multiples of 16 bytes.  cos and sin fp32 [n_pos, head_dim/2],
    None: no rotation; halves: pairs (i, i + head_dim/2) are turned instead of
    neighbours.  q_out may be q itself, or memory apart from all that is read, in
    the gaps between q's rows too; rows of tokens without a position (of a padded
    batch, below position 0, past the tables) are left as they were: where q_out is
    None zeros, but with n_new None whatever was there.
    """
    if k is None or k.dim() != 4:
        raise ValueError("k must be [n_seq, n_query, n_head_kv, head_dim]")
    dt, dev, shape = k.dtype, k.get_device(), k.shape
    kind = TYPE_IDS.get(dt)
    if kind is None:
        raise ValueError(f"dtype must be one of {list(TYPE_IDS)}")
    if dev < 0 or torch.cuda.current_device() != dev:
        raise ValueError("append: k and the current device differ")
    n_seq, n_query, heads, hd = shape
    a = AppendArgs(kind, n_seq, n_query, 0, heads, hd)
    if (st := k.stride())[3] != 1:
        _refuse(k, "k", shape, dt, dev)
    a.k, a.k_seq_stride, a.k_token_stride, a.k_head_stride = k.data_ptr(), st[0], st[1], st[2]
    if v is None or v.dtype is not dt or v.shape != shape or v.get_device() != dev or (st := v.stride())[3] != 1:
        _refuse(v, "v", shape, dt, dev)
    a.v, a.v_seq_stride, a.v_token_stride, a.v_head_stride = v.data_ptr(), st[0], st[1], st[2]
    _tables(a, cache, pages, n_seq, heads, hd, dev)
    a.lengths = _ints(lengths, "lengths", (n_seq,), dev)
    if n_new is not None:
        a.n_new = _ints(n_new, "n_new", (n_seq,), dev)
    if q is not None:
        if q.dim() != 4:
            raise ValueError("q must be [n_seq, n_query, n_head, head_dim]")
        qs = q.shape
        if (q.dtype is not dt or qs[0] != n_seq or qs[1] != n_query or qs[3] != hd or q.get_device() != dev
                or (st := q.stride())[3] != 1):
            _refuse(q, "q", torch.Size((n_seq, n_query, qs[2], hd)), dt, dev)
        a.n_head, a.q, a.q_seq_stride, a.q_token_stride, a.q_head_stride = qs[2], q.data_ptr(), st[0], st[1], st[2]
        if q_out is None:
            q_out = (torch.empty if n_new is None else torch.zeros)(qs, dtype=dt, device=k.device)
            so = q_out.stride()
        elif q_out.dtype is not dt or q_out.shape != qs or q_out.get_device() != dev or (so := q_out.stride())[3] != 1:
            _refuse(q_out, "q_out", qs, dt, dev)
        elif q_out is not q and (so != st or q_out.data_ptr() != a.q) and _overlap(q, q_out):
            raise ValueError("q_out must be q itself or memory apart from it")
        a.q_out, a.q_out_seq_stride, a.q_out_token_stride, a.q_out_head_stride = q_out.data_ptr(), so[0], so[1], so[2]
    elif q_out is not None:
        raise ValueError("q_out without q")
    if cos is not None or sin is not None:
        for t, what in ((cos, "cos"), (sin, "sin")):
            if (t is None or t.dtype is not torch.float32 or t.dim() != 2 or t.shape[1] * 2 != hd or t.get_device() != dev
                    or not t.is_contiguous()):
                raise ValueError(f"{what}: expected contiguous torch.float32 [n_pos, {hd // 2}] on cuda:{dev}")
        if cos.shape != sin.shape:
            raise ValueError("cos and sin must have the same shape")
        a.cos, a.sin, a.n_pos = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    if halves:
        a.halves = 1
    lib = native.product()
    if lib.fwb_kv4_append_dev(ctypes.byref(a), _raw_stream(dev)) != 0:
        raise FwbError(_err(lib))
    return q_out


def read(cache, pages, start, n: int, *, head_dim: int, dtype: torch.dtype, lengths=None, k=None, v=None):
    """Positions start[s] .. start[s] + n - 1 of every sequence (fwb_kv4_read_dev)
    -> (k, v), each [n_seq, n, n_head_kv, head_dim]; zeros at and past lengths."""
    kind = TYPE_IDS.get(dtype)
    if kind is None:
        raise ValueError(f"dtype must be one of {list(TYPE_IDS)}")
    if cache is None or cache.dim() != 3:
        raise ValueError("cache must be [n_page, n_head_kv, page bytes]")
    if start is None or start.dim() != 1:
        raise ValueError("start must be [n_seq]")
    dev, heads, n_seq = cache.get_device(), cache.shape[1], start.shape[0]
    if dev < 0 or torch.cuda.current_device() != dev:
        raise ValueError("read: the cache and the current device differ")
    if not 0 <= n < 1 << 32:
        raise ValueError(f"size {n} out of range")
    a = ReadArgs(kind, n_seq, n, heads, head_dim)
    _tables(a, cache, pages, n_seq, heads, head_dim, dev)
    a.start = _ints(start, "start", (n_seq,), dev)
    if lengths is not None:
        a.lengths = _ints(lengths, "lengths", (n_seq,), dev)
    if k is None and v is None:
        k, v = cache.new_empty((2, n_seq, n, heads, head_dim), dtype=dtype).unbind()
    else:
        shape = torch.Size((n_seq, n, heads, head_dim))
        k, v = (cache.new_empty(shape, dtype=dtype) if t is None else t for t in (k, v))
        for t, what in ((k, "k"), (v, "v")):
            if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
                _refuse(t, what, shape, dtype, dev)
    a.k, a.v = k.data_ptr(), v.data_ptr()
    lib = native.product()
    if lib.fwb_kv4_read_dev(ctypes.byref(a), _raw_stream(dev)) != 0:
        raise FwbError(_err(lib))
    return k, v


class Attention(_Plan):
    """Plan of fwb_kv4_attention_dev for fixed sizes.

    plan(q, cache, pages, lengths, n_new=None, out=None, lse=None) -> (out, lse):

    q      [n_seq, n_query, n_head, head_dim] (a view with a contiguous last
           dimension, address and strides multiples of 16 bytes)
    cache  uint8 [n_page, n_head_kv, page bytes]
    pages  int32 [n_seq, max_pages], lengths and n_new int32 [n_seq]
    out    like q, contiguous; lse fp32 [n_seq, n_query, n_head]: memory apart
           from all that is read.  Rows of
           tokens that a padded batch lacks are left as they were (zeros
           where out and lse are None)

    One plan is used from one thread at a time; each stream that it is used on
    gets a workspace of its own, and so does each call captured into a CUDA
    graph, from the graph's memory pool.
    """

    def __init__(self, *, n_seq: int, n_head: int, n_head_kv: int, head_dim: int, dtype: torch.dtype, page_size: int,
                 n_page: int, max_pages: int, n_query: int = 1, scale: float = 0.0, device: int | None = None):
        if dtype not in TYPE_IDS:
            raise ValueError(f"dtype must be one of {list(TYPE_IDS)}")
        for x in (n_seq, n_head, n_head_kv, head_dim, page_size, n_page, max_pages, n_query):
            if not 0 <= x < 1 << 32:
                raise ValueError(f"size {x} out of range")
        a = self.a = AttnArgs(type=TYPE_IDS[dtype], n_seq=n_seq, n_query=n_query, n_head=n_head, n_head_kv=n_head_kv,
                              head_dim=head_dim, page_size=page_size, n_page=n_page, max_pages=max_pages, scale=scale)
        self._ref = ctypes.byref(a)
        super().__init__(device, lambda: native.product().fwb_kv4_attention_workspace(self._ref))
        self.dtype = dtype
        self._q = torch.Size((n_seq, n_query, n_head, head_dim))
        self._lse = self._q[:3]
        self._cache = torch.Size((n_page, n_head_kv, page_bytes(head_dim, page_size)))
        self._pages, self._n = torch.Size((n_seq, max_pages)), torch.Size((n_seq,))
        self._strides = None

    def _workspace(self, stream: int) -> torch.Tensor:
        """As a plan's, but with zeros where the kernel counts, which a call leaves so."""
        ws = self._ws.get(stream)
        if ws is None or _capturing():
            ws = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=f"cuda:{self.device}")
            ws[:4096].zero_()
            if not _capturing():
                self._ws[stream] = ws
        return ws

    def __call__(self, q, cache, pages, lengths, n_new=None, out=None, lse=None):
        a, dt, dev, i32 = self.a, self.dtype, self.device, torch.int32
        if q is None or q.dtype is not dt or q.shape != self._q or q.get_device() != dev or (st := q.stride())[3] != 1:
            _refuse(q, "q", self._q, dt, dev)
        if st != self._strides:
            a.q_seq_stride, a.q_token_stride, a.q_head_stride, _ = self._strides = st
        if (cache is None or cache.dtype is not torch.uint8 or cache.shape != self._cache or cache.get_device() != dev
                or not cache.is_contiguous()):
            _refuse(cache, "cache", self._cache, torch.uint8, dev)
        if (pages is None or pages.dtype is not i32 or pages.shape != self._pages or pages.get_device() != dev
                or ((st := pages.stride())[1] != 1 and a.max_pages > 1)):
            _refuse(pages, "pages", self._pages, i32, dev)
        a.pages_stride = st[0]
        a.lengths = _ints(lengths, "lengths", self._n, dev)
        a.n_new = None if n_new is None else _ints(n_new, "n_new", self._n, dev)
        if out is None:
            out = (torch.empty if n_new is None else torch.zeros)(self._q, dtype=dt, device=q.device)
        elif out.dtype is not dt or out.shape != self._q or out.get_device() != dev or not out.is_contiguous():
            _refuse(out, "out", self._q, dt, dev)
        if lse is None:
            lse = (torch.empty if n_new is None else torch.zeros)(self._lse, dtype=torch.float32, device=q.device)
        elif (lse.dtype is not torch.float32 or lse.shape != self._lse or lse.get_device() != dev
              or not lse.is_contiguous()):
            _refuse(lse, "lse", self._lse, torch.float32, dev)
        a.q, a.cache, a.pages, a.out, a.lse = q.data_ptr(), cache.data_ptr(), pages.data_ptr(), out.data_ptr(), lse.data_ptr()
        self._on_device()
        stream = _raw_stream(dev)
        ws = self._workspace(stream)
        if self.lib.fwb_kv4_attention_dev(self._ref, ws.data_ptr(), self.workspace_bytes, stream) != 0:
            raise FwbError(_err(self.lib))
        return out, lse


def check_status() -> None:
    """Waits for the current stream and raises FwbError if a call on this device met a
    page or position outside its tables since the last look (fwb_kv4_status)."""
    lib = native.product()
    if lib.fwb_kv4_status(_raw_stream(torch.cuda.current_device())) != 0:
        raise FwbError(_err(lib))
