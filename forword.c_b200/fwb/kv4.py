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


def _cache(cache, heads: int, head_dim: int, dev: int):
    """(page size, pages) of a cache."""
    if cache is None:
        raise ValueError("cache is missing")
    shape = cache.shape
    if (cache.dtype is not torch.uint8 or len(shape) != 3 or shape[1] != heads or cache.get_device() != dev
            or not cache.is_contiguous()):
        raise ValueError(f"cache: expected contiguous torch.uint8 [n_page, {heads}, page bytes] on cuda:{dev}, "
                         f"got {cache.dtype} {tuple(shape)} on {cache.device}")
    return _page_size(head_dim, shape[2]), shape[0]


def _table(pages, n: int, dev: int):
    """(max_pages, row stride) of a page table."""
    if pages is None:
        raise ValueError("pages is missing")
    shape = pages.shape
    if pages.dtype is not torch.int32 or len(shape) != 2 or shape[0] != n or pages.get_device() != dev:
        raise ValueError(f"pages: expected torch.int32 [{n}, max_pages] on cuda:{dev}, "
                         f"got {pages.dtype} {tuple(shape)} on {pages.device}")
    st = pages.stride()
    if st[1] != 1 and shape[1] > 1:
        raise ValueError("pages: the last dimension must be contiguous")
    return shape[1], st[0]


def _ints(t, what: str, shape, dev: int) -> int:
    if t is None or t.dtype is not torch.int32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        _refuse(t, what, shape, torch.int32, dev)
    return t.data_ptr()


def _rows(t, what: str, shape, dtype, dev: int):
    """(address, strides) of rows [n_seq, n_query, heads, head_dim]."""
    if t is None or t.dtype is not dtype or t.shape != shape or t.get_device() != dev or (st := t.stride())[3] != 1:
        _refuse(t, what, shape, dtype, dev)
    return t.data_ptr(), st


def _overlap(a, b) -> bool:
    """Whether the bytes from first to last of two tensors meet."""
    def span(t):
        p = t.data_ptr()
        return p, p + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def append(q, k, v, cache, pages, lengths, cos=None, sin=None, halves: bool = False, n_new=None, q_out=None):
    """New tokens into the cache (fwb_kv4_append_dev) -> q_out, the rotated queries.

    q [n_seq, n_query, n_head, head_dim] or None, k and v [n_seq, n_query,
    n_head_kv, head_dim]: views with a contiguous last dimension, addresses
    and strides multiples of 16 bytes.  cos and sin fp32 [n_pos, head_dim/2],
    None: no rotation; halves: pairs (i, i + head_dim/2) are turned instead of
    neighbours.  q_out may be q itself; rows of tokens that a padded batch
    lacks are left as they were (zeros where q_out is None).
    """
    if k is None or k.dim() != 4:
        raise ValueError("k must be [n_seq, n_query, n_head_kv, head_dim]")
    dt, dev, shape = k.dtype, k.get_device(), k.shape
    if dt not in TYPE_IDS:
        raise ValueError(f"dtype must be one of {list(TYPE_IDS)}")
    if dev < 0 or torch.cuda.current_device() != dev:
        raise ValueError("append: k and the current device differ")
    n_seq, n_query, heads, hd = shape
    a = AppendArgs()
    a.type, a.n_seq, a.n_query, a.n_head_kv, a.head_dim = TYPE_IDS[dt], n_seq, n_query, heads, hd
    a.k, st = _rows(k, "k", shape, dt, dev)
    a.k_seq_stride, a.k_token_stride, a.k_head_stride, _ = st
    a.v, st = _rows(v, "v", shape, dt, dev)
    a.v_seq_stride, a.v_token_stride, a.v_head_stride, _ = st
    a.page_size, a.n_page = _cache(cache, heads, hd, dev)
    a.cache = cache.data_ptr()
    a.max_pages, a.pages_stride = _table(pages, n_seq, dev)
    a.pages = pages.data_ptr()
    a.lengths = _ints(lengths, "lengths", (n_seq,), dev)
    if n_new is not None:
        a.n_new = _ints(n_new, "n_new", (n_seq,), dev)
    if q is not None:
        if q.dim() != 4:
            raise ValueError("q must be [n_seq, n_query, n_head, head_dim]")
        qs = torch.Size((n_seq, n_query, q.shape[2], hd))
        a.n_head = qs[2]
        a.q, st = _rows(q, "q", qs, dt, dev)
        a.q_seq_stride, a.q_token_stride, a.q_head_stride, _ = st
        if q_out is None:
            q_out = torch.empty(qs, dtype=dt, device=k.device) if n_new is None else torch.zeros(qs, dtype=dt, device=k.device)
        a.q_out, so = _rows(q_out, "q_out", qs, dt, dev)
        a.q_out_seq_stride, a.q_out_token_stride, a.q_out_head_stride, _ = so
        if (a.q != a.q_out or st != so) and q.numel() and _overlap(q, q_out):
            raise ValueError("q_out must be q itself or memory apart from it")
    elif q_out is not None:
        raise ValueError("q_out without q")
    if cos is not None or sin is not None:
        for t, what in ((cos, "cos"), (sin, "sin")):
            if (t is None or t.dtype is not torch.float32 or t.dim() != 2 or t.shape != (cos if cos is not None else t).shape
                    or t.shape[1] * 2 != hd or t.get_device() != dev or not t.is_contiguous()):
                raise ValueError(f"{what}: expected contiguous torch.float32 [n_pos, {hd // 2}] on cuda:{dev}, cos and sin alike")
        a.cos, a.sin, a.n_pos = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    a.halves = 1 if halves else 0
    lib = native.product()
    if lib.fwb_kv4_append_dev(ctypes.byref(a), _raw_stream(dev)) != 0:
        raise FwbError(_err(lib))
    return q_out


def read(cache, pages, start, n: int, *, head_dim: int, dtype: torch.dtype, lengths=None, k=None, v=None):
    """Positions start[s] .. start[s] + n - 1 of every sequence (fwb_kv4_read_dev)
    -> (k, v), each [n_seq, n, n_head_kv, head_dim]; zeros at and past lengths."""
    if dtype not in TYPE_IDS:
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
    a = ReadArgs()
    a.type, a.n_seq, a.n, a.n_head_kv, a.head_dim = TYPE_IDS[dtype], n_seq, n, heads, head_dim
    a.page_size, a.n_page = _cache(cache, heads, head_dim, dev)
    a.cache = cache.data_ptr()
    a.max_pages, a.pages_stride = _table(pages, n_seq, dev)
    a.pages = pages.data_ptr()
    a.start = _ints(start, "start", (n_seq,), dev)
    if lengths is not None:
        a.lengths = _ints(lengths, "lengths", (n_seq,), dev)
    shape = torch.Size((n_seq, n, heads, head_dim))
    if k is None:
        k = torch.empty(shape, dtype=dtype, device=cache.device)
    elif k.dtype is not dtype or k.shape != shape or k.get_device() != dev or not k.is_contiguous():
        _refuse(k, "k", shape, dtype, dev)
    if v is None:
        v = torch.empty(shape, dtype=dtype, device=cache.device)
    elif v.dtype is not dtype or v.shape != shape or v.get_device() != dev or not v.is_contiguous():
        _refuse(v, "v", shape, dtype, dev)
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
    out    like q, contiguous; lse fp32 [n_seq, n_query, n_head].  Rows of
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
        """As a plan's, but zeros at first, as the kernel wants it; a call leaves it so."""
        if _capturing():
            return torch.zeros(self.workspace_bytes, dtype=torch.uint8, device=f"cuda:{self.device}")
        ws = self._ws.get(stream)
        if ws is None:
            ws = self._ws[stream] = torch.zeros(self.workspace_bytes, dtype=torch.uint8, device=f"cuda:{self.device}")
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
