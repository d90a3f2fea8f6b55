"""Beam search and parallel continuations: the operators of
include/forword_b200.h on torch CUDA tensors.

``PrefixAttention``  attention of sequences that share a prefix
``BeamSelect``       the best of beams x vocabulary
``reorder``          per-beam state moved by the selected parents

Thin plumbing over the CUDA library (no CPU fallback): a plan checks sizes
once and keeps its workspace; a call checks its tensors and enqueues on the
current stream of torch.  Plans and calls work on the current device.  One
plan is used from one thread at a time; each stream that it is used on gets a
workspace of its own.
"""
from __future__ import annotations

import ctypes

import torch

from . import native
from .model import FwbError, _err

TYPE_IDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}  # GGML type ids

_u32, _u64, _vp = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_void_p


class PrefixAttnArgs(ctypes.Structure):
    """fwb_prefix_attn_t."""
    _fields_ = ([(n, _u32) for n in ("type", "n_group", "n_beam", "n_query", "n_head", "n_head_kv", "head_dim",
                                     "prefix_cap", "suffix_cap")]
                + [("scale", ctypes.c_float), ("q", _vp)]
                + [(n, _u64) for n in ("q_seq_stride", "q_token_stride", "q_head_stride")]
                + [("prefix_k", _vp), ("prefix_v", _vp)]
                + [(n, _u64) for n in ("prefix_group_stride", "prefix_head_stride", "prefix_pos_stride")]
                + [("suffix_k", _vp), ("suffix_v", _vp)]
                + [(n, _u64) for n in ("suffix_seq_stride", "suffix_head_stride", "suffix_pos_stride")]
                + [("prefix_len", _vp), ("suffix_len", _vp), ("slots", _vp), ("slots_stride", _u64),
                   ("out", _vp), ("lse", _vp)])


def _check(t, what: str, shape, dtype, device: int, last: bool = True) -> None:
    if t.dtype is not dtype or t.shape != shape or not t.is_cuda or t.get_device() != device:
        raise ValueError(f"{what}: expected {dtype} {tuple(shape)} on cuda:{device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    if last and t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")


class _Plan:
    def __init__(self, device: int | None, bytes_of):
        self.lib = native.product()
        self.device = torch.cuda.current_device() if device is None else int(device)
        self.workspace_bytes = int(bytes_of())
        if not self.workspace_bytes:
            raise FwbError(_err(self.lib))
        self._ws: dict[int, torch.Tensor] = {}

    def _stream(self) -> tuple[int, int]:
        """The current stream and the address of this plan's workspace for it."""
        if torch.cuda.current_device() != self.device:
            raise ValueError(f"the plan is for cuda:{self.device}, the current device is "
                             f"cuda:{torch.cuda.current_device()}")
        st = torch.cuda.current_stream().cuda_stream
        ws = self._ws.get(st)
        if ws is None:
            ws = self._ws[st] = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=f"cuda:{self.device}")
        return st, ws.data_ptr()


class PrefixAttention(_Plan):
    """Plan of fwb_prefix_attention_dev for fixed sizes.

    plan(q, prefix_k, prefix_v, suffix_k, suffix_v, prefix_len=None,
    suffix_len=None, slots=None, out=None, lse=None) -> (out, lse):

    q          [n_group*n_beam, n_query, n_head, head_dim]
    prefix_k/v [n_group, n_head_kv, prefix_cap, head_dim] (None when prefix_cap is 0)
    suffix_k/v [n_group*n_beam, n_head_kv, suffix_cap, head_dim] (None when suffix_cap is 0)
    prefix_len [n_group], suffix_len [n_group*n_beam], slots [n_group*n_beam, suffix_cap]: int32 or None
    out        like q, contiguous; lse fp32 [n_group*n_beam, n_query, n_head]

    q, K and V may be views (last dimension contiguous, strides multiples of
    16 bytes); a K and its V have equal strides.
    """

    def __init__(self, *, n_group: int, n_beam: int, n_head: int, n_head_kv: int, head_dim: int, dtype: torch.dtype,
                 prefix_cap: int, suffix_cap: int, n_query: int = 1, scale: float = 0.0, device: int | None = None):
        if dtype not in TYPE_IDS:
            raise ValueError(f"dtype must be one of {list(TYPE_IDS)}")
        for v in (n_group, n_beam, n_head, n_head_kv, head_dim, prefix_cap, suffix_cap, n_query):
            if not 0 <= v < 1 << 32:
                raise ValueError(f"size {v} out of range")
        a = self.a = PrefixAttnArgs(type=TYPE_IDS[dtype], n_group=n_group, n_beam=n_beam, n_query=n_query,
                                    n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, prefix_cap=prefix_cap,
                                    suffix_cap=suffix_cap, scale=scale)
        self._ref = ctypes.byref(a)
        super().__init__(device, lambda: native.product().fwb_prefix_attention_workspace(self._ref))
        n = n_group * n_beam
        self.dtype = dtype
        self._q = torch.Size((n, n_query, n_head, head_dim))
        self._p = torch.Size((n_group, n_head_kv, prefix_cap, head_dim))
        self._s = torch.Size((n, n_head_kv, suffix_cap, head_dim))
        self._plen, self._slen = torch.Size((n_group,)), torch.Size((n,))
        self._slots = torch.Size((n, suffix_cap))

    def __call__(self, q, prefix_k, prefix_v, suffix_k, suffix_v, prefix_len=None, suffix_len=None, slots=None,
                 out=None, lse=None):
        a, dt, dev = self.a, self.dtype, self.device
        _check(q, "q", self._q, dt, dev)
        a.q = q.data_ptr()
        a.q_seq_stride, a.q_token_stride, a.q_head_stride, _ = q.stride()
        if a.prefix_cap:
            _check(prefix_k, "prefix_k", self._p, dt, dev)
            _check(prefix_v, "prefix_v", self._p, dt, dev)
            st = prefix_k.stride()
            if prefix_v.stride() != st:
                raise ValueError("prefix_k and prefix_v must have equal strides")
            a.prefix_k, a.prefix_v = prefix_k.data_ptr(), prefix_v.data_ptr()
            a.prefix_group_stride, a.prefix_head_stride, a.prefix_pos_stride, _ = st
        if a.suffix_cap:
            _check(suffix_k, "suffix_k", self._s, dt, dev)
            _check(suffix_v, "suffix_v", self._s, dt, dev)
            st = suffix_k.stride()
            if suffix_v.stride() != st:
                raise ValueError("suffix_k and suffix_v must have equal strides")
            a.suffix_k, a.suffix_v = suffix_k.data_ptr(), suffix_v.data_ptr()
            a.suffix_seq_stride, a.suffix_head_stride, a.suffix_pos_stride, _ = st
        a.prefix_len = a.suffix_len = a.slots = None
        if prefix_len is not None:
            _check(prefix_len, "prefix_len", self._plen, torch.int32, dev)
            a.prefix_len = prefix_len.data_ptr()
        if suffix_len is not None:
            _check(suffix_len, "suffix_len", self._slen, torch.int32, dev)
            a.suffix_len = suffix_len.data_ptr()
        if slots is not None and a.suffix_cap:
            _check(slots, "slots", self._slots, torch.int32, dev)
            a.slots, a.slots_stride = slots.data_ptr(), slots.stride(0)
        if out is None:
            out = torch.empty(self._q, dtype=dt, device=q.device)
        else:
            _check(out, "out", self._q, dt, dev)
            if not out.is_contiguous():
                raise ValueError("out must be contiguous")
        if lse is None:
            lse = torch.empty(self._q[:3], dtype=torch.float32, device=q.device)
        else:
            _check(lse, "lse", self._q[:3], torch.float32, dev)
            if not lse.is_contiguous():
                raise ValueError("lse must be contiguous")
        a.out, a.lse = out.data_ptr(), lse.data_ptr()
        stream, ws = self._stream()
        if self.lib.fwb_prefix_attention_dev(self._ref, ws, self.workspace_bytes, stream) != 0:
            raise FwbError(_err(self.lib))
        return out, lse


class BeamSelect(_Plan):
    """Plan of fwb_beam_select_dev for fixed sizes.

    plan(logits, scores, out_scores=None, parent=None, token=None) ->
    (out_scores, parent, token), each [n_group, n_select]; logits [n_group,
    n_beam, n_vocab] (rows may be strided), scores fp32 [n_group, n_beam].
    """

    def __init__(self, *, n_group: int, n_beam: int, n_vocab: int, n_select: int, dtype: torch.dtype = torch.float32,
                 device: int | None = None):
        if dtype not in TYPE_IDS:
            raise ValueError(f"dtype must be one of {list(TYPE_IDS)}")
        if min(n_group, n_beam, n_vocab, n_select) < 0:
            raise ValueError("negative size")
        self._sizes = (TYPE_IDS[dtype], n_group, n_beam, n_vocab)
        super().__init__(device, lambda: native.product().fwb_beam_select_workspace(*self._sizes, n_select))
        self.dtype, self.n_select = dtype, n_select
        self._x, self._c = torch.Size((n_group, n_beam, n_vocab)), torch.Size((n_group, n_beam))
        self._o = torch.Size((n_group, n_select))

    def __call__(self, logits, scores, out_scores=None, parent=None, token=None):
        dev = self.device
        _check(logits, "logits", self._x, self.dtype, dev)
        _check(scores, "scores", self._c, torch.float32, dev)
        sg, sw, _ = logits.stride()
        if self._x[1] == 1:
            sw = sg if self._x[0] > 1 else self._x[2]
        elif self._x[0] > 1 and sg != self._x[1] * sw:
            raise ValueError("logits: all rows must be equally far apart")
        if not scores.is_contiguous():
            raise ValueError("scores must be contiguous")
        if out_scores is None:
            out_scores = torch.empty(self._o, dtype=torch.float32, device=logits.device)
        if parent is None:
            parent = torch.empty(self._o, dtype=torch.int32, device=logits.device)
        if token is None:
            token = torch.empty(self._o, dtype=torch.int32, device=logits.device)
        for t, what, dt in ((out_scores, "out_scores", torch.float32), (parent, "parent", torch.int32),
                            (token, "token", torch.int32)):
            _check(t, what, self._o, dt, dev)
            if not t.is_contiguous():
                raise ValueError(f"{what} must be contiguous")
        stream, ws = self._stream()
        if self.lib.fwb_beam_select_dev(logits.data_ptr(), *self._sizes, sw, scores.data_ptr(), self.n_select,
                                        out_scores.data_ptr(), parent.data_ptr(), token.data_ptr(), ws,
                                        self.workspace_bytes, stream) != 0:
            raise FwbError(_err(self.lib))
        return out_scores, parent, token


def _runs(shape, strides, size: int):
    """State [n_outer, slots, ...] of one or two tensors (their strides) as
    (n_inner, run bytes, inner stride of each in bytes): the trailing
    dimensions as one level of equally spaced runs."""
    run, d = 1, len(shape) - 1
    while d >= 2 and (shape[d] == 1 or all(st[d] == run for st in strides)):  # contiguous in each
        run *= shape[d]
        d -= 1
    if d < 2:
        return 1, run * size, [0] * len(strides)
    n, inner = shape[d], [st[d] for st in strides]
    for k in range(d - 1, 1, -1):                                             # dimensions that nest into that spacing
        if shape[k] == 1:
            continue
        if any(st[k] != i * n for st, i in zip(strides, inner)):
            raise ValueError("reorder: the dimensions after the slots must be contiguous runs at one spacing")
        n *= shape[k]
    return n, run * size, [i * size for i in inner]


def reorder(src, parent, dst=None):
    """dst[:, g*n_beam + b] = src[:, g*n_beam + parent[g, b]] (fwb_beam_reorder_dev).

    src [n_outer, n_group*n_beam, ...] of any type; views are moved as views
    (the dimensions after the slots must form equally spaced contiguous
    runs).  parent int32 [n_group, n_beam].  dst None: in place."""
    if dst is None:
        dst = src
    if not src.is_cuda or src.dim() < 2 or dst.shape != src.shape or dst.dtype is not src.dtype:
        raise ValueError("reorder: src and dst must be CUDA tensors of the same shape and type, [n_outer, slots, ...]")
    dev = src.get_device()
    if dst.get_device() != dev or torch.cuda.current_device() != dev:
        raise ValueError("reorder: src, dst and the current device differ")
    if parent.dim() != 2 or parent.numel() != src.shape[1]:
        raise ValueError("reorder: parent must be [n_group, n_beam] with n_group * n_beam slots")
    _check(parent, "parent", parent.shape, torch.int32, dev)
    if not parent.is_contiguous():
        raise ValueError("parent must be contiguous")
    if src.numel() == 0:
        return dst
    size = src.element_size()
    st, dt = src.stride(), dst.stride()
    n_in, run, inner = _runs(src.shape, (st, dt), size)
    lib = native.product()
    if lib.fwb_beam_reorder_dev(src.data_ptr(), dst.data_ptr(), parent.data_ptr(), src.shape[0], *parent.shape, n_in,
                                run, st[0] * size, st[1] * size, inner[0], dt[0] * size, dt[1] * size, inner[1],
                                torch.cuda.current_stream().cuda_stream) != 0:
        raise FwbError(_err(lib))
    return dst
