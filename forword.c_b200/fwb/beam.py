"""Beam search and parallel continuations: the operators of
include/forword_b200.h on torch CUDA tensors.

``PrefixAttention``  attention of sequences that share a prefix
``BeamSelect``       the best of beams x vocabulary
``reorder``          per-beam state moved by the selected parents
``check_status``     whether every attention kernel so far completed

(``Model.beam_search`` runs them on a model.)

Thin plumbing over the CUDA library (no CPU fallback): a plan checks sizes
once and keeps its workspace; a call checks its tensors and enqueues on the
current stream of torch.  Plans and calls work on the current device.  One
plan is used from one thread at a time; each stream that it is used on gets a
workspace of its own, and so does each call captured into a CUDA graph, from
the graph's memory pool.
"""
from __future__ import annotations

import ctypes
import functools

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


# the current stream of torch as a cudaStream_t (the public call builds an object, 3 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)
_capturing = torch.cuda.is_current_stream_capturing


def _refuse(t, what: str, shape, dtype, device: int):
    if t is None:
        raise ValueError(f"{what} is missing")
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device:
        raise ValueError(f"{what}: expected {dtype} {tuple(shape)} on cuda:{device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    raise ValueError(f"{what}: the last dimension must be contiguous" if t.dim() > 1 and t.stride(-1) != 1
                     else f"{what} must be contiguous")


def _apart(shape, one, other) -> bool:
    """Whether the strides of two tensors of this shape differ where they matter."""
    return any(n > 1 and x != y for n, x, y in zip(shape, one, other))


class _Plan:
    def __init__(self, device: int | None, bytes_of):
        self.lib = native.product()
        self.device = torch.cuda.current_device() if device is None else int(device)
        if not 0 <= self.device < torch.cuda.device_count():
            raise ValueError(f"no device cuda:{self.device}")
        with torch.cuda.device(self.device):
            self.workspace_bytes = int(bytes_of())
        if not self.workspace_bytes:
            raise FwbError(_err(self.lib))
        self._ws: dict[int, torch.Tensor] = {}

    def _workspace(self, stream: int) -> torch.Tensor:
        """This plan's workspace for a stream.  A captured call's belongs to its graph, which may be replayed on any
        stream beside other graphs and calls of this plan: it is not kept here, the graph's memory pool holds it."""
        if _capturing():
            return torch.empty(self.workspace_bytes, dtype=torch.uint8, device=f"cuda:{self.device}")
        ws = self._ws.get(stream)
        if ws is None:
            ws = self._ws[stream] = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=f"cuda:{self.device}")
        return ws

    def _on_device(self) -> None:
        if torch.cuda.current_device() != self.device:
            raise ValueError(f"the plan is for cuda:{self.device}, the current device is "
                             f"cuda:{torch.cuda.current_device()}")


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
        self._lse = self._q[:3]
        self._strides = [None, None, None]     # of q, prefix and suffix, as the arguments hold them

    def __call__(self, q, prefix_k, prefix_v, suffix_k, suffix_v, prefix_len=None, suffix_len=None, slots=None,
                 out=None, lse=None):
        a, dt, dev, seen = self.a, self.dtype, self.device, self._strides
        if q is None or q.dtype is not dt or q.shape != self._q or q.get_device() != dev or (st := q.stride())[3] != 1:
            _refuse(q, "q", self._q, dt, dev)
        if st != seen[0]:
            a.q_seq_stride, a.q_token_stride, a.q_head_stride, _ = seen[0] = st
        a.q = q.data_ptr()
        if a.prefix_cap:
            k, v, shape = prefix_k, prefix_v, self._p
            if k is None or k.dtype is not dt or k.shape != shape or k.get_device() != dev or (st := k.stride())[3] != 1:
                _refuse(k, "prefix_k", shape, dt, dev)
            if v is None or v.dtype is not dt or v.shape != shape or v.get_device() != dev:
                _refuse(v, "prefix_v", shape, dt, dev)
            if v.stride() != st and _apart(shape, v.stride(), st):
                raise ValueError("prefix_k and prefix_v must have equal strides")
            if st != seen[1]:
                a.prefix_group_stride, a.prefix_head_stride, a.prefix_pos_stride, _ = seen[1] = st
            a.prefix_k, a.prefix_v = k.data_ptr(), v.data_ptr()
        if a.suffix_cap:
            k, v, shape = suffix_k, suffix_v, self._s
            if k is None or k.dtype is not dt or k.shape != shape or k.get_device() != dev or (st := k.stride())[3] != 1:
                _refuse(k, "suffix_k", shape, dt, dev)
            if v is None or v.dtype is not dt or v.shape != shape or v.get_device() != dev:
                _refuse(v, "suffix_v", shape, dt, dev)
            if v.stride() != st and _apart(shape, v.stride(), st):
                raise ValueError("suffix_k and suffix_v must have equal strides")
            if st != seen[2]:
                a.suffix_seq_stride, a.suffix_head_stride, a.suffix_pos_stride, _ = seen[2] = st
            a.suffix_k, a.suffix_v = k.data_ptr(), v.data_ptr()
        i32 = torch.int32
        if prefix_len is None:
            a.prefix_len = None
        else:
            t = prefix_len
            if t.dtype is not i32 or t.shape != self._plen or t.get_device() != dev or not t.is_contiguous():
                _refuse(t, "prefix_len", self._plen, i32, dev)
            a.prefix_len = t.data_ptr()
        if suffix_len is None:
            a.suffix_len = None
        else:
            t = suffix_len
            if t.dtype is not i32 or t.shape != self._slen or t.get_device() != dev or not t.is_contiguous():
                _refuse(t, "suffix_len", self._slen, i32, dev)
            a.suffix_len = t.data_ptr()
        if slots is None or not a.suffix_cap:
            a.slots = None
        else:
            t = slots
            st = t.stride()
            if (t.dtype is not i32 or t.shape != self._slots or t.get_device() != dev
                    or (st[1] != 1 and a.suffix_cap > 1)):
                _refuse(t, "slots", self._slots, i32, dev)
            a.slots, a.slots_stride = t.data_ptr(), st[0]
        if out is None:
            out = torch.empty(self._q, dtype=dt, device=q.device)
        elif out.dtype is not dt or out.shape != self._q or out.get_device() != dev or not out.is_contiguous():
            _refuse(out, "out", self._q, dt, dev)
        if lse is None:
            lse = torch.empty(self._lse, dtype=torch.float32, device=q.device)
        elif (lse.dtype is not torch.float32 or lse.shape != self._lse or lse.get_device() != dev
              or not lse.is_contiguous()):
            _refuse(lse, "lse", self._lse, torch.float32, dev)
        a.out, a.lse = out.data_ptr(), lse.data_ptr()
        self._on_device()
        stream = _raw_stream(dev)
        ws = self._workspace(stream)
        if self.lib.fwb_prefix_attention_dev(self._ref, ws.data_ptr(), self.workspace_bytes, stream) != 0:
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
        dev, o, f32, i32 = self.device, self._o, torch.float32, torch.int32
        n_group, n_beam, n_vocab = self._x
        if (logits is None or logits.dtype is not self.dtype or logits.shape != self._x or logits.get_device() != dev
                or (logits.stride(2) != 1 and n_vocab > 1)):
            _refuse(logits, "logits", self._x, self.dtype, dev)
        sg, sw, _ = logits.stride()
        if n_beam == 1:
            sw = sg if n_group > 1 else n_vocab
        elif n_group > 1 and sg != n_beam * sw:
            raise ValueError("logits: all rows must be equally far apart")
        if (scores is None or scores.dtype is not f32 or scores.shape != self._c or scores.get_device() != dev
                or not scores.is_contiguous()):
            _refuse(scores, "scores", self._c, f32, dev)
        if out_scores is None:
            out_scores = torch.empty(o, dtype=f32, device=logits.device)
        elif (out_scores.dtype is not f32 or out_scores.shape != o or out_scores.get_device() != dev
              or not out_scores.is_contiguous()):
            _refuse(out_scores, "out_scores", o, f32, dev)
        if parent is None:
            parent = torch.empty(o, dtype=i32, device=logits.device)
        elif parent.dtype is not i32 or parent.shape != o or parent.get_device() != dev or not parent.is_contiguous():
            _refuse(parent, "parent", o, i32, dev)
        if token is None:
            token = torch.empty(o, dtype=i32, device=logits.device)
        elif token.dtype is not i32 or token.shape != o or token.get_device() != dev or not token.is_contiguous():
            _refuse(token, "token", o, i32, dev)
        self._on_device()
        stream = _raw_stream(dev)
        ws = self._workspace(stream)
        if self.lib.fwb_beam_select_dev(logits.data_ptr(), *self._sizes, sw, scores.data_ptr(), self.n_select,
                                        out_scores.data_ptr(), parent.data_ptr(), token.data_ptr(),
                                        ws.data_ptr(), self.workspace_bytes, stream) != 0:
            raise FwbError(_err(self.lib))
        return out_scores, parent, token


@functools.lru_cache(maxsize=256)
def _runs(shape, st, dt, size: int):
    """State [n_outer, slots, ...] with the strides st and dt of its source and
    destination as (n_inner, run bytes, inner stride of each in bytes): the
    trailing dimensions as one level of equally spaced runs."""
    run, d = 1, len(shape) - 1
    while d >= 2 and (shape[d] == 1 or st[d] == dt[d] == run):  # contiguous in both
        run *= shape[d]
        d -= 1
    if d < 2:
        return 1, run * size, 0, 0
    n = shape[d]
    for k in range(d - 1, 1, -1):                               # dimensions that nest into that spacing
        if shape[k] == 1:
            continue
        if st[k] != st[d] * n or dt[k] != dt[d] * n:
            raise ValueError("reorder: the dimensions after the slots must be contiguous runs at one spacing")
        n *= shape[k]
    return n, run * size, st[d] * size, dt[d] * size


def reorder(src, parent, dst=None):
    """dst[:, g*n_beam + b] = src[:, g*n_beam + parent[g, b]] (fwb_beam_reorder_dev).

    src [n_outer, n_group*n_beam, ...] of any type; views are moved as views
    (the dimensions after the slots must form equally spaced contiguous
    runs).  parent int32 [n_group, n_beam].  dst None: in place."""
    if src is None or parent is None:
        raise ValueError("reorder: src or parent is missing")
    if dst is None:
        dst = src
    shape, st, dt, dev = src.shape, src.stride(), dst.stride(), src.get_device()
    if len(shape) < 2 or dev < 0 or dst.shape != shape or dst.dtype is not src.dtype:
        raise ValueError("reorder: src and dst must be CUDA tensors of the same shape and type, [n_outer, slots, ...]")
    if dst.get_device() != dev or torch.cuda.current_device() != dev:
        raise ValueError("reorder: src, dst and the current device differ")
    ps = parent.shape
    if len(ps) != 2 or ps[0] * ps[1] != shape[1]:
        raise ValueError("reorder: parent must be [n_group, n_beam] with n_group * n_beam slots")
    if parent.dtype is not torch.int32 or parent.get_device() != dev or not parent.is_contiguous():
        _refuse(parent, "parent", ps, torch.int32, dev)
    if src.numel() == 0:
        return dst
    size = src.element_size()
    n_in, run, si, di = _runs(shape, st, dt, size)
    lib = native.product()
    if lib.fwb_beam_reorder_dev(src.data_ptr(), dst.data_ptr(), parent.data_ptr(), shape[0], ps[0], ps[1], n_in, run,
                                st[0] * size, st[1] * size, si, dt[0] * size, dt[1] * size, di, _raw_stream(dev)) != 0:
        raise FwbError(_err(lib))
    return dst


def check_status() -> None:
    """Waits for the current stream and raises FwbError if a bounded wait of an
    attention kernel on this device ran out since the last look (fwb_beam_status)."""
    lib = native.product()
    if lib.fwb_beam_status(_raw_stream(torch.cuda.current_device())) != 0:
        raise FwbError(_err(lib))
