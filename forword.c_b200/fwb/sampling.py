"""A token for each of many rows of logits by temperature, top-k, top-p and
min-p (fwb_sample_rows_dev of include/forword_b200.h) on torch CUDA tensors.
``Model.sample`` is the single-sequence form on a model's own logits.
"""
from __future__ import annotations

import torch

from . import native
from .beam import TYPE_IDS, _raw_stream, _refuse
from .model import FwbError, _err


def sample_rows(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, token=None, logprob=None):
    """-> (token int32 [n_row], logprob fp32 [n_row]).

    logits [n_row, n_vocab] fp32, fp16 or bf16 (rows may be strided); uniform
    [n_row] in [0, 1).  temperature, top_p and min_p fp32 [n_row], top_k int32
    [n_row], each None for no such setting (temperature 1).  The entries that
    stay are ranked by logit, equal ones by index; the token is the first at
    which their running mass exceeds uniform times all their mass, logprob the
    log of its share.  Temperature 0: the largest logit.  -1 and -inf where a
    row holds a NaN or +inf or nothing but -inf, or its uniform number or
    temperature is NaN.
    """
    if logits is None or logits.dim() != 2:
        raise ValueError("logits must be [n_row, n_vocab]")
    dt, dev, (n, vocab), (stride, last) = logits.dtype, logits.get_device(), logits.shape, logits.stride()
    if dt not in TYPE_IDS:
        raise ValueError(f"dtype must be one of {list(TYPE_IDS)}")
    if dev < 0 or torch.cuda.current_device() != dev:
        raise ValueError("sample_rows: logits and the current device differ")
    if last != 1 and vocab > 1:
        raise ValueError("logits: the last dimension must be contiguous")
    f32, i32 = torch.float32, torch.int32
    at = []
    for t, what, kind in ((uniform, "uniform", f32), (temperature, "temperature", f32), (top_k, "top_k", i32),
                          (top_p, "top_p", f32), (min_p, "min_p", f32)):
        if t is None and what != "uniform":
            at.append(None)
            continue
        if t is None or t.dtype is not kind or t.shape != (n,) or t.get_device() != dev or not t.is_contiguous():
            _refuse(t, what, (n,), kind, dev)
        at.append(t.data_ptr())
    if token is None:
        token = torch.empty(n, dtype=i32, device=logits.device)
    elif token.dtype is not i32 or token.shape != (n,) or token.get_device() != dev or not token.is_contiguous():
        _refuse(token, "token", (n,), i32, dev)
    if logprob is None:
        logprob = torch.empty(n, dtype=f32, device=logits.device)
    elif logprob.dtype is not f32 or logprob.shape != (n,) or logprob.get_device() != dev or not logprob.is_contiguous():
        _refuse(logprob, "logprob", (n,), f32, dev)
    lib = native.product()
    if lib.fwb_sample_rows_dev(logits.data_ptr(), TYPE_IDS[dt], n, vocab, stride, *at, token.data_ptr(), logprob.data_ptr(),
                               _raw_stream(dev)) != 0:
        raise FwbError(_err(lib))
    return token, logprob
