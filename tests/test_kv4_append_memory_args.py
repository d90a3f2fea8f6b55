"""CPU: the append of the 4-bit cache refuses memory for rotated queries in which one row lies over another, before any
device work."""
import ctypes

import pytest

from fwb import native
from test_kv4_args import PTR, append_args, ids

# append_args: 3 sequences of 2 tokens, 4 heads of 64 fp16 values; rows of 128 bytes


@pytest.mark.parametrize("bad", [
    dict(q_out_head_stride=0), dict(q_out_token_stride=0), dict(q_out_seq_stride=0), dict(q_out_head_stride=56),
    dict(q_out_token_stride=248), dict(q_out_seq_stride=504), dict(q_out_token_stride=64), dict(q_out_head_stride=(1 << 60)),
    # in place, expanded
    dict(q_head_stride=0, q_out_head_stride=0), dict(q_seq_stride=0, q_out_seq_stride=0),
], ids=ids)
def test_rows_over_one_another(built, bad):
    lib = native.product()
    assert lib.fwb_kv4_append_dev(ctypes.byref(append_args(**bad)), None) == -1
    assert "overlap one another" in lib.fwb_last_error().decode()


@pytest.mark.parametrize("bad", [
    # a part of q's rows: 16 bytes on, a row on, a token on, before it
    dict(q_out=PTR + 16), dict(q_out=PTR + 128), dict(q_out=PTR + 512), dict(q_out=PTR - 128),
    # other strides than q's on the same memory
    dict(q_out_seq_stride=1024), dict(q_out_token_stride=64, q_out_head_stride=128, q_out_seq_stride=1024),
    # expanded queries under their own result
    dict(q_head_stride=0), dict(q_seq_stride=0, q_token_stride=0, q_head_stride=0, q_out=PTR - 256),
    # rows with gaps between them, half a row off
    dict(q_head_stride=128, q_token_stride=512, q_seq_stride=1024, q_out_head_stride=128, q_out_token_stride=512, q_out_seq_stride=1024,
         q_out=PTR + 64),
], ids=ids)
def test_results_over_other_queries(built, bad):
    lib = native.product()
    assert lib.fwb_kv4_append_dev(ctypes.byref(append_args(**bad)), None) == -1
    assert "q_out must be q itself or memory apart from it" in lib.fwb_last_error().decode()
