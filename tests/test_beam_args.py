"""CPU: the beam-search operators refuse bad arguments before any device work."""
import ctypes

import pytest

from fwb import native

PTR = 1 << 20   # an aligned address that is never read


@pytest.fixture(scope="module")
def lib(built):
    return native.product()


def attn_args(**kw):
    beam = pytest.importorskip("fwb.beam")
    a = beam.PrefixAttnArgs(type=1, n_group=1, n_beam=2, n_query=1, n_head=4, n_head_kv=2, head_dim=64, prefix_cap=10,
                            suffix_cap=4, q=PTR, prefix_k=PTR, prefix_v=PTR, suffix_k=PTR, suffix_v=PTR, out=PTR,
                            q_seq_stride=256, q_token_stride=256, q_head_stride=64, prefix_group_stride=1280,
                            prefix_head_stride=640, prefix_pos_stride=64, suffix_seq_stride=512, suffix_head_stride=256,
                            suffix_pos_stride=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    dict(type=2), dict(n_group=0), dict(n_beam=0), dict(n_query=0), dict(n_head=0), dict(n_head_kv=0), dict(n_head_kv=3),
    dict(head_dim=0), dict(head_dim=72), dict(head_dim=144), dict(prefix_cap=1 << 31), dict(n_group=1 << 24),
    dict(n_beam=40000), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(q=None), dict(out=None), dict(prefix_k=None), dict(suffix_v=None), dict(q=PTR + 2), dict(prefix_v=PTR + 8),
    dict(suffix_pos_stride=65), dict(q_head_stride=60), dict(lse=PTR + 1), dict(slots=PTR + 2),
], ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_attention_refuses(lib, bad):
    a = attn_args(**bad)
    assert lib.fwb_prefix_attention_dev(ctypes.byref(a), PTR, 1 << 40, None) == -1
    assert "fwb_prefix_attention" in lib.fwb_last_error().decode()


def test_attention_workspace(lib):
    a = attn_args()
    need = lib.fwb_prefix_attention_workspace(ctypes.byref(a))
    assert need > 0
    for ws, size in ((None, need), (PTR + 4, need), (PTR, need - 1)):
        assert lib.fwb_prefix_attention_dev(ctypes.byref(a), ws, size, None) == -1
        assert "workspace" in lib.fwb_last_error().decode()
    assert lib.fwb_prefix_attention_workspace(None) == 0
    a.head_dim = 8
    assert lib.fwb_prefix_attention_workspace(ctypes.byref(a)) == 0


SELECT = dict(logits=PTR, type=0, n_group=1, n_beam=4, n_vocab=100, row_stride=100, scores=PTR, n_select=8, out=PTR,
              parent=PTR, token=PTR, ws=PTR, ws_bytes=1 << 40)


@pytest.mark.parametrize("bad", [
    dict(type=8), dict(n_group=0), dict(n_beam=0), dict(n_vocab=0), dict(n_select=0), dict(n_beam=65), dict(n_select=129),
    dict(n_vocab=1, n_select=5), dict(n_vocab=1 << 30), dict(n_group=1 << 26), dict(row_stride=99), dict(logits=None),
    dict(scores=None), dict(out=None), dict(parent=None), dict(token=None), dict(logits=PTR + 2), dict(token=PTR + 1),
    dict(ws=None), dict(ws=PTR + 8), dict(ws_bytes=16),
], ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_select_refuses(lib, bad):
    assert lib.fwb_beam_select_dev(*{**SELECT, **bad}.values(), None) == -1
    assert "fwb_beam_select" in lib.fwb_last_error().decode()


REORDER = dict(src=PTR, dst=PTR, parent=PTR, n_outer=2, n_group=1, n_beam=4, n_inner=3, run=64, so=4096, ss=1024, si=128,
               do=4096, ds=1024, di=128)


@pytest.mark.parametrize("bad", [
    dict(src=None), dict(dst=None), dict(parent=None), dict(n_outer=0), dict(n_group=0), dict(n_beam=0), dict(n_inner=0),
    dict(run=0), dict(n_beam=65), dict(parent=PTR + 2), dict(dst=PTR + 64), dict(ds=2048), dict(n_outer=1 << 32),
], ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_reorder_refuses(lib, bad):
    assert lib.fwb_beam_reorder_dev(*{**REORDER, **bad}.values(), None) == -1
    assert "fwb_beam_reorder" in lib.fwb_last_error().decode()


def test_beam_search_refuses_without_a_model(lib):
    assert lib.fwb_beam_search(None, None, 1, 1, 1, -1, 0.0, None, None, None) == -1
    assert "fwb_beam_search" in lib.fwb_last_error().decode()
