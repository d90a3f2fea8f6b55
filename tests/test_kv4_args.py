"""CPU: the operators of the 4-bit cache and the sampling of rows refuse bad
arguments before any device work."""
import ctypes

import pytest

from fwb import native

PTR = 1 << 20   # an aligned address that is never read


@pytest.fixture(scope="module")
def lib(built):
    return native.product()


def ids(d):
    return ",".join(f"{k}={v}" for k, v in d.items())


SIZES = dict(type=1, n_seq=3, n_head_kv=2, head_dim=64, page_size=32, n_page=10, max_pages=4)
BAD_SIZES = [dict(type=2), dict(n_seq=0), dict(n_head_kv=0), dict(head_dim=0), dict(head_dim=40), dict(head_dim=144),
             dict(page_size=0), dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(n_page=0), dict(n_page=1 << 31),
             dict(max_pages=0), dict(max_pages=1 << 26), dict(n_seq=1 << 24), dict(n_head_kv=65536), dict(cache=None),
             dict(cache=PTR + 8), dict(pages=None), dict(pages=PTR + 2)]


def append_args(**kw):
    kv4 = pytest.importorskip("fwb.kv4")
    a = kv4.AppendArgs(**SIZES, n_query=2, n_head=4, n_pos=100, q=PTR, q_seq_stride=512, q_token_stride=256, q_head_stride=64,
                       k=PTR, v=PTR, k_seq_stride=256, k_token_stride=128, k_head_stride=64, v_seq_stride=256,
                       v_token_stride=128, v_head_stride=64, q_out=PTR, q_out_seq_stride=512, q_out_token_stride=256,
                       q_out_head_stride=64, cache=PTR, pages=PTR, pages_stride=4, lengths=PTR, n_new=PTR, cos=PTR, sin=PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", BAD_SIZES + [
    dict(n_query=0), dict(n_query=1 << 24), dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(n_head=0), dict(n_head=65536),
    dict(cos=None), dict(sin=None), dict(n_pos=0), dict(cos=PTR + 4), dict(lengths=None), dict(lengths=PTR + 1),
    dict(n_new=PTR + 2), dict(q=PTR + 2), dict(k=PTR + 8), dict(v_token_stride=65), dict(q_out_head_stride=66),
], ids=ids)
def test_append_refuses(lib, bad):
    a = append_args(**bad)
    assert lib.fwb_kv4_append_dev(ctypes.byref(a), None) == -1
    assert "fwb_kv4_append" in lib.fwb_last_error().decode()


def read_args(**kw):
    kv4 = pytest.importorskip("fwb.kv4")
    a = kv4.ReadArgs(**SIZES, n=7, cache=PTR, pages=PTR, pages_stride=4, start=PTR, lengths=PTR, k=PTR, v=PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", BAD_SIZES + [dict(n=0), dict(n=1 << 24), dict(start=None), dict(start=PTR + 1), dict(k=None),
                                             dict(v=None), dict(k=PTR + 4), dict(lengths=PTR + 2)], ids=ids)
def test_read_refuses(lib, bad):
    a = read_args(**bad)
    assert lib.fwb_kv4_read_dev(ctypes.byref(a), None) == -1
    assert "fwb_kv4_read" in lib.fwb_last_error().decode()


def attn_args(**kw):
    kv4 = pytest.importorskip("fwb.kv4")
    a = kv4.AttnArgs(**SIZES, n_query=2, n_head=4, q=PTR, q_seq_stride=512, q_token_stride=256, q_head_stride=64, cache=PTR,
                     pages=PTR, pages_stride=4, lengths=PTR, n_new=PTR, out=PTR, lse=PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", BAD_SIZES + [
    dict(n_query=0), dict(n_head=0), dict(n_head=3), dict(n_head=65536), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(q=None), dict(out=None), dict(lengths=None), dict(n_new=PTR + 1), dict(q=PTR + 4),
    dict(q_token_stride=100), dict(out=PTR + 8), dict(lse=PTR + 1), dict(n_seq=4100, n_query=4100),
    dict(max_pages=1 << 25, n_seq=1 << 10),
], ids=ids)
def test_attention_refuses(lib, bad):
    a = attn_args(**bad)
    assert lib.fwb_kv4_attention_dev(ctypes.byref(a), PTR, 1 << 40, None) == -1
    assert "fwb_kv4_attention" in lib.fwb_last_error().decode()


def test_attention_workspace(lib):
    a = attn_args()
    need = lib.fwb_kv4_attention_workspace(ctypes.byref(a))
    assert need > 0
    for ws, size in ((None, need), (PTR + 4, need), (PTR, need - 1)):
        assert lib.fwb_kv4_attention_dev(ctypes.byref(a), ws, size, None) == -1
        assert "workspace" in lib.fwb_last_error().decode()
    assert lib.fwb_kv4_attention_workspace(None) == 0
    a.head_dim = 8
    assert lib.fwb_kv4_attention_workspace(ctypes.byref(a)) == 0


def test_null_arguments(lib):
    assert lib.fwb_kv4_append_dev(None, None) == -1
    assert lib.fwb_kv4_read_dev(None, None) == -1
    assert lib.fwb_kv4_attention_dev(None, PTR, 1 << 40, None) == -1


def test_page_bytes(lib):
    # 4.5 bits a value, K and V, head_dim filled up to 32s
    for hd in (16, 32, 48, 64, 96, 112, 128):
        for page in (16, 32, 64, 128, 256):
            assert lib.fwb_kv4_page_bytes(hd, page) == page * 2 * (-(-hd // 32) * 18)
    for hd, page in ((0, 16), (8, 16), (144, 16), (64, 0), (64, 24), (64, 512)):
        assert lib.fwb_kv4_page_bytes(hd, page) == 0


SAMPLE = dict(logits=PTR, type=0, n_row=4, n_vocab=100, row_stride=100, uniform=PTR, temperature=PTR, top_k=PTR, top_p=PTR,
              min_p=PTR, token=PTR, logprob=PTR)


@pytest.mark.parametrize("bad", [
    dict(type=8), dict(n_row=0), dict(n_vocab=0), dict(n_vocab=262145, row_stride=262145), dict(n_row=1 << 29), dict(row_stride=99),
    dict(logits=None), dict(uniform=None), dict(token=None), dict(logits=PTR + 2), dict(token=PTR + 1), dict(top_k=PTR + 2),
    dict(min_p=PTR + 1), dict(logprob=PTR + 3),
], ids=ids)
def test_sample_refuses(lib, bad):
    assert lib.fwb_sample_rows_dev(*{**SAMPLE, **bad}.values(), None) == -1
    assert "fwb_sample_rows" in lib.fwb_last_error().decode()
