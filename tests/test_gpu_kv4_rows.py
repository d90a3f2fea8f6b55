"""GPU: attention of many query rows over the 4-bit cache (chunks of prompts of several sequences), which takes another
kernel than test_gpu_kv4.py's calls once there are tiles enough for the device."""
import math

import pytest

import kv4_ref as ref
from test_gpu_kv4 import kv4, noise, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def plan_of(kv4, p, q, nkv, **kw):
    n, nq, nh, hd = q.shape
    return kv4.Attention(n_seq=n, n_query=nq, n_head=nh, n_head_kv=nkv, head_dim=hd, dtype=q.dtype, page_size=p.page,
                         n_page=p.n_page, max_pages=p.table.shape[1], **kw)


SHAPES = [  # sequences, tokens, query heads, KV heads, head_dim, page, longest
    (16, 16, 32, 8, 128, 64, 300), (16, 33, 16, 8, 64, 16, 130), (60, 64, 2, 2, 128, 32, 200), (20, 40, 16, 8, 112, 16, 170),
    (14, 130, 8, 8, 128, 128, 700), (37, 13, 32, 4, 64, 16, 1000), (16, 70, 8, 8, 48, 32, 90), (1, 600, 32, 8, 128, 256, 650)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("n,nq,nh,nkv,hd,page,longest", SHAPES)
def test_many_rows(torch, kv4, dtype, n, nq, nh, nkv, hd, page, longest):
    lens = [max(nq, longest - i * 37 % longest) if i % 5 else longest for i in range(n)]
    lens[n // 2] = nq                                              # a prompt's beginning
    p, k, v = ref.filled(kv4, lens, nkv, hd, page, seed=n)
    q = noise(torch, 5, n, nq, nh, hd, dtype=ref.DTYPES[dtype], sd=2.0)
    plan = plan_of(kv4, p, q, nkv)
    out, lse = plan(q, p.cache, p.table, p.lengths)
    ref.check_attention(out, lse, q, k, v, lens)
    again = plan(q, p.cache, p.table, p.lengths)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    kv4.check_status()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_items_are_cut(torch, kv4, dtype, hd):
    """More items than CTAs, of many tiles and unequal: their parts are added."""
    n, nq, nkv = 24, 64, 8
    lens = [2500 if i % 7 == 0 else 1100 + 60 * i for i in range(n)]
    p, k, v = ref.filled(kv4, lens, nkv, hd, 64, seed=2)
    q = noise(torch, 6, n, nq, nkv, hd, dtype=ref.DTYPES[dtype], sd=2.0)
    plan = plan_of(kv4, p, q, nkv)
    out, lse = plan(q, p.cache, p.table, p.lengths)
    ref.check_attention(out, lse, q, k, v, lens)
    again = plan(q, p.cache, p.table, p.lengths)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_padded_batch(torch, kv4, dtype):
    n, nq, nkv, gq, hd = 16, 40, 8, 2, 128
    lens = [40 + 23 * i for i in range(n)]
    lens[3], lens[4], lens[5] = 0, 7, 39                           # shorter than their new tokens
    new = [40, 1, 0, 40, 40, 39, 13] + [40 - i for i in range(n - 7)]
    p, k, v = ref.filled(kv4, lens, nkv, hd, 32)
    q = noise(torch, 5, n, nq, nkv * gq, hd, dtype=ref.DTYPES[dtype])
    n_new = torch.tensor(new, dtype=torch.int32, device="cuda")
    for s in range(n):
        q[s, new[s]:] = math.nan
    out, lse = torch.full_like(q, 5.0), torch.full(q.shape[:3], 5.0, device="cuda")
    plan_of(kv4, p, q, nkv)(q, p.cache, p.table, p.lengths, n_new=n_new, out=out, lse=lse)
    ref.check_attention(out, lse, q, k, v, lens, n_new)
    for s in range(n):
        assert bool((out[s, new[s]:] == 5).all()) and bool((lse[s, new[s]:] == 5).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_finite_reaches_those_that_see_it(torch, kv4, dtype, which, bad):
    n, nq, nkv, hd, at = 16, 70, 8, 128, 130
    dt = ref.DTYPES[dtype]
    lens = [200] * n
    kv = noise(torch, 6, 2, n, 200, nkv, hd, dtype=dt)
    clean = kv.clone()
    kv[0 if which == "k" else 1, 2, at, 1, 70] = bad               # sequence 2, head 1, block 2
    q = noise(torch, 7, n, nq, nkv, hd, dtype=dt)
    got = []
    for x in (kv, clean):
        p = ref.Pages(kv4, lens, nkv, hd, 16)
        kv4.append(None, x[0], x[1], p.cache, p.table, p.lengths)
        got.append(plan_of(kv4, p, q, nkv)(q, p.cache, p.table, p.lengths))
    (out, lse), (want, want_lse) = got
    hit = torch.zeros(n, nq, nkv, dtype=torch.bool, device="cuda")
    hit[2, :, 1] = torch.arange(131, 201, device="cuda") > at      # token t sees 131 + t positions
    assert torch.equal(out[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])
    if which == "k":
        assert bool(torch.isnan(out[hit]).all()) and bool(torch.isnan(lse[hit]).all())
    else:
        assert bool(torch.isnan(out[hit][:, 64:96]).all()) and torch.equal(lse, want_lse)
        # the others' weights are formed with another largest scale, a power of two: nothing but subnormal products change
        rest = torch.cat([out[hit][:, :64], out[hit][:, 96:]], 1)
        assert torch.equal(rest, torch.cat([want[hit][:, :64], want[hit][:, 96:]], 1))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_queries_and_sizes(torch, kv4, dtype):
    """Queries that are not finite; values that grow by 10^8 along the sequence; keys of very unequal positions."""
    n, nq, nkv, hd = 16, 64, 8, 64
    lens = [150 + 11 * i for i in range(n)]
    p = ref.Pages(kv4, lens, nkv, hd, 64)
    most = max(lens)
    kv = noise(torch, 6, 2, n, most, nkv, hd)
    kv[1] *= torch.logspace(-4, 4, most, device="cuda")[:, None, None]
    kv[0, :, ::3] *= 1e-3
    kv[0, :, 7] = 0
    kv[1, :, 9] = 0
    kv4.append(None, kv[0], kv[1], p.cache, p.table, p.lengths, n_new=p.lengths)
    k, v = kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), most, head_dim=hd, dtype=torch.float32, lengths=p.lengths)
    q = noise(torch, 7, n, nq, nkv, hd, dtype=ref.DTYPES[dtype], sd=2.0)
    plan = plan_of(kv4, p, q, nkv)
    out, lse = plan(q, p.cache, p.table, p.lengths)
    ref.check_attention(out, lse, q, k, v, lens)
    odd = q.clone()
    odd[1, 5, 2, 63], odd[3, 60, 7, 0] = math.nan, math.inf
    got, got_lse = plan(odd, p.cache, p.table, p.lengths)
    hit = torch.zeros(n, nq, nkv, dtype=torch.bool, device="cuda")
    hit[1, 5, 2] = hit[3, 60, 7] = True
    assert bool(torch.isnan(got[hit]).all()) and bool(torch.isnan(got_lse[hit]).all())
    assert not bool(torch.isnan(got[~hit]).any())
    ref.check_attention(torch.where(hit[..., None], out, got), torch.where(hit, lse, got_lse), q, k, v, lens)


def test_bad_pages(torch, kv4):
    from fwb.model import FwbError
    n, nq, nkv, hd = 16, 64, 8, 128
    lens = [300] * n
    p, k, v = ref.filled(kv4, lens, nkv, hd, 64)
    q = noise(torch, 7, n, nq, nkv, hd, dtype=torch.float16)
    table = p.table.clone()
    table[4, 1], table[9, 2] = p.n_page, -7                        # positions 64..127, 128..191
    out, lse = plan_of(kv4, p, q, nkv)(q, p.cache, table, p.lengths)
    with pytest.raises(FwbError, match="page outside"):
        kv4.check_status()
    kv4.check_status()
    good = [s for s in range(n) if s not in (4, 9)]
    ref.check_attention(out[good], lse[good], q[good], k[good], v[good], [300] * len(good))
    for s, first in ((4, 64), (9, 128)):
        keep = [i for i in range(300) if not first <= i < first + 64]
        ref.check_attention(out[s:s + 1], lse[s:s + 1], q[s:s + 1], k[s:s + 1, keep], v[s:s + 1, keep], [236])


def test_graphs_and_streams_side_by_side(torch, kv4):
    n, nq, nkv, hd = 24, 64, 8, 128
    lens = [900 + 40 * i for i in range(n)]
    p, _, _ = ref.filled(kv4, lens, nkv, hd, 64)
    qs = [noise(torch, i, n, nq, nkv, hd, dtype=torch.float16) for i in range(3)]
    plan = plan_of(kv4, p, qs[0], nkv)
    wants = [plan(q, p.cache, p.table, p.lengths) for q in qs]
    outs = [tuple(torch.empty_like(t) for t in w) for w in wants]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan(qs[0], p.cache, p.table, p.lengths, out=outs[0][0], lse=outs[0][1])
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for o in outs:
            o[0].zero_(), o[1].zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(streams[0]):
                g.replay()
            for q, o, st in zip(qs[1:], outs[1:], streams[1:]):
                with torch.cuda.stream(st):
                    plan(q, p.cache, p.table, p.lengths, out=o[0], lse=o[1])
        torch.cuda.synchronize()
        for o, w in zip(outs, wants):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])
    kv4.check_status()
