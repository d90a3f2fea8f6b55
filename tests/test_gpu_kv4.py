"""GPU: append, read and attention of the paged 4-bit cache against their definitions in 64 bits."""
import math

import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(built):
    return pytest.importorskip("torch")


@pytest.fixture(scope="module")
def kv4(torch):
    from fwb import kv4
    torch.zeros(1, device="cuda")
    yield kv4
    kv4.check_status()   # nothing but the tests of bad tables, which look themselves, met one


def noise(torch, seed, *shape, dtype=None, sd=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=gen) * sd).to(dtype or torch.float32)


def angles(torch, n_pos, hd):
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
    return a.cos().float().cuda(), a.sin().float().cuda()


# --- append and read ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 128), (6, 6, 48), (3, 1, 16), (8, 8, 32), (5, 5, 80), (2, 1, 96), (4, 4, 64), (2, 2, 112)])
@pytest.mark.parametrize("halves", [False, True])
def test_append(torch, kv4, dtype, nh, nkv, hd, halves):
    dt = ref.DTYPES[dtype]
    for page, lens, new, nq in ((16, [1, 40, 17, 3], [1, 5, 3, 0], 5), (64, [130], [130], 130), (256, [300, 7], [1, 1], 1)):
        p = ref.Pages(kv4, lens, nkv, hd, page)
        n = len(lens)
        q, k, v = (noise(torch, i, n, nq, h, hd, dtype=dt) for i, h in enumerate((nh, nkv, nkv)))
        cos, sin = angles(torch, 300, hd)
        n_new = torch.tensor(new, dtype=torch.int32, device="cuda")
        q_out = torch.full_like(q, 7.0)
        assert kv4.append(q, k, v, p.cache, p.table, p.lengths, cos=cos, sin=sin, halves=halves, n_new=n_new, q_out=q_out) is q_out
        start = p.lengths - n_new
        outs = {d: kv4.read(p.cache, p.table, start, nq, head_dim=hd, dtype=ref.DTYPES[d], lengths=p.lengths) for d in ("f32", dtype)}
        for s in range(n):
            at = slice(lens[s] - new[s], lens[s])
            want = ref.turned(q[s, :new[s]], cos[at], sin[at], halves)
            # |a||cos| + |b||sin| of the one and |a||sin| + |b||cos| of the other: an fp32 product (2^-24 of it) and an
            # fma of the two (2^-24 of their sum), before the type's rounding
            size = torch.maximum(*(ref.turned(q[s, :new[s]].abs(), cos[at].abs(), e * sin[at].abs(), halves).abs() for e in (-1, 1)))
            far = (q_out[s, :new[s]].double() - want).abs()
            assert bool((far <= want.abs() * ref.half_step(dt) + size * 2.0 ** -22 + 2.0 ** -25).all())
            assert bool((q_out[s, new[s]:] == 7.0).all())
            for got, x in zip(outs["f32"], (ref.turned(k[s, :new[s]], cos[at], sin[at], halves), v[s, :new[s]])):
                assert torch.equal(got[s, :new[s]].double(), ref.held(x))
                assert bool((got[s, new[s]:] == 0).all())
        for a, b in zip(outs["f32"], outs[dtype]):
            assert torch.equal(a.to(dt), b)


def test_append_writes_its_positions_only(torch, kv4):
    nkv, hd, page, lens, new = 2, 80, 32, [45, 64, 9], [3, 33, 9]
    k, v = (noise(torch, i, 3, 40, nkv, hd, dtype=torch.float16) for i in range(2))
    n_new = torch.tensor(new, dtype=torch.int32, device="cuda")
    caches = []
    for fill in (0, 0xff):
        p = ref.Pages(kv4, lens, nkv, hd, page, fill=fill)
        kv4.append(None, k, v, p.cache, p.table, p.lengths, n_new=n_new)
        caches.append(p.cache)
    written = caches[0] == caches[1]
    assert int(written.sum()) == sum(new) * nkv * 2 * 18 * 3          # 3 blocks of 18 bytes each
    assert bool((caches[0][~written] == 0).all()) and bool((caches[1][~written] == 0xff).all())


@pytest.mark.parametrize("halves", [False, True])
def test_append_in_place_on_views(torch, kv4, halves):
    """q, k and v as parts of one projection's rows, q turned in place; the same from copies."""
    nh, nkv, hd, n, nq = 8, 2, 64, 3, 7
    rows = noise(torch, 5, n, nq, nh + 2 * nkv, hd, dtype=torch.bfloat16)
    q, k, v = rows[:, :, :nh], rows[:, :, nh:nh + nkv], rows[:, :, nh + nkv:]
    cos, sin = angles(torch, 64, hd)
    lens = [7, 20, 50]
    a, b = ref.Pages(kv4, lens, nkv, hd, 16), ref.Pages(kv4, lens, nkv, hd, 16)
    want = kv4.append(q.contiguous(), k.contiguous(), v.contiguous(), b.cache, b.table, b.lengths, cos=cos, sin=sin, halves=halves)
    before = rows[:, :, nh:].clone()
    kv4.append(q, k, v, a.cache, a.table, a.lengths, cos=cos, sin=sin, halves=halves, q_out=q)
    assert torch.equal(q, want) and torch.equal(a.cache, b.cache) and torch.equal(rows[:, :, nh:], before)


def test_append_without_rotation(torch, kv4):
    q, k, v = noise(torch, 1, 2, 3, 4, 32), noise(torch, 2, 2, 3, 2, 32), noise(torch, 3, 2, 3, 2, 32)
    p = ref.Pages(kv4, [3, 9], 2, 32, 16)
    assert torch.equal(kv4.append(q, k, v, p.cache, p.table, p.lengths), q)
    got = kv4.read(p.cache, p.table, p.lengths - 3, 3, head_dim=32, dtype=torch.float32)
    assert torch.equal(got[0].double(), ref.held(k)) and torch.equal(got[1].double(), ref.held(v))


def test_blocks_of_extremes(torch, kv4):
    """Blocks of zeros, of subnormal scales, past the scales' range, on code borders, with two largest magnitudes, not finite."""
    rows = torch.zeros(1, 16, 1, 64)
    rows[0, 1] = 1e-30
    rows[0, 2, 0, :32] = torch.linspace(-3e-6, 3e-6, 32)
    rows[0, 3, 0, 5], rows[0, 3, 0, 7] = 1e30, -3.0
    rows[0, 4, 0, :32] = torch.arange(32) * 0.25 - 4.0            # d = 0.5 exactly: every second value on a border
    rows[0, 5, 0, :32] = (torch.arange(32) % 16).float() * 0.5 - 3.5
    rows[0, 5, 0, 3], rows[0, 5, 0, 30] = 4.0, -4.0               # the positive one decides
    rows[0, 6, 0, 40] = math.inf
    rows[0, 7, 0, 2] = math.nan
    rows[0, 8, 0, 33] = -math.inf
    rows[0, 9] = 524032.0
    rows[0, 10] = -600000.0
    rows[0, 11] = noise(torch, 9, 64).cpu() * 1e-7
    rows[0, 12] = noise(torch, 10, 64).cpu() * 1e5
    rows[0, 13, 0, :] = 2.0 ** -24 * 8
    rows[0, 14, 0, :] = -1.0
    rows[0, 15, 0, ::2] = 1.0
    rows = rows.cuda()
    p = ref.Pages(kv4, [16], 1, 64, 16)
    kv4.append(None, rows, rows, p.cache, p.table, p.lengths)
    for got in kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), 16, head_dim=64, dtype=torch.float32):
        want = ref.held(rows).float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
        assert int(torch.isnan(got).sum()) == 3 * 32


def test_read_ranges(torch, kv4):
    lens = [0, 1, 100, 33]
    p, k, v = ref.filled(kv4, lens, 2, 48, 32)
    for first, n in ((0, 100), (-5, 20), (31, 3), (90, 50)):
        start = torch.full((4,), first, dtype=torch.int32, device="cuda")
        got = kv4.read(p.cache, p.table, start, n, head_dim=48, dtype=torch.float32, lengths=p.lengths)
        for x, whole in zip(got, (k, v)):
            for s in range(4):
                for i in range(n):
                    at = first + i
                    want = whole[s, at] if 0 <= at < lens[s] else torch.zeros(2, 48, device="cuda")
                    assert torch.equal(x[s, i], want), (s, at)


# --- attention ------------------------------------------------------------------------------------------
SHAPES = [  # heads, tokens, page, lengths
    (4, 2, 128, 1, 16, [0, 1, 2, 15, 16, 17, 200]), (32, 8, 128, 1, 64, [777]), (6, 6, 48, 1, 32, [251, 33, 5]),
    (8, 1, 64, 1, 128, [129, 128]), (64, 8, 128, 1, 64, [300, 64, 1, 0]), (16, 1, 96, 1, 16, [90, 300]), (40, 1, 80, 1, 32, [70, 33]),
    (4, 2, 128, 7, 16, [7, 8, 90, 3]), (5, 1, 32, 3, 256, [500, 3]), (2, 2, 16, 33, 64, [33, 100]), (12, 4, 112, 40, 32, [64, 41, 39]),
    (4, 4, 64, 130, 16, [130, 200]), (3, 3, 96, 2, 64, [1000, 4])]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,nq,page,lens", SHAPES, ids=lambda x: str(x).replace(" ", ""))
def test_attention(torch, kv4, dtype, nh, nkv, hd, nq, page, lens):
    p, k, v = ref.filled(kv4, lens, nkv, hd, page, seed=len(lens))
    q = noise(torch, 77, len(lens), nq, nh, hd, dtype=ref.DTYPES[dtype], sd=2.0)
    plan = kv4.Attention(n_seq=len(lens), n_query=nq, n_head=nh, n_head_kv=nkv, head_dim=hd, dtype=q.dtype, page_size=page,
                         n_page=p.n_page, max_pages=p.table.shape[1])
    out, lse = plan(q, p.cache, p.table, p.lengths)
    ref.check_attention(out, lse, q, k, v, lens)
    again = plan(q, p.cache, p.table, p.lengths)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,nq,n", [(8, 2, 1, 20011), (4, 1, 5, 9001), (2, 2, 64, 4500), (16, 1, 1, 6001)])
def test_attention_long(torch, kv4, dtype, nh, nkv, nq, n):
    p, k, v = ref.filled(kv4, [n, n // 3], nkv, 128, 64)
    q = noise(torch, 3, 2, nq, nh, 128, dtype=ref.DTYPES[dtype], sd=2.0)
    plan = kv4.Attention(n_seq=2, n_query=nq, n_head=nh, n_head_kv=nkv, head_dim=128, dtype=q.dtype, page_size=64,
                         n_page=p.n_page, max_pages=p.table.shape[1])
    out, lse = plan(q, p.cache, p.table, p.lengths)
    ref.check_attention(out, lse, q, k, v, [n, n // 3])
    again = plan(q, p.cache, p.table, p.lengths)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("nq,gq", [(4, 1), (4, 3), (9, 4), (50, 2), (100, 8)])
def test_attention_of_a_padded_batch(torch, kv4, dtype, nq, gq):
    lens = [60, 200, 33, 9, 0, 120]
    new = torch.tensor([nq, 1, 0, min(nq, 9), 0, max(1, nq - 1)], dtype=torch.int32, device="cuda")
    p, k, v = ref.filled(kv4, lens, 2, 64, 16)
    q = noise(torch, 4, 6, nq, 2 * gq, 64, dtype=ref.DTYPES[dtype])
    plan = kv4.Attention(n_seq=6, n_query=nq, n_head=2 * gq, n_head_kv=2, head_dim=64, dtype=q.dtype, page_size=16,
                         n_page=p.n_page, max_pages=p.table.shape[1])
    for s in range(6):
        q[s, int(new[s]):] = math.nan                              # rows that nobody reads
    out, lse = torch.full_like(q, 5.0), torch.full(q.shape[:3], 5.0, device="cuda")
    plan(q, p.cache, p.table, p.lengths, n_new=new, out=out, lse=lse)
    ref.check_attention(out, lse, q, k, v, lens, new)
    for s in range(6):
        assert bool((out[s, int(new[s]):] == 5).all()) and bool((lse[s, int(new[s]):] == 5).all())
    fresh = plan(q, p.cache, p.table, p.lengths, n_new=new)
    for s in range(6):
        assert torch.equal(fresh[0][s, :int(new[s])], out[s, :int(new[s])]) and bool((fresh[0][s, int(new[s]):] == 0).all())


def test_attention_of_strided_queries(torch, kv4):
    lens = [100, 30]
    p, k, v = ref.filled(kv4, lens, 2, 64, 32)
    rows = noise(torch, 4, 2, 3, 12, 64, dtype=torch.float16)
    q = rows[:, :, 2:10]
    plan = kv4.Attention(n_seq=2, n_query=3, n_head=8, n_head_kv=2, head_dim=64, dtype=q.dtype, page_size=32, n_page=p.n_page,
                         max_pages=p.table.shape[1], scale=0.3)
    out, lse = plan(q, p.cache, p.table, p.lengths)
    ref.check_attention(out, lse, q, k, v, lens, scale=0.3)
    t = q.transpose(1, 2).contiguous().transpose(1, 2)             # heads outside of tokens
    assert torch.equal(plan(t, p.cache, p.table, p.lengths)[0], out)


def test_sequences_share_pages(torch, kv4):
    p, k, v = ref.filled(kv4, [96, 96], 2, 128, 32)
    table = p.table.clone()
    table[1, :2] = table[0, :2]                                    # 64 positions in common
    k[1, :64], v[1, :64] = k[0, :64], v[0, :64]
    q = noise(torch, 4, 2, 1, 8, 128)
    plan = kv4.Attention(n_seq=2, n_head=8, n_head_kv=2, head_dim=128, dtype=q.dtype, page_size=32, n_page=p.n_page, max_pages=3)
    ref.check_attention(*plan(q, p.cache, table, p.lengths), q, k, v, [96, 96])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_finite_reaches_those_that_see_it(torch, kv4, dtype, which, bad):
    """Position 40 of 50 holds it; tokens 0..9 see 41..50 positions less the later ones."""
    dt = ref.DTYPES[dtype]
    p = ref.Pages(kv4, [50], 2, 64, 16)
    kv = noise(torch, 6, 2, 1, 50, 2, 64, dtype=dt)
    clean = kv.clone()
    kv[0 if which == "k" else 1, 0, 40, 1, 3] = bad
    kv4.append(None, kv[0], kv[1], p.cache, p.table, p.lengths)
    q = noise(torch, 7, 1, 20, 4, 64, dtype=dt)
    plan = kv4.Attention(n_seq=1, n_query=20, n_head=4, n_head_kv=2, head_dim=64, dtype=dt, page_size=16, n_page=p.n_page,
                         max_pages=p.table.shape[1])
    out, lse = plan(q, p.cache, p.table, p.lengths)
    o = ref.Pages(kv4, [50], 2, 64, 16)
    kv4.append(None, clean[0], clean[1], o.cache, o.table, o.lengths)
    want, want_lse = plan(q, o.cache, o.table, o.lengths)
    seen = torch.arange(31, 51, device="cuda") > 40                # positions that token t sees: 31 + t
    assert torch.equal(out[0, ~seen], want[0, ~seen]) and torch.equal(out[0, :, :2], want[0, :, :2])
    assert torch.equal(lse[0, ~seen], want_lse[0, ~seen])
    got = out[0, seen][:, 2:]
    if which == "k":
        assert bool(torch.isnan(got).all()) and bool(torch.isnan(lse[0, seen][:, 2:]).all())
    else:
        assert bool(torch.isnan(got[..., :32]).all())              # its block of 32 dimensions
        assert torch.equal(got[..., 32:], want[0, seen][:, 2:, 32:]) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_queries_that_are_not_finite(torch, kv4, dtype):
    p, k, v = ref.filled(kv4, [50, 0], 1, 64, 16)
    q = noise(torch, 7, 2, 3, 4, 64, dtype=ref.DTYPES[dtype])
    q[0, 1, 2, 5], q[0, 2, 3, 60], q[1, 2, 0, 0] = math.nan, math.inf, math.nan
    plan = kv4.Attention(n_seq=2, n_query=3, n_head=4, n_head_kv=1, head_dim=64, dtype=q.dtype, page_size=16, n_page=p.n_page,
                         max_pages=p.table.shape[1])
    out, lse = plan(q, p.cache, p.table, p.lengths)
    odd = torch.zeros(2, 3, 4, dtype=torch.bool, device="cuda")
    odd[0, 1, 2] = odd[0, 2, 3] = True
    assert torch.equal(torch.isnan(out).all(-1), odd) and torch.equal(torch.isnan(out).any(-1), odd)
    assert torch.equal(torch.isnan(lse), odd)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())   # they see nothing


@pytest.mark.parametrize("dtype,size", [("f32", 1e-20), ("f32", 1e15), ("bf16", 1e-30), ("bf16", 1e10), ("f16", 6e4), ("f16", 1e-6)])
def test_sizes_of_queries(torch, kv4, dtype, size):
    """Scores that are all nearly equal, or one that has all the weight."""
    p, k, v = ref.filled(kv4, [300], 2, 128, 32)
    q = noise(torch, 8, 1, 1, 8, 128).clamp(-1, 1).mul(size).to(ref.DTYPES[dtype])
    scale = 1.0 / size / math.sqrt(128) if size > 1 else None      # (else exp of 1e15)
    plan = kv4.Attention(n_seq=1, n_head=8, n_head_kv=2, head_dim=128, dtype=q.dtype, page_size=32, n_page=p.n_page,
                         max_pages=p.table.shape[1], scale=scale or 0.0)
    ref.check_attention(*plan(q, p.cache, p.table, p.lengths), q, k, v, [300], scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_one_score_far_above(torch, kv4, dtype):
    """The last position's score passes the first ones' by far more than fp16 holds, and the other way round."""
    for at in (0, 250, 499):
        p = ref.Pages(kv4, [500], 1, 64, 16)
        kv = noise(torch, 6, 2, 1, 500, 1, 64) * 0.5
        q = noise(torch, 7, 1, 1, 4, 64, dtype=ref.DTYPES[dtype])
        kv[0, 0, at, 0] = q[0, 0, 0].float() * 8
        kv4.append(None, kv[0], kv[1], p.cache, p.table, p.lengths)
        k, v = kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), 500, head_dim=64, dtype=torch.float32)
        plan = kv4.Attention(n_seq=1, n_head=4, n_head_kv=1, head_dim=64, dtype=q.dtype, page_size=16, n_page=p.n_page,
                             max_pages=p.table.shape[1])
        ref.check_attention(*plan(q, p.cache, p.table, p.lengths), q, k, v, [500])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gq", [1, 12, 30])
def test_codes_that_are_zero_add_nothing(torch, kv4, dtype, gq):
    """A score of a few small products keeps its digits beside large query values that meet zeros."""
    hd, n = 64, 37
    p = ref.Pages(kv4, [n], 1, hd, 16)
    k = torch.zeros(1, n, 1, hd, device="cuda")
    k[..., 5], k[..., 37] = -8.0, -8.0       # the blocks' scales are 1
    k[..., 11], k[..., 50] = 1.0, 3.0
    kv4.append(torch.zeros(1, n, gq, hd, device="cuda"), k, k, p.cache, p.table, p.lengths)
    q = noise(torch, 3, 1, 1, gq, hd).abs().add(1.0)
    q[..., 5], q[..., 37] = 0.0, 0.0
    q[..., 11], q[..., 50] = q[..., 11] / 1024, q[..., 50] / 2048
    q = q.to(ref.DTYPES[dtype])
    plan = kv4.Attention(n_seq=1, n_query=1, n_head=gq, n_head_kv=1, head_dim=hd, dtype=q.dtype, page_size=16, n_page=p.cache.shape[0],
                         max_pages=p.table.shape[1], scale=1024.0)
    lse = torch.empty(1, 1, gq, device="cuda")
    plan(q, p.cache, p.table, p.lengths, lse=lse)
    want = 1024 * (q[0, 0, :, 11].double() + 3 * q[0, 0, :, 50].double()) + math.log(n)
    # two products and their sum at 2^-23 of their size, the factor back at 2^-23, the log of the sum and its addition
    # 2^-22: below 2^-20 of all of it (fp32 queries: their two halves carry 22 bits of the row's largest, 4 / 2^22 * 2^10 more)
    slack = 2 * 1024 * 4 * 2.0 ** -22 if dtype == "f32" else 0.0
    assert bool(((lse[0, 0].double() - want).abs() <= want.abs() * 2.0 ** -20 + slack).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("sizes", [(1e-4, 1e-4), (1.0, 1e4), (1e4, 1.0), (1e-3, 30.0)])
def test_sizes_of_values(torch, kv4, dtype, sizes):
    """Values whose scales grow or shrink along the sequence."""
    n = 400
    p = ref.Pages(kv4, [n], 2, 64, 16)
    kv = noise(torch, 6, 2, 1, n, 2, 64)
    kv[1] *= torch.logspace(math.log10(sizes[0]), math.log10(sizes[1]), n, device="cuda")[None, :, None, None]
    kv4.append(None, kv[0], kv[1], p.cache, p.table, p.lengths)
    k, v = kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), n, head_dim=64, dtype=torch.float32)
    q = noise(torch, 7, 1, 2, 4, 64, dtype=ref.DTYPES[dtype])
    plan = kv4.Attention(n_seq=1, n_query=2, n_head=4, n_head_kv=2, head_dim=64, dtype=q.dtype, page_size=16, n_page=p.n_page,
                         max_pages=p.table.shape[1])
    ref.check_attention(*plan(q, p.cache, p.table, p.lengths), q, k, v, [n])


def test_many_short_sequences(torch, kv4):
    lens = [(i * 37) % 90 for i in range(300)]
    p, k, v = ref.filled(kv4, lens, 2, 32, 16)
    q = noise(torch, 9, 300, 1, 4, 32)
    plan = kv4.Attention(n_seq=300, n_head=4, n_head_kv=2, head_dim=32, dtype=q.dtype, page_size=16, n_page=p.n_page,
                         max_pages=p.table.shape[1])
    ref.check_attention(*plan(q, p.cache, p.table, p.lengths), q, k, v, lens)


# --- tables -----------------------------------------------------------------------------------------------
def test_bad_tables_are_told(torch, kv4):
    from fwb.model import FwbError
    hd, page = 32, 16
    p, k, v = ref.filled(kv4, [60], 1, hd, page)
    kv4.check_status()
    before = p.cache.clone()
    row = noise(torch, 1, 1, 1, 1, hd)
    q = noise(torch, 2, 1, 1, 2, hd)
    for entry in (p.n_page, -1, 1 << 30, -(1 << 31)):
        table = p.table.clone()
        table[0, 1] = entry                                        # positions 16..31
        at = torch.tensor([20], dtype=torch.int32, device="cuda")
        kv4.append(None, row, row, p.cache, table, at)
        with pytest.raises(FwbError, match="page outside"):
            kv4.check_status()
        kv4.check_status()
        x, y = kv4.read(p.cache, table, torch.zeros_like(at), 60, head_dim=hd, dtype=torch.float32)
        assert bool((x[0, 16:32] == 0).all()) and torch.equal(x[0, :16], k[0, :16]) and torch.equal(y[0, 32:], v[0, 32:])
        with pytest.raises(FwbError, match="page outside"):
            kv4.check_status()
        plan = kv4.Attention(n_seq=1, n_head=2, n_head_kv=1, head_dim=hd, dtype=q.dtype, page_size=page, n_page=p.n_page, max_pages=4)
        got = plan(q, p.cache, table, p.lengths)
        with pytest.raises(FwbError, match="page outside"):
            kv4.check_status()
        keep = [i for i in range(60) if not 16 <= i < 32]
        ref.check_attention(*got, q, k[:, keep], v[:, keep], [44])
    cos, sin = angles(torch, 30, hd)
    q_out = torch.full_like(q, 3.0)
    for length, c, s in ((65, None, None), (31, cos, sin)):         # past the table, past the angles
        kv4.append(q, row, row, p.cache, p.table, torch.tensor([length], dtype=torch.int32, device="cuda"), cos=c, sin=s, q_out=q_out)
        with pytest.raises(FwbError, match="position past"):
            kv4.check_status()
        assert bool((q_out == 3).all())
    kv4.append(q, row, row, p.cache, p.table, torch.tensor([0], dtype=torch.int32, device="cuda"), q_out=q_out)  # position -1
    kv4.check_status()
    assert bool((q_out == 3).all()) and torch.equal(p.cache, before)


def test_lengths_are_held_to_the_table(torch, kv4):
    p, k, v = ref.filled(kv4, [64], 1, 32, 16)
    q = noise(torch, 2, 1, 1, 2, 32)
    plan = kv4.Attention(n_seq=1, n_head=2, n_head_kv=1, head_dim=32, dtype=q.dtype, page_size=16, n_page=p.n_page, max_pages=4)
    want = plan(q, p.cache, p.table, p.lengths)
    for n in (65, 1 << 30, (1 << 31) - 1):
        got = plan(q, p.cache, p.table, torch.tensor([n], dtype=torch.int32, device="cuda"))
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    out, lse = plan(q, p.cache, p.table, torch.tensor([-5], dtype=torch.int32, device="cuda"))
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_pages_past_4_gb(torch, kv4):
    """A cache of over 2^32 bytes whose pages in use lie at its end and beginning."""
    hd, page, heads = 128, 256, 8
    n_page = (1 << 32) // (heads * kv4.page_bytes(hd, page)) + 40
    cache = kv4.empty(n_page, heads, hd, page)
    table = torch.tensor([[n_page - 1, 0, n_page - 30, 1]], dtype=torch.int32, device="cuda")
    n = 900
    kv = noise(torch, 6, 2, 1, n, heads, hd, dtype=torch.float16)
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    kv4.append(None, kv[0], kv[1], cache, table, lengths)
    k, v = kv4.read(cache, table, torch.zeros_like(lengths), n, head_dim=hd, dtype=torch.float32)
    assert torch.equal(k.double(), ref.held(kv[0])) and torch.equal(v.double(), ref.held(kv[1]))
    q = noise(torch, 7, 1, 1, 32, hd, dtype=torch.float16)
    plan = kv4.Attention(n_seq=1, n_head=32, n_head_kv=heads, head_dim=hd, dtype=q.dtype, page_size=page, n_page=n_page, max_pages=4)
    ref.check_attention(*plan(q, cache, table, lengths), q, k, v, [n])


# --- streams, graphs, workspaces ------------------------------------------------------------------------------
def test_graphs_and_streams_side_by_side(torch, kv4):
    lens = [3000, 700]
    p, k, v = ref.filled(kv4, lens, 2, 128, 64)
    plan = kv4.Attention(n_seq=2, n_head=8, n_head_kv=2, head_dim=128, dtype=torch.float16, page_size=64, n_page=p.n_page,
                         max_pages=p.table.shape[1])
    qs = [noise(torch, i, 2, 1, 8, 128, dtype=torch.float16) for i in range(4)]
    wants = [plan(q, p.cache, p.table, p.lengths) for q in qs]
    outs = [tuple(torch.empty_like(t) for t in w) for w in wants]
    graphs = []
    for q, o in zip(qs[:2], outs[:2]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plan(q, p.cache, p.table, p.lengths, out=o[0], lse=o[1])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o[0].zero_(), o[1].zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            for q, o, st in zip(qs[2:], outs[2:], streams[2:]):
                with torch.cuda.stream(st):
                    plan(q, p.cache, p.table, p.lengths, out=o[0], lse=o[1])
        torch.cuda.synchronize()
        for o, w in zip(outs, wants):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


def test_one_workspace_for_calls_of_other_sizes(torch, kv4):
    """A workspace serves calls of any sizes one after the other (the C interface's promise)."""
    import ctypes
    lib = kv4.native.product()
    calls = []
    for nh, nkv, hd, nq, lens in ((8, 2, 128, 1, [5000]), (32, 2, 64, 3, [900, 40]), (64, 8, 128, 1, [300] * 9), (4, 4, 32, 64, [700])):
        p, _, _ = ref.filled(kv4, lens, nkv, hd, 16)
        q = noise(torch, 1, len(lens), nq, nh, hd, dtype=torch.float16)
        plan = kv4.Attention(n_seq=len(lens), n_query=nq, n_head=nh, n_head_kv=nkv, head_dim=hd, dtype=q.dtype, page_size=16,
                             n_page=p.n_page, max_pages=p.table.shape[1])
        out, lse = plan(q, p.cache, p.table, p.lengths)
        calls.append((plan, p, q, out, lse, out.clone(), lse.clone()))
    ws = torch.zeros(max(c[0].workspace_bytes for c in calls), dtype=torch.uint8, device="cuda")
    for _ in range(3):
        for plan, p, q, out, lse, want, want_lse in calls:
            out.zero_(), lse.zero_()
            assert lib.fwb_kv4_attention_dev(ctypes.byref(plan.a), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
            assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_append_and_attention_in_a_replayed_graph(torch, kv4):
    """A step captured once and replayed while the lengths grow on the device."""
    n, nh, nkv, hd, page, steps = 3, 8, 2, 64, 16, 40
    p = ref.Pages(kv4, [0] * n, nkv, hd, page, room=steps)
    cos, sin = angles(torch, steps, hd)
    q, k, v = (torch.zeros(n, 1, h, hd, device="cuda") for h in (nh, nkv, nkv))
    plan = kv4.Attention(n_seq=n, n_head=nh, n_head_kv=nkv, head_dim=hd, dtype=q.dtype, page_size=page, n_page=p.n_page,
                         max_pages=p.table.shape[1])
    out, lse, turned = torch.empty_like(q), torch.empty(n, 1, nh, device="cuda"), torch.empty_like(q)

    def step():
        p.lengths.add_(1)
        kv4.append(q, k, v, p.cache, p.table, p.lengths, cos=cos, sin=sin, q_out=turned)
        plan(turned, p.cache, p.table, p.lengths, out=out, lse=lse)

    step()                                                         # (its position is written again below)
    p.lengths.zero_()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    p.lengths.zero_()
    for i in range(steps):
        for j, t in enumerate((q, k, v)):
            t.copy_(noise(torch, 100 * i + j, *t.shape))
        g.replay()
        got = kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), i + 1, head_dim=hd, dtype=torch.float32, lengths=p.lengths)
        ref.check_attention(out, lse, turned, *got, [i + 1] * n)


# --- refusals of the Python layer --------------------------------------------------------------------------------
def test_refusals(torch, kv4):
    p, _, _ = ref.filled(kv4, [40, 20], 2, 64, 32)
    plan = kv4.Attention(n_seq=2, n_head=4, n_head_kv=2, head_dim=64, dtype=torch.float16, page_size=32, n_page=p.n_page,
                         max_pages=p.table.shape[1])
    good = dict(q=noise(torch, 1, 2, 1, 4, 64, dtype=torch.float16), cache=p.cache, pages=p.table, lengths=p.lengths)
    plan(**good)
    for bad in (dict(q=None), dict(q=good["q"].float()), dict(q=good["q"][:1]), dict(q=good["q"].cpu()), dict(cache=None),
                dict(cache=p.cache[1:]), dict(cache=p.cache.float()), dict(pages=None), dict(pages=p.table.long()), dict(pages=p.table[:, :1]),
                dict(lengths=None), dict(lengths=p.lengths.long()), dict(lengths=p.lengths[:1]), dict(n_new=p.lengths[:1]),
                dict(out=good["q"].float()), dict(lse=torch.zeros(2, 1, 4, device="cuda", dtype=torch.float16))):
        with pytest.raises(ValueError):
            plan(**{**good, **bad})
    k = noise(torch, 1, 2, 3, 2, 64)
    q = noise(torch, 2, 2, 3, 4, 64)
    cos, sin = angles(torch, 50, 64)
    good = dict(q=q, k=k, v=k, cache=p.cache, pages=p.table, lengths=p.lengths, cos=cos, sin=sin)
    for bad in (dict(k=None), dict(k=k.double()), dict(v=None), dict(v=k[:1]), dict(v=k.half()), dict(q=q.half()), dict(q=None, q_out=q),
                dict(q_out=q[:, :, :2]), dict(cos=None), dict(sin=None), dict(cos=cos[:, :8]), dict(cos=cos[:9]), dict(cache=p.cache[:, :1]),
                dict(cache=p.cache[:, :, :100]), dict(pages=p.table[:1]), dict(lengths=p.lengths.cpu()), dict(k=k.cpu()),
                dict(n_new=p.lengths.long()), dict(q_out=torch.zeros(2 * 3 * 4 * 64 + 64, device="cuda")[64:].view(2, 3, 4, 64).to(torch.float16))):
        with pytest.raises(ValueError):
            kv4.append(**{**good, **bad})
    whole = torch.zeros(2 * 3 * 4 * 64 + 64, device="cuda")
    with pytest.raises(ValueError, match="apart"):
        kv4.append(**{**good, "q": whole[:-64].view(2, 3, 4, 64), "q_out": whole[64:].view(2, 3, 4, 64)})
    for bad in (dict(cache=None), dict(start=None), dict(start=p.lengths.long()), dict(n=-1), dict(head_dim=96), dict(dtype=torch.float64),
                dict(lengths=p.lengths[:1]), dict(k=k)):
        with pytest.raises(ValueError):
            kv4.read(**{**dict(cache=p.cache, pages=p.table, start=p.lengths, n=3, head_dim=64, dtype=torch.float16), **bad})
