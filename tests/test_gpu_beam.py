"""GPU: the beam-search operators (fwb.beam) against their definitions in 64
bits, at the sizes, lengths, masks and layouts where such kernels go wrong."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# unit roundoff of the type that outputs and, for the 16-bit types, the
# probabilities are rounded to
ROUND = {"torch.float32": 2.0 ** -24, "torch.float16": 2.0 ** -11, "torch.bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch(built):
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.fixture(scope="module")
def beam(torch):
    from fwb import beam
    return beam


def dtype_of(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


# --- attention -------------------------------------------------------------------
def attn_ref(torch, q, pk, pv, sk, sv, plen, slen, slots, n_beam, scale):
    """(out, lse, tolerance of out, tolerance of lse without the type's rounding) in 64 bits.

    A score is a sum of head_dim products of which the kernel rounds each at
    most 16 times by 2^-23 of the absolute products (fp32 sums; split fp32
    products drop 2^-22 of each): d = 16 * 2^-23 * scale * max_j sum_i |q_i k_ij|.
    A change of every score by at most d changes out by at most 2 d sum_j p_j |v_j|;
    sums of n terms add 4 sqrt(n) 2^-24 of the same, exp another 2^-20."""
    n, nq, nh, hd = q.shape
    nkv = (pk if pk is not None else sk).shape[1]
    gq = nh // nkv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    tol, dl = torch.zeros_like(out), torch.zeros_like(lse)
    for s in range(n):
        g = s // n_beam
        P = plen[g]
        parts = []
        if pk is not None:
            parts.append((pk[g, :, :P].double(), pv[g, :, :P].double()))
        if sk is not None and slen[s]:
            at = torch.arange(slen[s], device="cuda")
            src = torch.full_like(at, s)
            if slots is not None:
                own = slots[s, :slen[s]].long()
                src = torch.where((own >= 0) & (own < n_beam), own + g * n_beam, src)
            parts.append((sk[src, :, at].transpose(0, 1).double(), sv[src, :, at].transpose(0, 1).double()))
        k = torch.cat([a for a, _ in parts], 1) if parts else torch.zeros(nkv, 0, hd, device="cuda").double()
        v = torch.cat([b for _, b in parts], 1) if parts else k
        for t in range(nq):
            m = (P if pk is not None else 0) + max(0, (slen[s] if sk is not None else 0) - (nq - 1 - t))
            if m == 0:
                continue
            qq = q[s, t].double().reshape(nkv, gq, hd)
            x = torch.einsum("hgd,hjd->hgj", qq, k[:, :m]) * scale
            p = x.softmax(2)
            d = 16 * 2.0 ** -23 * scale * torch.einsum("hgd,hjd->hgj", qq.abs(), k[:, :m].abs()).amax(2)
            av = torch.einsum("hgj,hjd->hgd", p, v[:, :m].abs())
            out[s, t] = torch.einsum("hgj,hjd->hgd", p, v[:, :m]).reshape(nh, hd)
            lse[s, t] = x.logsumexp(2).flatten()
            tol[s, t] = (av * (2 * d[..., None] + 4 * math.sqrt(m) * 2.0 ** -24 + 2.0 ** -20)).reshape(nh, hd)
            dl[s, t] = (d + 2.0 ** -20).flatten() + 2.0 ** -22 * lse[s, t].abs()
            if q.dtype is not torch.float32:   # the probabilities' rounding: at most this share of sum p |v|
                tol[s, t] += ROUND[str(q.dtype)] * av.reshape(nh, hd)
    return out, lse, tol, dl



def attn_case(torch, dtype, G, W, nq, nh, nkv, hd, P, S, slots=True, plen=None, slen=None, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = dtype_of(torch, dtype)
    n = G * W

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dt)

    c = {"q": rand(n, nq, nh, hd) * 1.5, "pk": rand(G, nkv, P, hd) if P else None,
         "pv": rand(G, nkv, P, hd) if P else None, "sk": rand(n, nkv, S, hd) if S else None,
         "sv": rand(n, nkv, S, hd) if S else None, "slots": None, "n_beam": W}
    c["q"] = c["q"].to(dt)
    if slots and S:
        c["slots"] = torch.randint(0, W, (n, S), device="cuda", generator=gen, dtype=torch.int32)
    c["plen"] = plen if plen is not None else [max(0, P - 7 * g) for g in range(G)]
    c["slen"] = slen if slen is not None else [max(0, min(S, nq + (S - nq) * (i % 5) // 4)) for i in range(n)]
    return c


def attn_check(torch, beam, c, scale=0.0):
    q = c["q"]
    n, nq, nh, hd = q.shape
    W = c["n_beam"]
    some = c["pk"] if c["pk"] is not None else c["sk"]
    plan = beam.PrefixAttention(n_group=n // W, n_beam=W, n_query=nq, n_head=nh, n_head_kv=some.shape[1], head_dim=hd,
                                dtype=q.dtype, prefix_cap=0 if c["pk"] is None else c["pk"].shape[2],
                                suffix_cap=0 if c["sk"] is None else c["sk"].shape[2], scale=scale)
    pl = torch.tensor(c["plen"], dtype=torch.int32, device="cuda")
    sl = torch.tensor(c["slen"], dtype=torch.int32, device="cuda")
    out, lse = plan(q, c["pk"], c["pv"], c["sk"], c["sv"], prefix_len=pl, suffix_len=sl, slots=c["slots"])
    again, lse2 = plan(q, c["pk"], c["pv"], c["sk"], c["sv"], prefix_len=pl, suffix_len=sl, slots=c["slots"])
    assert torch.equal(out, again) and torch.equal(lse, lse2), "two calls differ"
    plen = [0 if c["pk"] is None else min(max(v, 0), c["pk"].shape[2]) for v in c["plen"]]
    slen = [0 if c["sk"] is None else min(max(v, 0), c["sk"].shape[2]) for v in c["slen"]]
    want, wl, tol, dl = attn_ref(torch, q, c["pk"], c["pv"], c["sk"], c["sv"], plen, slen, c["slots"], W,
                                 scale or 1 / math.sqrt(hd))
    tol = tol + ROUND[str(q.dtype)] * want.abs() + 2.0 ** -25   # the output's own rounding, and fp16's subnormal step
    assert torch.isfinite(out).all()
    worst = float(((out.double() - want).abs() / tol).max())
    assert worst <= 1, f"out is {worst:.2f} tolerances off"
    none = torch.isinf(wl)
    assert torch.equal(torch.isneginf(lse), none)
    assert (out[none] == 0).all()
    assert bool(((lse.double() - wl).abs()[~none] <= dl[~none]).all())
    return out, lse


SHAPES = [
    # G  W  nq  nh nkv  hd     P   S
    (1, 1, 1, 4, 2, 128, 1, 1),
    (1, 4, 1, 32, 8, 128, 200, 9),
    (2, 3, 2, 6, 6, 48, 65, 7),
    (1, 5, 3, 8, 1, 64, 129, 5),
    (1, 64, 1, 8, 1, 128, 300, 40),
    (3, 1, 1, 4, 4, 16, 63, 0),
    (1, 2, 1, 16, 2, 32, 0, 17),
    (1, 11, 4, 8, 8, 80, 513, 12),
    (2, 9, 7, 32, 4, 128, 1030, 71),
    (1, 3, 1, 28, 4, 96, 257, 130),
    (1, 16, 8, 16, 2, 128, 2111, 33),
    (1, 2, 40, 8, 2, 64, 190, 64),
    (5, 7, 1, 12, 4, 112, 64, 64),
    (1, 1, 1, 1, 1, 128, 20011, 3),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("slots", [False, True], ids=["own", "slots"])
def test_attention(torch, beam, dtype, shape, slots):
    attn_check(torch, beam, attn_case(torch, dtype, *shape, slots=slots, seed=len(shape) + sum(shape)))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_empty_and_short_lengths(torch, beam, dtype):
    """Groups without a prefix, sequences without a suffix, tokens that see nothing, lengths outside the capacity."""
    c = attn_case(torch, dtype, 3, 4, 3, 8, 2, 64, 70, 20, plen=[0, -5, 99], slen=[0, 1, 2, 3, 0, 20, 25, -1, 0, 1, 2, 19])
    attn_check(torch, beam, c)
    c = attn_case(torch, dtype, 2, 2, 1, 8, 8, 128, 130, 5, plen=[0, 0], slen=[0, 0, 0, 0])
    out, lse = attn_check(torch, beam, c)
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 12, 40])
def test_attention_ignores_what_lies_past_the_lengths(torch, beam, dtype, rows):
    c = attn_case(torch, dtype, 2, rows, 1, 4, 1, 128, 201, 37, plen=[130, 67], slen=[i % 33 for i in range(2 * rows)])
    clean = attn_check(torch, beam, c)
    bad = [math.nan, math.inf, -math.inf, torch.finfo(c["q"].dtype).min]
    for g in range(2):
        for k in ("pk", "pv"):
            for i, b in enumerate(bad):
                c[k][g, :, c["plen"][g] + i::4] = b
    used = torch.zeros(c["sk"].shape[0], c["sk"].shape[2], dtype=torch.bool, device="cuda")
    for s in range(2 * rows):
        for t in range(c["slen"][s]):
            used[s // rows * rows + c["slots"][s, t], t] = True
    for i, b in enumerate(bad):
        hit = ~used & (torch.arange(used.shape[1], device="cuda") % 4 == i)
        for k in ("sk", "sv"):
            c[k].masked_fill_(hit[:, None, :, None], b)
    c["slots"].masked_fill_(torch.arange(37, device="cuda") >= torch.tensor(c["slen"], device="cuda")[:, None], -12345)
    dirty = attn_check(torch, beam, c)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 3, 5, 8, 2, 128, 70, 40), (2, 2, 40, 8, 2, 64, 190, 64), (1, 2, 17, 6, 6, 48, 0, 33),
                                   (1, 2, 3, 4, 4, 16, 5, 19)], ids=lambda s: "x".join(map(str, s)))
def test_attention_keeps_values_from_tokens_that_do_not_see_them(torch, beam, dtype, shape):
    """Infinite and NaN V (and NaN K) of a new token reach that token and later ones, and no earlier one."""
    nq, nh, nkv, hd, n = shape[2], shape[3], shape[4], shape[5], shape[0] * shape[1]
    c = attn_case(torch, dtype, *shape, slots=False, slen=[shape[7] - 3 * i for i in range(n)])
    clean, lse = attn_check(torch, beam, c)
    plan = beam.PrefixAttention(n_group=shape[0], n_beam=shape[1], n_query=nq, n_head=nh, n_head_kv=nkv, head_dim=hd,
                                dtype=c["q"].dtype, prefix_cap=shape[6], suffix_cap=shape[7])
    kw = {"suffix_len": torch.tensor(c["slen"], dtype=torch.int32, device="cuda")}
    if shape[6]:
        kw["prefix_len"] = torch.tensor(c["plen"], dtype=torch.int32, device="cuda")
    sv, sk, from_t = c["sv"].clone(), c["sk"].clone(), nq // 2
    hit = torch.zeros(n, nq, nh, hd, dtype=torch.bool, device="cuda")
    for s in range(n):
        for i, b in enumerate((math.nan, math.inf, -math.inf)):
            t, h, d = min(nq - 1, from_t + i), i % nkv, (5 * i + 3 * s) % hd
            sv[s, h, c["slen"][s] - nq + t, d] = b
            hit[s, t:, h * (nh // nkv):(h + 1) * (nh // nkv), d] = True
    out, l = plan(c["q"], c["pk"], c["pv"], sk, sv, **kw)
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(l, lse)
    assert not torch.isfinite(out[hit]).any()
    for s in range(n):
        sk[s, :, c["slen"][s] - nq + from_t] = math.nan
    out, l = plan(c["q"], c["pk"], c["pv"], sk, c["sv"], **kw)
    assert torch.equal(out[:, :from_t], clean[:, :from_t]) and torch.equal(l[:, :from_t], lse[:, :from_t])
    assert torch.isnan(out[:, from_t:]).all()


def test_attention_slots_out_of_range_count_as_own(torch, beam):
    c = attn_case(torch, "f16", 2, 4, 1, 8, 2, 128, 33, 30)
    c["slots"][:, ::3] = -1
    c["slots"][:, 1::3] = 4
    c["slots"][0, 2] = 2 ** 31 - 1
    attn_check(torch, beam, c)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_on_views(torch, beam, dtype):
    """q inside rows of q|k|v, caches in [position][kv_head][dim] order, a prefix inside a larger cache."""
    c = attn_case(torch, dtype, 2, 3, 2, 8, 2, 128, 150, 40)
    n, nq, nh, hd = c["q"].shape
    rows = torch.zeros(n, nq, nh + 4, hd, dtype=c["q"].dtype, device="cuda")
    rows[:, :, 1:nh + 1] = c["q"]
    c["q"] = rows[:, :, 1:nh + 1]
    for k in ("pk", "pv"):
        big = torch.full((2, 400, 3, hd), math.nan, dtype=c[k].dtype, device="cuda")
        big[:, 11:161, 1:] = c[k].transpose(1, 2)
        c[k] = big[:, 11:161, 1:].transpose(1, 2)
    for k in ("sk", "sv"):
        c[k] = c[k].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((n, 77), -1, dtype=torch.int32, device="cuda")
    wide[:, :40] = c["slots"]
    c["slots"] = wide[:, :40]
    attn_check(torch, beam, c)


def test_attention_offsets_past_32_bits(torch, beam):
    """KV heads more than 2^32 elements apart, in one allocation of about 13 GB."""
    far = (1 << 32) + 4096
    big = torch.zeros(far + (1 << 31), dtype=torch.bfloat16, device="cuda")
    c = attn_case(torch, "bf16", 1, 5, 1, 8, 2, 128, 100, 20)
    for i, k in enumerate(("pk", "pv", "sk", "sv")):
        x = c[k]
        st = (x.shape[2] * 128, far, 128, 1)
        v = big[i << 20:].as_strided(x.shape, st)
        v.copy_(x)
        c[k] = v
    attn_check(torch, beam, c)


def test_attention_scale_and_large_scores(torch, beam):
    """Scores of several hundred: exp of the difference from the maximum, not of the score."""
    c = attn_case(torch, "f32", 1, 4, 1, 8, 2, 64, 300, 10)
    c["q"] *= 40
    attn_check(torch, beam, c, scale=0.5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_rising_scores(torch, beam, dtype):
    """Every tile raises the running maximum: the earlier sums are scaled down each time."""
    c = attn_case(torch, dtype, 1, 8, 1, 16, 2, 128, 900, 8)
    c["q"].fill_(0)
    c["q"][..., 0] = 1
    c["pk"][..., 0] = torch.linspace(0, 100, 900, device="cuda").to(c["pk"].dtype)[None, None]
    attn_check(torch, beam, c, scale=1.0)


def test_attention_on_another_stream(torch, beam):
    c = attn_case(torch, "f16", 1, 6, 1, 8, 2, 128, 3000, 30)
    plan = beam.PrefixAttention(n_group=1, n_beam=6, n_head=8, n_head_kv=2, head_dim=128, dtype=torch.float16,
                                prefix_cap=3000, suffix_cap=30)
    args = [c[k] for k in ("q", "pk", "pv", "sk", "sv")]
    want, _ = plan(*args, slots=c["slots"])
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(plan(*args, slots=c["slots"])[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_attention_in_a_graph(torch, beam):
    c = attn_case(torch, "bf16", 1, 6, 1, 8, 2, 128, 700, 30)
    plan = beam.PrefixAttention(n_group=1, n_beam=6, n_head=8, n_head_kv=2, head_dim=128, dtype=torch.bfloat16,
                                prefix_cap=700, suffix_cap=30)
    args = [c[k] for k in ("q", "pk", "pv", "sk", "sv")]
    out, lse = plan(*args, slots=c["slots"])
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        plan(*args, slots=c["slots"], out=out, lse=lse)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        plan(*args, slots=c["slots"], out=out, lse=lse)
    c["q"].copy_(c["q"].flip(0))
    want, _ = plan(*args, slots=c["slots"])
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# --- selection ----------------------------------------------------------------------
def select_ref(x, c, K):
    """(scores, parent, token) in 64 bits; x [G][W][V], c [G][W] as numpy arrays."""
    G, W, V = x.shape
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        top = x.max(2, keepdims=True)
        lse = top + np.log(np.exp(x - top).sum(2, keepdims=True))
        s = c.astype(np.float64)[:, :, None] + (x - lse)
    s[~(np.isfinite(lse[..., 0]) & np.isfinite(c))] = -np.inf
    s = s.reshape(G, W * V)
    at = np.argsort(-s, axis=1, kind="stable")[:, :K]
    return s, at


def select_decided(x, s, at, V, gap=3e-5):
    """Whether no two neighbours of the best are nearer than fp32 scores tell apart (equal logits of one row tie exactly)."""
    for g in range(s.shape[0]):
        order = np.argsort(-s[g], kind="stable")[:at.shape[1] + 1]
        for a, b in zip(order[:-1], order[1:]):
            same = a // V == b // V and x[g].reshape(-1)[a] == x[g].reshape(-1)[b]
            if not same and np.isfinite(s[g][a]) and s[g][a] - s[g][b] < gap:
                return False
    return True


def select_check(torch, beam, x, c, K, dtype="f32", stride=None):
    """x, c: numpy; the logits are rounded to the type first."""
    G, W, V = x.shape
    t = torch.from_numpy(x.astype(np.float32)).to(dtype_of(torch, dtype)).cuda()
    xr = t.float().cpu().numpy()
    s, at = select_ref(xr, c, K)
    assert select_decided(xr, s, at, V), "the test's own input leaves the order to rounding"
    if stride:
        wide = torch.full((G, W, stride), math.nan, dtype=t.dtype, device="cuda")
        wide[:, :, :V] = t
        t = wide[:, :, :V]
    plan = beam.BeamSelect(n_group=G, n_beam=W, n_vocab=V, n_select=K, dtype=t.dtype)
    cc = torch.from_numpy(c.astype(np.float32)).cuda()
    sc, par, tok = plan(t, cc)
    flat = par.cpu().numpy().astype(np.int64) * V + tok.cpu().numpy()
    assert np.array_equal(flat, at)
    want = np.take_along_axis(s, at, 1)
    got = sc.cpu().numpy()
    assert np.array_equal(np.isneginf(want), np.isneginf(got))
    fin = np.isfinite(want)
    # x - top, its difference from the log-sum and the sum with the score round once each; the log-sum of V terms 4 more
    mag = np.abs(xr[np.isfinite(xr)]).max(initial=1) + np.abs(c[np.isfinite(c)]).max(initial=1) + math.log(V) + 1
    assert np.abs(got[fin] - want[fin]).max(initial=0) <= 16 * 2.0 ** -24 * mag
    return sc, par, tok


def select_inputs(G, W, V, seed, grid=1 / 64):
    """Logits on a grid (many equal ones) and scores that keep the rows' offsets apart."""
    r = np.random.default_rng(seed)
    x = np.round(r.normal(0, 2, (G, W, V)) / grid) * grid
    return x, -8 * r.random((G, W)).astype(np.float32)


def decided(make, K, dtype="f32"):
    import torch as T
    for seed in range(50):
        x, c = make(seed)
        xr = T.from_numpy(x.astype(np.float32)).to(dtype_of(T, dtype)).float().numpy()
        s, at = select_ref(xr, c, K)
        if select_decided(xr, s, at, x.shape[2]):
            return x, c
    raise AssertionError("no decided input")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,W,V,K", [
    (1, 1, 1, 1), (1, 1, 7, 7), (1, 4, 33, 8), (2, 3, 1000, 6), (1, 4, 32000, 8), (3, 8, 5003, 16), (1, 64, 2048, 128),
    (1, 32, 4099, 64), (5, 2, 128256, 4), (1, 1, 128256, 128), (40, 4, 1001, 8), (1, 5, 50257, 1), (1, 2, 3, 6),
])
def test_select(torch, beam, dtype, G, W, V, K):
    x, c = decided(lambda s: select_inputs(G, W, V, 1000 * s + V), K, dtype)
    select_check(torch, beam, x, c, K, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("stride", [1001, 1004, 1024])
def test_select_strided_rows(torch, beam, dtype, stride):
    x, c = decided(lambda s: select_inputs(2, 3, 1001, s), 6, dtype)
    select_check(torch, beam, x, c, 6, dtype, stride=stride)


def test_select_first_step_and_barred_tokens(torch, beam):
    """Only beam 0 is alive; nine tokens in ten are barred; then fewer candidates than are selected."""
    def make(s):
        x, c = select_inputs(2, 4, 4000, s)
        x[np.random.default_rng(s).random(x.shape) < 0.9] = -np.inf
        c[:, 1:] = -np.inf
        return x, c
    x, c = decided(make, 8)
    select_check(torch, beam, x, c, 8)
    x[0, 0] = -np.inf
    x[0, 0, [7, 3999, 12]] = [1, 2, 3]     # three candidates for eight places: the rest by index
    select_check(torch, beam, x, c, 8)
    x[0, 0, 0] = 5                         # one of them at index 0
    select_check(torch, beam, x, c, 8)


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_select_rows_without_candidates(torch, beam, what):
    def make(s):
        x, c = select_inputs(2, 3, 3000, s)
        x[0, 1, 1234] = what
        if what == -math.inf:
            x[0, 1] = what
        c[1, 0] = what
        return x, c
    x, c = decided(make, 6)
    select_check(torch, beam, x, c, 6)
    x[:] = what                            # nothing anywhere: the lowest indexes, at -inf
    _, par, tok = select_check(torch, beam, x, c, 6)
    assert (par == 0).all() and torch.equal(tok[0].cpu(), torch.arange(6, dtype=torch.int32))


@pytest.mark.parametrize("order", ["rising", "falling", "equal", "block"])
@pytest.mark.parametrize("V", [9000, 128256])
def test_select_ordered_logits(torch, beam, order, V):
    """Orders that put the best entries into one thread's, one warp's or every thread's share."""
    r = np.arange(V) / 64.0 / (V / 1024.0)
    row = {"rising": r, "falling": r[::-1], "equal": np.zeros(V), "block": np.where(np.arange(V) // 64 == 70, 8 + np.arange(V) % 64 / 8, -r)}[order]
    x = np.stack([row, row, np.roll(row, 17)])[None]
    c = np.array([[-1.0, -1.5, -9.0]], np.float32)
    def make(s):
        return x, c - np.float32(s) * np.array([[0.0, 0.0137, 0.0071]], np.float32)
    for K in (1, 16, 128):
        select_check(torch, beam, *decided(make, K), K)


def test_select_equal_rows_take_the_lowest_index(torch, beam):
    """Beams with the same logits and score tie exactly, across rows too."""
    row = np.round(np.random.default_rng(3).normal(0, 2, 6000) * 4) / 4
    x = np.stack([row, row, row])[None].astype(np.float32)
    plan = beam.BeamSelect(n_group=1, n_beam=3, n_vocab=6000, n_select=64)
    _, par, tok = plan(torch.from_numpy(x).cuda(), torch.full((1, 3), -2.0, device="cuda"))
    key = sorted(range(18000), key=lambda i: (-x.reshape(-1)[i], i))[:64]
    assert (par[0].cpu().numpy().astype(int) * 6000 + tok[0].cpu().numpy()).tolist() == key


# --- reordering -----------------------------------------------------------------------
def reorder_ref(src, par, n_beam):
    import torch
    idx = []
    for g, row in enumerate(par):
        idx += [g * n_beam + (p if 0 <= p < n_beam else b) for b, p in enumerate(row)]
    return src[:, torch.tensor(idx)]


@pytest.mark.parametrize("shape,G,W", [
    ((1, 4, 131), 1, 4), ((3, 6, 5, 7), 2, 3), ((2, 8, 4, 16, 48), 1, 8), ((1, 64, 9, 128), 1, 64), ((5, 34, 2, 3, 16), 2, 17),
    ((1, 1, 1), 1, 1), ((2, 60, 33), 4, 15),
])
@pytest.mark.parametrize("kind", ["int32", "float16", "uint8", "float32"])
@pytest.mark.parametrize("place", ["in", "out"])
def test_reorder(torch, beam, shape, G, W, kind, place):
    gen = torch.Generator().manual_seed(sum(shape))
    x = torch.randint(0, 200, shape, generator=gen).to(getattr(torch, kind)).cuda()
    for trial in range(4):
        if trial == 0:      # a cycle through all beams
            par = [[(b + 1) % W for b in range(W)] for _ in range(G)]
        elif trial == 1:    # all from one
            par = [[W - 1] * W for _ in range(G)]
        else:
            par = torch.randint(-1, W + 1, (G, W), generator=gen).tolist()
        want = reorder_ref(x.cpu(), par, W)
        p = torch.tensor(par, dtype=torch.int32, device="cuda")
        if place == "in":
            y = x.clone()
            assert beam.reorder(y, p) is y
        else:
            y = torch.zeros_like(x)
            beam.reorder(x, p, y)
        assert torch.equal(y.cpu(), want)


def test_reorder_views_leave_the_rest(torch, beam):
    x = torch.randn(6, 8, 3, 40, 64, device="cuda")
    y = x.clone()
    p = torch.tensor([[3, 3, 0, 1], [0, 0, 0, 2]], dtype=torch.int32, device="cuda")
    beam.reorder(y[:, :, :, 5:33], p)
    want = x.clone()
    want[:, :, :, 5:33] = reorder_ref(x.cpu(), p.tolist(), 4)[:, :, :, 5:33].cuda()
    assert torch.equal(y, want)
    z = torch.zeros(6, 8, 3, 28, 64, device="cuda")
    beam.reorder(x[:, :, :, 5:33], p, z)
    assert torch.equal(z, want[:, :, :, 5:33])


def test_reorder_past_32_bits(torch, beam):
    """Slots more than 4 GB apart."""
    big = torch.zeros(3, (1 << 32) + 4096, dtype=torch.uint8, device="cuda")
    v = big[:, -4096:][None]
    v.copy_(torch.randint(0, 255, v.shape, device="cuda", dtype=torch.uint8))
    want = reorder_ref(v.cpu(), [[2, 0, 1]], 3)
    beam.reorder(v, torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda"))
    assert torch.equal(v.cpu(), want)


# --- refusals ---------------------------------------------------------------------------
def test_refusals(torch, beam):
    from fwb.model import FwbError
    ok = dict(n_group=1, n_beam=2, n_head=4, n_head_kv=2, head_dim=64, dtype=torch.float16, prefix_cap=10, suffix_cap=4)
    for bad in (dict(head_dim=40), dict(head_dim=256), dict(n_head=5), dict(n_beam=0), dict(n_query=0)):
        with pytest.raises(FwbError):
            beam.PrefixAttention(**{**ok, **bad})
    with pytest.raises(ValueError):
        beam.PrefixAttention(**{**ok, "dtype": torch.float64})
    plan = beam.PrefixAttention(**ok)
    q = torch.zeros(2, 1, 4, 64, dtype=torch.float16, device="cuda")
    pk = torch.zeros(1, 2, 10, 64, dtype=torch.float16, device="cuda")
    sk = torch.zeros(2, 2, 4, 64, dtype=torch.float16, device="cuda")
    plan(q, pk, pk, sk, sk)
    with pytest.raises(ValueError):
        plan(q.float(), pk, pk, sk, sk)
    with pytest.raises(ValueError):
        plan(q, pk[:, :, :9], pk, sk, sk)
    with pytest.raises(ValueError):
        plan(q, pk, pk, sk, sk.cpu())
    with pytest.raises(ValueError):
        plan(q, pk, pk, sk, sk, suffix_len=torch.zeros(2, dtype=torch.int64, device="cuda"))
    odd = torch.zeros(1, 2, 10, 65, dtype=torch.float16, device="cuda")[..., :64]
    with pytest.raises(FwbError):
        plan(q, odd, odd, sk, sk)
    for bad in (dict(n_select=129), dict(n_beam=65), dict(n_select=0), dict(n_vocab=2, n_select=9)):
        with pytest.raises(FwbError):
            beam.BeamSelect(**{**dict(n_group=1, n_beam=4, n_vocab=100, n_select=8), **bad})
    x = torch.zeros(1, 4, 8, device="cuda")
    with pytest.raises(ValueError):
        beam.reorder(x, torch.zeros(1, 3, dtype=torch.int32, device="cuda"))
    with pytest.raises(FwbError):
        beam.reorder(x[:, :3], torch.zeros(1, 3, dtype=torch.int32, device="cuda"), x[:, 1:])
    with pytest.raises(FwbError):
        beam.reorder(torch.zeros(1, 65, 4, device="cuda"), torch.zeros(1, 65, dtype=torch.int32, device="cuda"))


# --- many rows over long prefixes: the tcgen05 kernel -------------------------------------
# n_group * n_head_kv * prefix_cap * (rows / 64 - rows / 128, each rounded up) is at least
# 36000 in all of these, which is where that kernel takes the prefixes over.
LONG = [
    # G  W   nq nh nkv  hd    P    S
    (1, 40, 2, 8, 4, 128, 9001, 6),
    (1, 9, 7, 32, 4, 128, 2611, 71),
    (2, 33, 1, 16, 4, 64, 4609, 5),
    (1, 20, 4, 8, 8, 96, 4513, 12),
    (1, 64, 1, 8, 1, 48, 9100, 3),
    (3, 128, 1, 2, 2, 16, 6144, 0),
    (1, 300, 1, 4, 2, 112, 4096, 1),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", LONG, ids=lambda s: "x".join(map(str, s)))
def test_attention_many_rows(torch, beam, dtype, shape):
    attn_check(torch, beam, attn_case(torch, dtype, *shape, seed=sum(shape)))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_many_rows_short_lengths(torch, beam, dtype):
    """Lengths of a tile's fractions in a large cache, of nothing, and past it; poison behind them."""
    for plen in ([0, 1, 15], [127, 128, 129], [16, 0, 20000], [-3, 4100, 500]):
        c = attn_case(torch, dtype, 3, 24, 1, 32, 8, 128, 4100, 9, plen=plen, slen=[i % 10 for i in range(72)])
        clean = attn_check(torch, beam, c)
        for g in range(3):
            for k in ("pk", "pv"):
                for i, b in enumerate((math.nan, math.inf, -math.inf)):
                    c[k][g, :, max(0, plen[g]) + i::3] = b
        dirty = attn_check(torch, beam, c)
        assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_many_rows_rising_scores(torch, beam, dtype):
    """Tiles that raise the references again and again, by little and by much, for some rows only."""
    c = attn_case(torch, dtype, 1, 48, 1, 16, 4, 128, 9500, 8)
    c["q"].fill_(0)
    c["q"][..., 0] = torch.linspace(0, 1, 48, device="cuda")[:, None, None].to(c["q"].dtype)
    c["q"][..., 1] = 0.25
    at = torch.arange(9500, device="cuda")
    c["pk"][..., 0] = (at / 95.0).to(c["pk"].dtype)
    c["pk"][..., 1] = (((at * 7919) % 9500) / 40.0).to(c["pk"].dtype)
    attn_check(torch, beam, c, scale=1.0)
    c["pk"][..., 0] = (-at / 50.0).to(c["pk"].dtype)
    attn_check(torch, beam, c, scale=1.0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("W,P", [(3, 150), (32, 2400)])
def test_attention_broadcast_caches(torch, beam, dtype, W, P):
    """One prefix for all groups and one KV head for all (strides of 0), one suffix for all sequences."""
    c = attn_case(torch, dtype, 2, W, 1, 32, 8, 128, P, 20, slots=False)
    for k in ("pk", "pv"):
        c[k] = c[k][:1, :1].expand(2, 8, -1, -1)
    for k in ("sk", "sv"):
        c[k] = c[k][:1].expand(2 * W, -1, -1, -1)
    c["plen"] = [P, P - 1]
    attn_check(torch, beam, c)


def test_attention_status(torch, beam):
    beam.check_status()
