"""GPU: sampling of rows against its definition in 64 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(built):
    return pytest.importorskip("torch")


@pytest.fixture(scope="module")
def sample_rows(torch):
    from fwb.sampling import sample_rows
    torch.zeros(1, device="cuda")
    return sample_rows


def definition(torch, x, u, temp, k, p, low):
    """(token, logprob, clearance, near) of one row: clearance is how near a limit comes to a border, relative to the mass;
    near the tokens that either side of the borders in reach could give."""
    x = x.double().cpu()
    if bool((x == math.inf).any()) or bool(torch.isnan(x).any()) or not bool((x > -math.inf).any()) or temp != temp or u != u:
        return -1, -math.inf, 1.0, ()
    if temp <= 0:
        return int(x.argmax()), 0.0, 1.0, ()
    s, order = torch.sort(x, descending=True, stable=True)
    y = (s - s[0]) / temp
    if math.isinf(temp):
        y = torch.where(s == -math.inf, -math.inf, 0.0)
    w = torch.exp(y)
    n = int((w > 2.0 ** -64).sum())
    w, clear = w[:n], 1.0
    if 0 < k < n:
        w = w[:k]
    cum = cum_all = torch.cumsum(w, 0)
    stay, total = len(w), float(cum[-1])
    reach = 2.0 ** -20
    if p < 1:
        before = cum - w
        edge = (before[1:] - p * total).abs() < 2.0 ** -20 * total
        reach += float(w[1:][edge].sum() + w[:-1][edge].sum()) / (p * total) if p > 0 else 0.0
        stay = max(1, int((before < p * total).sum()))
        clear = min(clear, float((before[1:] - p * total).abs().min()) / total if len(w) > 1 else 1.0)
    if low > 0:
        stay = max(1, min(stay, int((w >= low).sum())))
        clear = min(clear, float((w - low).abs().min()) / low)
        reach += float(w[(w - low).abs() < 2.0 ** -20 * low].sum()) / float(cum[stay - 1])
    cum = cum[:stay]
    target = u * float(cum[-1])
    wide, most = reach * float(cum[-1]), min(stay + 3, len(w))
    near = order[:most][(cum_all[:most] >= target - wide) & (cum_all[:most] - w[:most] <= target + wide)]
    at = min(int((cum <= u * cum[-1]).sum()), stay - 1)
    clear = min(clear, float((cum[:-1] - u * cum[-1]).abs().min()) / float(cum[-1]) if stay > 1 else 1.0)
    return int(order[at]), math.log(float(w[at]) / float(cum[-1])), clear, set(near.tolist())


def check(torch, sample_rows, x, u, temp=None, k=None, p=None, low=None):
    """Rows whose limits come nearer to a border than 2^-20 of the mass (four of the weights' steps) may fall on either side
    of it, and nowhere else."""
    n = x.shape[0]

    def given(v, dtype):
        return None if v is None else torch.tensor(v, dtype=dtype, device="cuda")
    f32 = torch.float32
    t = given(temp, f32), given(k, torch.int32), given(p, f32), given(low, f32)
    token, logprob = sample_rows(x, given(u, f32), temperature=t[0], top_k=t[1], top_p=t[2], min_p=t[3])
    us, ts, ks, ps, ls = (d.tolist() if d is not None else [e] * n for d, e in zip((given(u, f32), *t), (0, 1.0, 0, 1.0, 0.0)))
    for i in range(n):
        want, lp, clear, near = definition(torch, x[i], us[i], ts[i], ks[i], ps[i], ls[i])
        if clear < 2.0 ** -20:
            assert int(token[i]) in near, (i, int(token[i]), want, clear)
            continue
        assert int(token[i]) == want, (i, int(token[i]), want, clear)
        got = float(logprob[i])
        assert got == lp or abs(got - lp) <= 2.0 ** -20 + abs(lp) * 2.0 ** -22, (i, got, lp)
    return token, logprob


def logits(torch, seed, n, V, dtype=None, sd=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, V, device="cuda", generator=gen) * sd
    x.masked_fill_(torch.rand(n, V, device="cuda", generator=gen) < 0.02, -math.inf)
    x[:, 0] = 1.0
    return x.to(dtype or torch.float32)


def draws(torch, seed, n):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed)).tolist()


SETTINGS = {
    "plain": dict(), "temperature": dict(temp=[0.3, 0.7, 1.0, 1.5]), "top_k": dict(k=[1, 2, 50, 300]), "top_p": dict(p=[0.1, 0.5, 0.9, 0.99]),
    "min_p": dict(low=[0.5, 0.1, 0.01, 0.001]), "all": dict(temp=[0.6, 0.8, 1.0, 1.2], k=[5, 40, 100, 0], p=[0.95, 0.9, 1.0, 0.7], low=[0.0, 0.05, 0.02, 0.1]),
    "mixed": dict(temp=[0.0, 1.0, 0.9, 1.1], k=[0, 0, 20, -3], p=[1.0, 1.0, 1.5, 0.8], low=[0.0, 0.0, 0.0, 0.02]),
    "wide": dict(temp=[3.0, 5.0, 8.0, 20.0], k=[0, 5000, 0, 700], p=[0.9, 1.0, 0.5, 0.95], low=[0.0, 0.0, 0.2, 0.01]),
    "wide k": dict(temp=[4.0] * 4, k=[2500, 3000, 9000, 20000]), "wide min": dict(temp=[6.0] * 4, low=[0.3, 0.1, 0.5, 1e-9])}


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("V", [1, 7, 100, 1000, 4099, 32000, 128256])
@pytest.mark.parametrize("name", list(SETTINGS))
def test_rows(torch, sample_rows, dtype, V, name):
    n = 12
    st = {k: (v * 3)[:n] for k, v in SETTINGS[name].items()}
    check(torch, sample_rows, logits(torch, V, n, V, getattr(torch, dtype)), draws(torch, V, n), **st)


@pytest.mark.parametrize("V", [262144, 200001])
def test_largest_vocabulary(torch, sample_rows, V):
    check(torch, sample_rows, logits(torch, 1, 3, V), draws(torch, 2, 3), temp=[1.0, 2.0, 10.0], p=[0.9, 1.0, 0.8])


def test_many_rows(torch, sample_rows):
    n = 700
    check(torch, sample_rows, logits(torch, 3, n, 500), draws(torch, 4, n), temp=[0.5 + i % 7 * 0.2 for i in range(n)],
          k=[i % 50 for i in range(n)], p=[0.7 + 0.003 * (i % 100) for i in range(n)])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [3000, 128256])
def test_equal_logits(torch, sample_rows, dtype, V):
    """All weights alike: the ranking is the index, and limits count."""
    x = torch.full((8, V), -3.25, device="cuda", dtype=getattr(torch, dtype))
    u = [0.0, 0.25001, 0.5, 0.75, 0.9999, 0.31, 0.62, 1.0 - 2.0 ** -24]
    k, p, low = [0, 0, 2600, 2999, 0, 0, 10, 0], [1.0, 1.0, 1.0, 0.5, 0.9001, 1.0, 1.0, 1.0], [0.0, 0.0, 0.0, 0.0, 0.0, 1.0, 0.5, 0.0]
    t = lambda v, d: torch.tensor(v, dtype=d, device="cuda")  # noqa: E731
    u32 = t(u, torch.float32)
    token, logprob = sample_rows(x, u32, top_k=t(k, torch.int32), top_p=t(p, torch.float32), min_p=t(low, torch.float32))
    for i in range(8):
        n = V if k[i] == 0 else min(k[i], V)
        p32 = float(t(p, torch.float32)[i])
        if p32 < 1:
            n = math.ceil(p32 * n)
        want = min(math.floor(float(u32[i]) * n), n - 1)
        assert int(token[i]) == want, (i, n)
        assert abs(float(logprob[i]) + math.log(n)) <= 2.0 ** -20


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_two_levels_of_equal_logits(torch, sample_rows, dtype):
    """Thousands of ties above thousands of others, scattered; limits fall in either."""
    V, n = 50000, 10
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.where(torch.rand(n, V, device="cuda", generator=gen) < 0.3, 2.0, 1.5).to(getattr(torch, dtype))
    check(torch, sample_rows, x, draws(torch, 9, n), k=[0, 0, 3000, 14000, 20000, 0, 0, 30000, 1, 49999],
          p=[1.0, 0.3, 1.0, 1.0, 0.9, 0.6, 0.99, 1.0, 1.0, 0.5], low=[0.0, 0.0, 0.0, 0.0, 0.0, 0.7, 0.5, 0.0, 0.0, 0.0])


def test_near_ties(torch, sample_rows):
    """Logits one step of fp32 apart, more of them in a bin than a list holds."""
    V = 40000
    base = torch.tensor([8.0], device="cuda")
    steps = (torch.randperm(V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) % 3000).float() * 2.0 ** -20
    x = (base + steps)[None].repeat(6, 1)
    check(torch, sample_rows, x, [0.1, 0.35, 0.62, 0.88, 0.5, 0.999], k=[0, 0, 5000, 25000, 0, 0], p=[1.0, 0.5, 1.0, 1.0, 0.9, 1.0])


def test_limits_of_the_settings(torch, sample_rows):
    V = 1000
    x = logits(torch, 8, 12, V)
    x[:, 5] = 50.0                                                 # nearly all the mass
    x[6:, 5] = 9.0
    u = [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, 0.4, 0.3, 0.6, 0.2, 0.9, 0.1, 0.7]
    check(torch, sample_rows, x, u, temp=[1.0, 1.0, 1.0, 1e-30, 1e-4, math.inf, math.inf, 1e30, 1.0, 1.0, 1.0, -2.0],
          k=[5, 0, 7, 0, 0, 0, 10, 0, V, 10 * V, 2 ** 31 - 1, 0], p=[1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 0.0, -1.0, 2.0, 1.0],
          low=[0.0] * 6 + [0.0, 0.0, 0.0, 0.0, 2.0, 1.0])


def test_dead_rows(torch, sample_rows):
    x = logits(torch, 8, 8, 300)
    x[0, 17] = math.nan
    x[1, 299] = math.inf
    x[2] = -math.inf
    x[4] = -math.inf
    x[4, 123] = -5.0                                               # one token left
    x[6, 0] = math.nan                                             # greedy, but dead
    token, logprob = check(torch, sample_rows, x, [0.5, 0.5, 0.5, math.nan, 0.5, 0.5, 0.5, 0.5],
                           temp=[1.0, 1.0, 1.0, 1.0, 1.0, math.nan, 0.0, 0.0])
    assert token[[0, 1, 2, 3, 5, 6]].tolist() == [-1] * 6 and bool((logprob[[0, 1, 2, 3, 5, 6]] == -math.inf).all())
    assert int(token[4]) == 123 and float(logprob[4]) == 0.0 and float(logprob[7]) == 0.0


def test_lowest_values_bar(torch, sample_rows):
    """Tokens masked with the type's lowest value instead of -inf."""
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = torch.full((4, 5000), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        x[:, [7, 99, 4321]] = torch.tensor([1.0, 2.0, 1.5], dtype=dtype, device="cuda")
        token, _ = check(torch, sample_rows, x, [0.05, 0.3, 0.6, 0.999], k=[0, 3, 100, 0])
        assert set(token.tolist()) <= {7, 99, 4321}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_of_any_stride(torch, sample_rows, dtype):
    dt = getattr(torch, dtype)
    whole = logits(torch, 5, 6, 3001, dt)
    for view in (whole[:, 1:2000], whole[::2, :2999], whole[:, 3:]):
        n = view.shape[0]
        got = check(torch, sample_rows, view, draws(torch, 6, n), p=[0.9] * n)
        same = sample_rows(view.contiguous(), torch.tensor(draws(torch, 6, n), device="cuda"), top_p=torch.full((n,), 0.9, device="cuda"))
        assert all(torch.equal(a, b) for a, b in zip(got, same))


def test_repeats_graphs_and_streams(torch, sample_rows):
    x = logits(torch, 5, 40, 32000)
    u = torch.tensor(draws(torch, 6, 40), device="cuda")
    temp = torch.full((40,), 1.3, device="cuda")
    want = sample_rows(x, u, temperature=temp)
    outs = [tuple(torch.empty_like(t) for t in want) for _ in range(3)]
    graphs = []
    for o in outs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            sample_rows(x, u, temperature=temp, token=o[0], logprob=o[1])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o[0].zero_(), o[1].zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            sample_rows(x, u, temperature=temp, token=outs[2][0], logprob=outs[2][1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


@pytest.mark.parametrize("setting", [dict(), dict(k=7), dict(k=300), dict(p=0.99999), dict(low=1e-6), dict(low=1e-12), dict(k=300, p=0.9999, low=1e-9)],
                         ids=lambda s: "-".join(s) + str(s.get("k", s.get("low", ""))) if s else "none")
@pytest.mark.parametrize("V", [1000, 32003])
def test_one_token_holds_nearly_all(torch, sample_rows, setting, V):
    """The first token's log keeps its digits where the others hold up to half and down to 2^-50 of the mass between them."""
    gaps = [7.0, 9.0, 14.0, 18.0, 21.5, 24.0, 27.0, 31.0, 36.0]
    n = len(gaps)
    # multiples of 2^-8: the differences of logits are exact in 32 bits
    x = torch.round(logits(torch, 8, n, V).clamp(-8, 5) * 256) / 256
    x[:, V // 3] = 5 + torch.tensor(gaps, device="cuda")
    full = {name: [setting.get(name, d)] * n for name, d in (("k", 0), ("p", 1.0), ("low", 0.0))}
    token, logprob = sample_rows(x, torch.full((n,), 0.25, device="cuda"), top_k=torch.tensor(full["k"], dtype=torch.int32, device="cuda"),
                                 top_p=torch.tensor(full["p"], device="cuda"), min_p=torch.tensor(full["low"], device="cuda"))
    for i in range(n):
        p, low = (float(torch.tensor(full[k][i])) for k in ("p", "low"))
        s = torch.sort(x[i].double(), descending=True)[0]
        w = torch.exp(s - s[0])
        w = w[w > 2.0 ** -64]
        w = w[:full["k"][i] or len(w)]
        before = torch.cumsum(w, 0) - w
        if p < 1:
            border = (before - p * float(w.sum())).abs()
            w = w[(before < p * float(w.sum())) | (before == 0)]
            if float(border[1:].min()) < 2.0 ** -20:   # the cut may be off by an entry
                continue
        w = w[w >= low]
        rest = float(w[1:].sum())
        want = -math.log1p(rest)
        # Each other weight: 2^-22 of the exponential, 2^-23 of its step in a bin; what lies below 2^-32 up to
        # V / 4096 in a row in 32 bits, 8 * 2^-24; what a filter leaves of it 2^-20.  Together below 2^-19.  The mass in
        # 64 bits, its quotient and its log: a step of 2^-52 each at most.
        assert int(token[i]) == V // 3
        assert abs(float(logprob[i]) - want) <= abs(want) * 2.0 ** -19 + 3 * 2.0 ** -52, (i, float(logprob[i]), want)


@pytest.mark.parametrize("setting", [dict(), dict(k=3), dict(k=4), dict(k=40), dict(p=0.5), dict(low=2.0 ** -32), dict(low=2.0 ** -33)], ids=str)
@pytest.mark.parametrize("u", [0.0, 0.5, 1.0])
def test_weights_at_a_step_of_32_octaves(torch, sample_rows, setting, u):
    """Logits whose weights are 2^-32 and its neighbours, to the last bit or nearly."""
    x = torch.full((1, 900), -math.inf, device="cuda")
    x[0, 10], x[0, 500] = 0.0, -1.0
    x[0, 20], x[0, 600], x[0, 30], x[0, 800] = -32.0, -32.0, -32.0 + 2.0 ** -18, -32.0 - 2.0 ** -18
    x[0, 700], x[0, 40] = -63.0, -40.0
    check(torch, sample_rows, x, [u], temp=[math.log2(math.e)], **{name: [v] for name, v in setting.items()})


def test_refusals(torch, sample_rows):
    from fwb.model import FwbError
    x, u = logits(torch, 1, 3, 100), torch.zeros(3, device="cuda")
    for bad in (dict(logits=None), dict(logits=x[0]), dict(logits=x.double()), dict(logits=x.cpu()), dict(logits=x.t()), dict(uniform=None),
                dict(uniform=u[:2]), dict(uniform=u.double()), dict(temperature=u[:1]), dict(top_k=u), dict(top_p=u.half()),
                dict(min_p=u.cpu()), dict(token=u), dict(logprob=u.int())):
        with pytest.raises(ValueError):
            sample_rows(**{**dict(logits=x, uniform=u), **bad})
    with pytest.raises(FwbError):
        sample_rows(torch.zeros(1, 262145, device="cuda"), u[:1])
