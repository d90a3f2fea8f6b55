"""GPU: the beam-search operators (fwb.beam) on extreme values: logits far below
zero and masks of the type's lowest value, against the definition in 64 bits."""
import math

import numpy as np
import pytest

from test_gpu_beam import (ROUND, attn_case, attn_ref, beam, dtype_of, select_decided, select_inputs,  # noqa: F401
                           torch)

pytestmark = pytest.mark.gpu


# --- selection ----------------------------------------------------------------------
def stable_scores(x, c):
    """c + ((x - max) - log sum exp(x - max)) in 64 bits, flat per group: logsumexp by itself may be too large to hold the logarithm."""
    x = x.astype(np.float64)
    d = x - x.max(2, keepdims=True)
    s = (d - np.log(np.exp(d).sum(2, keepdims=True))) + c.astype(np.float64)[:, :, None]
    return s.reshape(x.shape[0], -1)


def check_scores(torch, beam, x, c, K, dtype):
    """The selection of x (values of the type) and its scores.

    A score's logarithm of a sum of V terms rounds 16 times by 2^-24 of 1 + log V, the score's own sum once of its size."""
    G, W, V = x.shape
    s = stable_scores(x, c)
    at = np.argsort(-s, axis=1, kind="stable")[:, :K]
    plan = beam.BeamSelect(n_group=G, n_beam=W, n_vocab=V, n_select=K, dtype=dtype_of(torch, dtype))
    t = torch.from_numpy(x).to(dtype_of(torch, dtype)).cuda()
    assert np.array_equal(t.float().cpu().numpy(), x)
    got, par, tok = plan(t, torch.from_numpy(c).cuda())
    assert np.array_equal(par.cpu().numpy().astype(np.int64) * V + tok.cpu().numpy(), at)
    want = np.take_along_axis(s, at, 1)
    tol = 16 * 2.0 ** -24 * (1 + math.log(V) + np.abs(c).max() + np.abs(want))
    assert (np.abs(got.cpu().numpy() - want) <= tol).all()


def spoil(kind, x, low, seed):
    r = np.random.default_rng(seed)
    if kind == "by -100":
        return x - 100
    if kind == "by -1e4":
        return x - 10000
    if kind == "masked -1e4":
        return np.where(r.random(x.shape) < 0.75, -1e4, x)
    if kind == "masked lowest":
        return np.where(r.random(x.shape) < 0.95, low, x)
    if kind == "first half":
        return np.where(np.arange(x.shape[2]) < x.shape[2] // 2, low, x)
    if kind == "few allowed":
        y = np.full_like(x, low)
        for g in range(x.shape[0]):
            for w in range(x.shape[1]):
                at = r.choice(x.shape[2], 12, replace=False)
                y[g, w, at] = x[g, w, at]
        return y
    assert kind == "with barred"
    u = r.random(x.shape)
    return np.where(u < 0.5, -np.inf, np.where(u < 0.9, low, x))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["by -100", "by -1e4", "masked -1e4", "masked lowest", "first half", "few allowed", "with barred"])
@pytest.mark.parametrize("G,W,V", [(1, 4, 4000), (2, 3, 32003), (1, 1, 500)])
def test_select_far_below_zero(torch, beam, dtype, kind, G, W, V):
    """Finite logits, however low, are candidates with finite scores."""
    low = torch.finfo(dtype_of(torch, dtype)).min
    for seed in range(50):
        x, c = select_inputs(G, W, V, 1000 * seed + V)
        x = torch.from_numpy(spoil(kind, x, low, seed).astype(np.float32)).to(dtype_of(torch, dtype)).float().numpy()
        s = stable_scores(x, c)
        if select_decided(x, s, np.argsort(-s, axis=1, kind="stable")[:, :6], V):
            check_scores(torch, beam, x, c, 6, dtype)
            return
    raise AssertionError("no decided input")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [7, 5000, 40000])
@pytest.mark.parametrize("value", ["lowest", "highest", -1000.0])
def test_select_equal_extreme_logits(torch, beam, dtype, V, value):
    """A row of one value, the type's lowest or highest, is uniform: score c - log V, lowest tokens first."""
    info = torch.finfo(dtype_of(torch, dtype))
    value = {"lowest": info.min, "highest": info.max}.get(value, value)
    x = np.full((1, 1, V), value, np.float32)
    check_scores(torch, beam, x, np.array([[-2.5]], np.float32), 5, dtype)
    # beside an ordinary row that is better, and one that is worse
    y = np.concatenate([x, np.zeros((1, 1, V), np.float32), x], axis=1)
    check_scores(torch, beam, y, np.array([[-2.5, -1.0, -9.0]], np.float32), 5, dtype)
    check_scores(torch, beam, y, np.array([[-2.5, -7.0, -9.0]], np.float32), 5, dtype)


# --- attention ------------------------------------------------------------------------
# G  W  nq  nh nkv  hd    P   S: warp-level products with 16, 32 and 64 rows a tile, and the tcgen05 kernel in 16-bit types
ATTENTION = [(1, 4, 1, 8, 2, 128, 300, 40), (2, 3, 2, 8, 2, 64, 400, 9), (1, 12, 1, 16, 4, 128, 700, 20),
             (1, 9, 7, 4, 2, 48, 333, 30), (1, 40, 2, 8, 4, 128, 9001, 6), (1, 66, 1, 8, 8, 64, 4700, 3)]


def run_attention(torch, beam, c):
    n, nq, nh, hd = c["q"].shape
    W = c["n_beam"]
    plan = beam.PrefixAttention(n_group=n // W, n_beam=W, n_query=nq, n_head=nh, n_head_kv=c["pk"].shape[1], head_dim=hd,
                                dtype=c["q"].dtype, prefix_cap=c["pk"].shape[2], suffix_cap=c["sk"].shape[2])
    return plan(c["q"], c["pk"], c["pv"], c["sk"], c["sv"],
                prefix_len=torch.tensor(c["plen"], dtype=torch.int32, device="cuda"),
                suffix_len=torch.tensor(c["slen"], dtype=torch.int32, device="cuda"), slots=c["slots"])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", ATTENTION, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("value", ["-inf", "lowest"])
def test_attention_keys_that_score_minus_infinity(torch, beam, dtype, shape, value):
    """Visible keys whose scores are -inf, or so low that their weight is 0, change nothing: not in a row's first
    tile, not in whole tiles, in no kernel."""
    G, W, nq, nh, nkv, hd, P, S = shape
    c = attn_case(torch, dtype, *shape, slots=False, plen=[P] * G, slen=[S] * (G * W), seed=sum(shape))
    c["q"][..., 0] = c["q"][..., 0].abs() + 0.5
    at = torch.arange(P, device="cuda")
    hit = (at < 170) | (at % 3 == 1)
    late = torch.arange(S, device="cuda") < (S - nq) // 2
    want, wl, tol, dl = attn_ref(torch, c["q"], c["pk"][:, :, ~hit], c["pv"][:, :, ~hit], c["sk"][:, :, ~late],
                                 c["sv"][:, :, ~late], [int((~hit).sum())] * G, [int((~late).sum())] * (G * W), None, W,
                                 1 / math.sqrt(hd))
    low = -math.inf if value == "-inf" else torch.finfo(c["q"].dtype).min
    c["pk"][:, :, hit, 0] = low
    c["sk"][:, :, late, 0] = low
    out, lse = run_attention(torch, beam, c)
    tol = tol + ROUND[str(c["q"].dtype)] * want.abs() + 2.0 ** -25
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    assert bool(((out.double() - want).abs() <= tol).all())
    assert bool(((lse.double() - wl).abs() <= dl).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", ATTENTION, ids=lambda s: "x".join(map(str, s)))
def test_attention_all_scores_minus_infinity(torch, beam, dtype, shape):
    """A token all of whose scores are -inf is one that sees nothing."""
    G, W, nq, nh, nkv, hd, P, S = shape
    c = attn_case(torch, dtype, *shape, slots=False, plen=[P] * G, slen=[S] * (G * W), seed=sum(shape))
    c["q"][..., 0] = c["q"][..., 0].abs() + 0.5
    c["pk"][..., 0] = -math.inf
    c["sk"][..., 0] = -math.inf
    out, lse = run_attention(torch, beam, c)
    assert (out == 0).all() and torch.isneginf(lse).all()
    c["sk"][W - 1, :, 0, 0] = 1   # one position of one sequence is seen after all
    out, lse = run_attention(torch, beam, c)
    mine = torch.zeros(G * W, dtype=torch.bool, device="cuda")
    mine[W - 1] = True
    assert (out[~mine] == 0).all() and torch.isneginf(lse[~mine]).all()
    v = c["sv"][W - 1, :, 0].repeat_interleave(nh // nkv, 0).expand(nq, -1, -1)
    assert torch.equal(out[W - 1], v) and torch.isfinite(lse[W - 1]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", ATTENTION, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("where", ["prefix", "suffix"])
def test_attention_infinite_and_largest_values(torch, beam, dtype, shape, where):
    """Visible values of V: infinite ones keep their sign, opposite ones and NaN give NaN, the largest finite ones a
    finite result, and the other dimensions are as if they were not there."""
    G, W, nq, nh, nkv, hd, P, S = shape
    c = attn_case(torch, dtype, *shape, slots=False, plen=[P] * G, slen=[S] * (G * W), seed=sum(shape))
    k, v, at = (c["pk"], c["pv"], (P // 2, P - 1)) if where == "prefix" else (c["sk"], c["sv"], (0, (S - nq) // 2))
    for i in at:
        k[:, :, i] = 0            # a weight that is not lost in any type
    big = torch.finfo(v.dtype).max
    v[:, :, at[0], 1], v[:, :, at[1], 2] = big, -big
    want, wl, tol, dl = attn_ref(torch, c["q"], c["pk"], c["pv"], c["sk"], c["sv"], c["plen"], c["slen"], None, W,
                                 1 / math.sqrt(hd))
    tol = tol + ROUND[str(v.dtype)] * want.abs() + 2.0 ** -25
    v[:, :, at[0], 3] = math.inf
    v[:, :, at[1], 5] = -math.inf
    v[:, :, at[0], 7] = math.nan
    if at[0] != at[1]:
        v[:, :, at[0], 9], v[:, :, at[1], 9] = math.inf, -math.inf
    out, lse = run_attention(torch, beam, c)
    assert torch.isposinf(out[..., 3]).all() and torch.isneginf(out[..., 5]).all() and torch.isnan(out[..., 7]).all()
    assert at[0] == at[1] or torch.isnan(out[..., 9]).all()
    rest = [d for d in range(hd) if d not in (3, 5, 7, 9)]
    assert bool(((out.double() - want).abs() <= tol)[..., rest].all())
    assert bool(((lse.double() - wl).abs() <= dl).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", ATTENTION, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("low,high", [(2.0, 9.0), (-9.0, -2.0)])
def test_attention_enormous_scores(torch, beam, dtype, shape, low, high):
    """Scores of 2^28 to 2^40: the largest one takes all the weight, whatever its sign."""
    G, W, nq, nh, nkv, hd, P, S = shape
    c = attn_case(torch, dtype, *shape, slots=False, plen=[P] * G, slen=[S] * (G * W), seed=sum(shape))
    gen = torch.Generator(device="cuda").manual_seed(3)
    c["q"].zero_()
    c["q"][..., 0] = torch.randint(1, 5, c["q"].shape[:3], device="cuda", generator=gen).to(c["q"].dtype)
    for k in ("pk", "sk"):
        c[k][..., 0] = low
    c["pk"][:, :, P // 3, 0] = high
    if high < 0:
        c["pk"][:, :, P // 3 + 1:, 0] = low - 1
    scale = 1e9 / 3
    plan = beam.PrefixAttention(n_group=G, n_beam=W, n_query=nq, n_head=nh, n_head_kv=nkv, head_dim=hd, dtype=c["q"].dtype,
                                prefix_cap=P, suffix_cap=S, scale=scale)
    out, lse = plan(c["q"], c["pk"], c["pv"], c["sk"], c["sv"])
    want = c["pv"][:, :, P // 3].repeat_interleave(nh // nkv, 1).repeat_interleave(W, 0)[:, None].expand(-1, nq, -1, -1)
    assert torch.equal(out, want)
    top = c["q"][..., 0].double() * high * scale
    assert bool(((lse.double() - top).abs() <= 2.0 ** -21 * top.abs()).all())
