"""GPU: shared-prefix attention gives the same bits in every call, for each pair
of row tiles that prefixes and suffixes can have."""
import pytest

from test_gpu_beam import attn_case, attn_check, beam, torch  # noqa: F401

pytestmark = pytest.mark.gpu

# G  W  nq  nh nkv  hd    P   S: 16, 32 or 64 query rows in a prefix tile and in a suffix tile, many items of both
PAIRS = {
    "16,16": (3, 4, 1, 16, 4, 128, 900, 20),
    "32,16": (3, 7, 1, 16, 4, 128, 900, 20),
    "32,32": (5, 1, 7, 16, 4, 128, 900, 20),
    "64,16": (2, 32, 1, 32, 8, 128, 2400, 20),
    "64,32": (2, 12, 5, 16, 4, 128, 1100, 20),
    "64,64": (3, 3, 10, 16, 4, 128, 1100, 20),
}


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("broadcast", [False, True])
def test_attention_repeats(torch, beam, dtype, pair, broadcast):
    """CTAs that go from prefix items to suffix items, with fewer warps to a row or the same; broadcast caches are read
    without the copy engine, in other times."""
    c = attn_case(torch, dtype, *PAIRS[pair], slots=False, seed=len(pair))
    if broadcast:
        for k in ("pk", "pv"):
            c[k] = c[k][:1, :1].expand(c[k].shape)
        for k in ("sk", "sv"):
            c[k] = c[k][:1].expand(c[k].shape)
    out, lse = attn_check(torch, beam, c)
    n, nq, nh, hd = c["q"].shape
    plan = beam.PrefixAttention(n_group=c["pk"].shape[0], n_beam=c["n_beam"], n_query=nq, n_head=nh,
                                n_head_kv=c["pk"].shape[1], head_dim=hd, dtype=c["q"].dtype,
                                prefix_cap=c["pk"].shape[2], suffix_cap=c["sk"].shape[2])
    plen = torch.tensor(c["plen"], dtype=torch.int32, device="cuda")
    slen = torch.tensor(c["slen"], dtype=torch.int32, device="cuda")
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(200):
        o, l = plan(c["q"], c["pk"], c["pv"], c["sk"], c["sv"], prefix_len=plen, suffix_len=slen)
        differ += (o != out).sum() + (l != lse).sum()
    assert int(differ) == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("W,nq,S", [(4, 1, 500), (3, 2, 333)])
def test_slots_that_change_by_units(torch, beam, dtype, W, nq, S):
    """Units of 16 positions from one beam, which the copy engine brings, and units from several, which come row by row,
    in turn and through the same stages."""
    c = attn_case(torch, dtype, 2, W, nq, 8, 2, 128, 100, S, slen=[S - i for i in range(2 * W)], seed=S)
    unit = torch.arange(S, device="cuda") // 16
    c["slots"] = torch.where(unit % 3 != 1, (unit * 7 // 3) % W, c["slots"]).to(torch.int32)
    out, lse = attn_check(torch, beam, c)
    plan = beam.PrefixAttention(n_group=2, n_beam=W, n_query=nq, n_head=8, n_head_kv=2, head_dim=128, dtype=c["q"].dtype,
                                prefix_cap=100, suffix_cap=S)
    plen = torch.tensor(c["plen"], dtype=torch.int32, device="cuda")
    slen = torch.tensor(c["slen"], dtype=torch.int32, device="cuda")
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(100):
        o, l = plan(c["q"], c["pk"], c["pv"], c["sk"], c["sv"], prefix_len=plen, suffix_len=slen, slots=c["slots"])
        differ += (o != out).sum() + (l != lse).sum()
    assert int(differ) == 0
