"""GPU: attention over the 4-bit cache where values differ by many powers of two, in positions that a token does not see
and in blocks beside one another."""
import math

import pytest

import kv4_ref as ref
from test_gpu_kv4 import kv4, noise, torch  # noqa: F401

pytestmark = pytest.mark.gpu

# sequences, tokens, query heads, KV heads, head_dim, positions: one row tile of 8, 16 and 32 rows
FEW = [(1, 4, 4, 2, 128, 90), (3, 7, 8, 8, 64, 500), (2, 9, 4, 4, 48, 300), (2, 12, 2, 1, 96, 200), (1, 40, 8, 2, 128, 2000)]


def call(kv4, p, q, heads):
    n, nq, nh, hd = q.shape
    plan = kv4.Attention(n_seq=n, n_query=nq, n_head=nh, n_head_kv=heads, head_dim=hd, dtype=q.dtype, page_size=p.page,
                         n_page=p.n_page, max_pages=p.table.shape[1])
    return plan(q, p.cache, p.table, p.lengths)


def unseen(torch, kv4, dtype, n, nq, nh, nkv, hd, length):
    """Outputs of the tokens that do not see the last position or two, whatever these hold."""
    dt = ref.DTYPES[dtype]
    q = noise(torch, 1, n, nq, nh, hd, dtype=dt)
    got = []
    for value, key in ((0.02, 1.0), (5e5, 1.0), (0.02, 300.0), (5e5, 300.0)):
        kv = noise(torch, 2, 2, n, length, nkv, hd)
        kv[1] *= 0.05
        kv[1, :, -2:] *= value / 0.05
        kv[0, :, -2:] *= key
        p = ref.Pages(kv4, [length] * n, nkv, hd, 16)
        kv4.append(None, kv[0], kv[1], p.cache, p.table, p.lengths)
        got.append(call(kv4, p, q, nkv))
    for out, lse in got[1:]:
        assert torch.equal(out[:, :-2], got[0][0][:, :-2]) and torch.equal(lse[:, :-2], got[0][1][:, :-2])
    # and they are right
    p.lengths -= 2
    k, v = kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), length - 2, head_dim=hd, dtype=torch.float32)
    check_blocks(got[3][0][:, :-2], got[3][1][:, :-2], q[:, :-2], k, v, [length - 2] * n)


def check_blocks(got, got_lse, q, k, v, lens):
    """As ref.check_attention, but every dimension against its own mass: bounds without what it grants of the largest."""
    out, lse, mass, reach = ref.attention(q, k, v, lens)
    tol, tol_lse = ref.bounds(q, out, lse, mass, reach, k.shape[1], k.shape[2])
    tol = tol - mass.amax(-1, keepdim=True) * 2.0 ** -20
    d = (got.double() - out).abs()
    assert bool((d <= tol).all()), float((d / tol).max())
    assert bool(((got_lse.double() - lse).abs() <= tol_lse).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,nq,nh,nkv,hd,length", FEW)
def test_unseen_positions_change_nothing(torch, kv4, dtype, n, nq, nh, nkv, hd, length):
    unseen(torch, kv4, dtype, n, nq, nh, nkv, hd, length)


def unequal(torch, kv4, dtype, n, nq, nh, nkv, hd, length, apart):
    dt = ref.DTYPES[dtype]
    q = noise(torch, 1, n, nq, nh, hd, dtype=dt)
    kv = noise(torch, 2, 2, n, length, nkv, hd)
    blocks = -(-hd // 32)
    for b in range(blocks):
        kv[1, ..., 32 * b:32 * b + 32] *= 2.0 ** (apart / 2 - apart * b / (blocks - 1))
    p = ref.Pages(kv4, [length] * n, nkv, hd, 16)
    kv4.append(None, kv[0], kv[1], p.cache, p.table, p.lengths)
    k, v = kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), length, head_dim=hd, dtype=torch.float32)
    check_blocks(*call(kv4, p, q, nkv), q, k, v, [length] * n)


@pytest.mark.parametrize("dtype,apart", [("f32", 16), ("f32", 26), ("f16", 16), ("bf16", 16), ("bf16", 26)])
@pytest.mark.parametrize("n,nq,nh,nkv,hd,length", FEW)
def test_blocks_beside_one_another(torch, kv4, dtype, apart, n, nq, nh, nkv, hd, length):
    """Value blocks 2^apart from the first to the last."""
    unequal(torch, kv4, dtype, n, nq, nh, nkv, hd, length, apart)


def outweighed(torch, kv4, dtype, n, nq, nh, nkv, hd, length):
    dt = ref.DTYPES[dtype]
    q = noise(torch, 1, n, nq, nh, hd).abs().add(0.1).to(dt)       # all positive
    kv = noise(torch, 2, 2, n, length, nkv, hd)
    kv[1] *= 0.02
    big = torch.arange(length, device="cuda") % 9 == 4
    kv[1, :, big] *= 2.5e6
    kv[0, :, big] = -60.0 / hd * math.sqrt(hd)                     # scores of -48 and less
    p = ref.Pages(kv4, [length] * n, nkv, hd, 16)
    kv4.append(None, kv[0], kv[1], p.cache, p.table, p.lengths)
    k, v = kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), length, head_dim=hd, dtype=torch.float32)
    check_blocks(*call(kv4, p, q, nkv), q, k, v, [length] * n)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,nq,nh,nkv,hd,length", FEW)
def test_positions_of_unequal_values(torch, kv4, dtype, n, nq, nh, nkv, hd, length):
    """One position in nine has values of 5e4 where its score leaves it next to no weight."""
    outweighed(torch, kv4, dtype, n, nq, nh, nkv, hd, length)
