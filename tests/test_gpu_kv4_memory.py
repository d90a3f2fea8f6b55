"""GPU: the append's rotated queries beside, among and instead of what they are made from."""
import pytest

import kv4_ref as ref
from test_gpu_kv4 import angles, kv4, noise, torch  # noqa: F401

pytestmark = pytest.mark.gpu

N, NQ, NH, NKV, HD = 2, 3, 4, 2, 64


def append(torch, kv4, q, q_out=None, halves=False):
    k, v = (noise(torch, i, N, NQ, NKV, HD, dtype=q.dtype) for i in (1, 2))
    p = ref.Pages(kv4, [40, 7], NKV, HD, 16)
    cos, sin = angles(torch, 64, HD)
    return kv4.append(q, k, v, p.cache, p.table, p.lengths, cos=cos, sin=sin, halves=halves, q_out=q_out)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("dims", [(0,), (1,), (2,), (0, 1, 2)])
def test_broadcast_queries(torch, kv4, dtype, dims):
    """They are read as they are, and not turned in place."""
    from fwb.model import FwbError
    one = noise(torch, 3, *(1 if i in dims else n for i, n in enumerate((N, NQ, NH))), HD, dtype=ref.DTYPES[dtype])
    q = one.expand(N, NQ, NH, HD)
    before = one.clone()
    assert torch.equal(append(torch, kv4, q), append(torch, kv4, q.contiguous()))
    with pytest.raises(FwbError, match="overlap one another"):
        append(torch, kv4, q, q_out=q)
    assert torch.equal(one, before)
    kv4.check_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("at", ["head", "token", "seq"])
def test_results_among_the_queries(torch, kv4, dtype, halves, at):
    """Rows of q and of q_out in turn in one buffer, in each other's gaps."""
    shape = {"head": (N, NQ, NH, 2, HD), "token": (N, NQ, 2, NH, HD), "seq": (N, 2, NQ, NH, HD)}[at]
    dim = shape.index(2, 2 if at == "token" else 3 if at == "head" else 1)
    whole = noise(torch, 3, *shape, dtype=ref.DTYPES[dtype])
    for first in (0, 1):
        q, q_out = whole.select(dim, first), whole.select(dim, 1 - first)
        before = q.clone()
        want = append(torch, kv4, before, halves=halves)
        assert append(torch, kv4, q, q_out=q_out, halves=halves) is q_out
        assert torch.equal(q_out, want) and torch.equal(q, before)
    kv4.check_status()


def test_results_over_a_part_of_the_queries(torch, kv4):
    whole = torch.zeros(N, NQ, NH + 2, HD, device="cuda")
    q = whole[:, :, :NH]
    for q_out in (whole[:, :, 1:NH + 1], whole[:, :, 2:], whole.flatten()[16:16 + N * NQ * NH * HD].view(N, NQ, NH, HD)):
        with pytest.raises(ValueError, match="apart"):
            append(torch, kv4, q, q_out=q_out)
    assert bool((whole == 0).all())
    # the same memory by another view is q itself, whatever the strides of dimensions of one element
    x = noise(torch, 3, N, 1, NH, HD)
    k, p = noise(torch, 4, N, 1, NKV, HD), ref.Pages(kv4, [40, 7], NKV, HD, 16)
    cos, sin = angles(torch, 64, HD)
    want = kv4.append(x, k, k, p.cache, p.table, p.lengths, cos=cos, sin=sin)
    same = x.as_strided(x.shape, (NH * HD, 16, HD, 1))
    assert kv4.append(x, k, k, p.cache, p.table, p.lengths, cos=cos, sin=sin, q_out=same) is same and torch.equal(x, want)
