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
