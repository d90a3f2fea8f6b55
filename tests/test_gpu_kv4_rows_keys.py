"""GPU: a sequence's scores do not depend on how many others are in its call, which decides the kernel."""
import math

import pytest

import kv4_ref as ref
from test_gpu_kv4 import kv4, noise, torch  # noqa: F401
from test_gpu_kv4_sizes import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nh,nkv,hd,length", [(70, 8, 8, 128, 300), (40, 16, 8, 64, 900)])
def test_scores_alone_and_in_a_batch(torch, kv4, dtype, nq, nh, nkv, hd, length):
    """Scores of 30 and more, as ref.bounds has them for keys that are multiplied as they are."""
    n, dt = 16, ref.DTYPES[dtype]
    p, k, v = ref.filled(kv4, [length] * n, nkv, hd, 32, scale=3.0)
    q = noise(torch, 5, n, nq, nh, hd, dtype=dt, sd=4.0)
    out, lse = call(kv4, p, q, nkv)
    want, want_lse, mass, reach = ref.attention(q, k, v, [length] * n)
    assert float(want_lse.median()) > 30
    # 2^-17 of reach and the rounding of the log-sum-exp in 32 bits (of its sum, the logarithm and their addition)
    tol_lse = 2.0 ** -17 * reach + 2.0 ** -20 + want_lse.abs() * 2.0 ** -23
    d = (lse.double() - want_lse).abs()
    assert bool((d <= tol_lse).all()), float((d / tol_lse).max())
    # the average: twice the scores', 2^-11 for weights and values, and the rounding (fp16's subnormals are 2^-24 apart)
    tol = mass * (2.0 ** -11 + 2.0 ** -16 * reach + (length / 16 + 32) * 2.0 ** -23)[..., None] + want.abs() * ref.half_step(dt)
    tol += 2.0 ** -25 if dtype == "f16" else 0.0
    d = (out.double() - want).abs()
    assert bool((d <= tol).all()), float((d / tol).max())
    for s in (0, n - 1):
        p.table, p.lengths, whole = p.table[s:s + 1].contiguous(), p.lengths[s:s + 1], (p.table, p.lengths)
        one, one_lse = call(kv4, p, q[s:s + 1], nkv)
        p.table, p.lengths = whole
        d = (one_lse[0].double() - lse[s].double()).abs()
        assert bool((d <= 2 * tol_lse[s]).all()), float((d / tol_lse[s]).max())
        assert bool(((one[0].double() - out[s].double()).abs() <= 2 * tol[s]).all())
