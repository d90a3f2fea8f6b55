"""GPU: a uniform number of 1 and more draws the last token that stays, however little it weighs."""
import math

import pytest

from test_gpu_sample_rows import definition, sample_rows, torch  # noqa: F401

pytestmark = pytest.mark.gpu

SETTINGS = [dict(), dict(k=3), dict(k=12), dict(low=2.0 ** -33), dict(low=1e-16), dict(p=0.999)]


def rare(torch, sample_rows, dtype, V, setting, u):
    """(token, logprob) of four rows of 15 tokens, weights down to exp(-45), and what each should be."""
    x = torch.full((4, V), -math.inf, device="cuda")
    for i in range(4):                                             # steps of an eighth or more: no limit near a border
        at = torch.randperm(V, generator=torch.Generator().manual_seed(i))[:15]
        x[i, at.cuda()] = torch.tensor([5.0 - 3 * j - 0.125 * i * (j % 3) for j in range(15)], device="cuda")
    x = x.to(getattr(torch, dtype))
    f32, i32 = torch.float32, torch.int32
    kw = {a: torch.full((4,), setting[b], dtype=t, device="cuda") for a, b, t in
          (("top_k", "k", i32), ("top_p", "p", f32), ("min_p", "low", f32)) if b in setting}
    got = sample_rows(x, torch.full((4,), u, device="cuda"), **kw)
    p, low = (float(kw[n][0]) if n in kw else d for n, d in (("top_p", 1.0), ("min_p", 0.0)))
    return got, [definition(torch, x[i], 1.0, 1.0, setting.get("k", 0), p, low) for i in range(4)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [20, 1000, 128256])
@pytest.mark.parametrize("setting", SETTINGS, ids=str)
@pytest.mark.parametrize("u", [1.0, 3.0, math.inf])
def test_the_last_token_that_stays(torch, sample_rows, dtype, V, setting, u):
    (token, _), want = rare(torch, sample_rows, dtype, V, setting, u)
    assert token.tolist() == [w[0] for w in want]


def ties(torch, sample_rows):
    """Thousands of equal entries of weight 2^-60, more than a list holds, below one that has all the mass."""
    x = torch.full((3, 9000), -60.0, device="cuda")
    x[1, ::2] = -61.0
    x[2, 5000:] = -math.inf
    x[:, 77] = 0.0
    return sample_rows(x, torch.ones(3, device="cuda"), temperature=torch.full((3,), math.log2(math.e), device="cuda"))


def test_ties_of_the_last(torch, sample_rows):
    assert ties(torch, sample_rows)[0].tolist() == [8999, 8998, 4999]
