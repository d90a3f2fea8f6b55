"""GPU: the log-probability of a sampled token that weighs next to nothing."""
import math

import pytest

from test_gpu_sample_rows import sample_rows, torch  # noqa: F401
from test_gpu_sample_rows_last import SETTINGS, rare, ties

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [20, 1000, 128256])
@pytest.mark.parametrize("setting", SETTINGS, ids=str)
def test_rare_tokens(torch, sample_rows, dtype, V, setting):
    (token, logprob), want = rare(torch, sample_rows, dtype, V, setting, 1.0)
    for i, (at, lp, _, _) in enumerate(want):
        assert int(token[i]) == at
        # its weight and the others' sum to 2^-22 each, the logarithm's rounding to 32 bits
        assert abs(float(logprob[i]) - lp) <= 2.0 ** -20 + abs(lp) * 2.0 ** -23, (i, float(logprob[i]), lp)


def test_ties(torch, sample_rows):
    _, logprob = ties(torch, sample_rows)
    for got, octaves in zip(logprob.tolist(), (60, 61, 60)):
        # the temperature is held in 32 bits: 2^-24 of the exponent
        assert abs(got + octaves * math.log(2)) <= 2.0 ** -20 + octaves * 2.0 ** -23
