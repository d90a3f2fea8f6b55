"""GPU: a uniform number that is NaN gives no token, whatever the row's temperature."""
import math

import pytest

from test_gpu_sample_rows import check, logits, sample_rows, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1, 300, 128256])
def test_no_token(torch, sample_rows, V):
    token, logprob = check(torch, sample_rows, logits(torch, 8, 5, V), [math.nan, math.nan, math.nan, 0.5, 0.5],
                           temp=[0.0, -1.0, 1.0, 0.0, 1.0])
    assert token[:3].tolist() == [-1] * 3 and logprob[:3].tolist() == [-math.inf] * 3
    assert bool((token[3:] >= 0).all()) and float(logprob[3]) == 0.0
