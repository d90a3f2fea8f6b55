"""GPU: draws whose limit falls on the border of what a list holds, to the last bit of the running mass."""
import pytest

from test_gpu_sample_rows import sample_rows, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def test_draws_among_thousands_of_rare_ties(torch, sample_rows):
    """One token and 4999 equal ones of 2^-36 of it each: u of 1 - 2^-24 falls among these, at a place that the row's
    temperature moves.  Ten in a million draws fall between the sums of two divisions of the ties."""
    n, V = 32768, 5000
    x = torch.full((n, V), -24.75, device="cuda")
    x[:, 1234] = 0.0
    u = torch.full((n,), 1.0 - 2.0 ** -24, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(48):
        temp = 0.995 + 0.01 * torch.rand(n, device="cuda", generator=gen)
        token, logprob = sample_rows(x, u, temperature=temp)
        y = -24.75 / temp.double()
        rest = 4999 * torch.exp(y)
        # the tie at which the running mass passes u times all of it, from the definition; a weight carries 2^-22, their
        # sum and the limit 2^-52 of the mass: `wide` ties
        place = ((1 - 2.0 ** -24) * (1 + rest) - 1) / torch.exp(y)
        want = place + (place >= 1234)
        wide = place * 2.0 ** -21 + 2.0 ** -51 / torch.exp(y) + 2
        assert bool(((token >= 0) & (token < V)).all()), token[(token < 0) | (token >= V)].tolist()
        assert bool(((token - want).abs() <= wide).all()), float(((token - want).abs() - wide).max())
        # its rounding 2^-20, the weight 2^-22 twice, and where a weight lies on a border between bins the rounding of an
        # exponent of 32 to 64, 2^-19 ln 2: below 2^-18
        assert bool(((logprob.double() - y).abs() <= 2.0 ** -18).all())
