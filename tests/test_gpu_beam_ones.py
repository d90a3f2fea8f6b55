"""GPU: the strides of dimensions of one element do not matter to the beam-search
operators (views leave any number there)."""
import pytest

from test_gpu_beam import attn_case, attn_check, beam, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def odd(t):
    """The same tensor with other strides in its dimensions of one element."""
    return t.as_strided(t.shape, [s + 3 if n == 1 else s for n, s in zip(t.shape, t.stride())])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 4, 1, 64, 70, 9), (1, 1, 1, 1, 1, 128, 1, 1), (1, 5, 1, 8, 2, 128, 300, 1),
                                   (2, 3, 2, 2, 1, 32, 65, 7)], ids=lambda s: "x".join(map(str, s)))
def test_attention(torch, beam, dtype, shape):
    c = attn_case(torch, dtype, *shape, seed=7)
    want, lse = attn_check(torch, beam, c)
    for k in ("q", "pk", "sk", "slots"):
        c[k] = odd(c[k])
    out, l = attn_check(torch, beam, c)
    assert torch.equal(out, want) and torch.equal(l, lse)


def test_select(torch, beam):
    x = torch.randn(1, 1, 1000, device="cuda")
    plan = beam.BeamSelect(n_group=1, n_beam=1, n_vocab=1000, n_select=4)
    c = torch.zeros(1, 1, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(plan(x, c), plan(odd(x), c)))


def test_reorder(torch, beam):
    x = torch.randn(1, 4, 1, 33, device="cuda")
    p = torch.tensor([[1, 0, 0, 2]], dtype=torch.int32, device="cuda")
    y = beam.reorder(odd(x), p, torch.empty_like(x))
    assert torch.equal(y, x[:, [1, 0, 0, 2]])
    assert torch.equal(beam.reorder(x, p, odd(torch.empty_like(x))), y)
