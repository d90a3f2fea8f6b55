"""GPU: fwb.beam names a tensor that a call needs and did not get."""
import pytest

from test_gpu_beam import beam, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("missing", ["q", "prefix_k", "prefix_v", "suffix_k", "suffix_v"])
def test_attention_without_a_tensor(torch, beam, missing):
    plan = beam.PrefixAttention(n_group=1, n_beam=2, n_head=4, n_head_kv=2, head_dim=64, dtype=torch.float16, prefix_cap=10,
                                suffix_cap=4)
    pk = torch.zeros(1, 2, 10, 64, dtype=torch.float16, device="cuda")
    sk = torch.zeros(2, 2, 4, 64, dtype=torch.float16, device="cuda")
    args = dict(q=torch.zeros(2, 1, 4, 64, dtype=torch.float16, device="cuda"), prefix_k=pk, prefix_v=pk, suffix_k=sk, suffix_v=sk)
    plan(**args)
    with pytest.raises(ValueError, match=f"{missing} is missing"):
        plan(**{**args, missing: None})


@pytest.mark.parametrize("missing", ["logits", "scores"])
def test_select_without_a_tensor(torch, beam, missing):
    plan = beam.BeamSelect(n_group=1, n_beam=2, n_vocab=100, n_select=4)
    args = dict(logits=torch.zeros(1, 2, 100, device="cuda"), scores=torch.zeros(1, 2, device="cuda"))
    plan(**args)
    with pytest.raises(ValueError, match=f"{missing} is missing"):
        plan(**{**args, missing: None})


def test_reorder_without_a_tensor(torch, beam):
    x, p = torch.zeros(1, 2, 4, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    for args in ((None, p), (x, None)):
        with pytest.raises(ValueError, match="is missing"):
            beam.reorder(*args)
