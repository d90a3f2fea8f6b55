"""GPU: a beam search that does not fit the device's memory is refused, and that
is all that it leaves behind."""
import os
from dataclasses import replace

import numpy as np
import pytest

from fwb import configs, gguf_synth
from fwb.model import FwbError, Model
from test_gpu_beam_search import gpu  # noqa: F401

pytestmark = pytest.mark.gpu


def test_after_a_search_that_does_not_fit(gpu, tmp_path):
    import torch
    path = gguf_synth.write_model(os.path.join(tmp_path, "long.gguf"), replace(configs.SMALL_Q4_0, n_ctx=65536), seed=31)
    prompt = [4, 8, 15, 16, 23, 42]
    with Model(path, max_ctx=65536) as m:
        want = m.beam_search(prompt, 4, 6)
        free = torch.cuda.mem_get_info()[0]
        rest = torch.empty(free - (4 << 30), dtype=torch.uint8, device="cuda")
        try:
            # 64 beams of 2 layers x 2 KV heads x 128 x 4 bytes: 7.9 GB of keys
            with pytest.raises(FwbError, match="memory"):
                m.beam_search(prompt, 64, 60000)
            got = m.beam_search(prompt, 4, 6)
        finally:
            del rest
            torch.cuda.empty_cache()
    assert all(np.array_equal(t, u) and s == r for (t, s), (u, r) in zip(got, want)) and len(got) == len(want)
