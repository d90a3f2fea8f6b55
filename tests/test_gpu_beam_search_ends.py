"""GPU: what fwb_beam_search returns has ended, whatever ended the search."""
import os

import numpy as np
import pytest

from fwb import configs, gguf_synth
from fwb.model import Model
from test_gpu_beam_search import TOL, Oracle, gpu  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def small(built, tmp_path_factory):
    d = tmp_path_factory.mktemp("beam_ends")
    return gguf_synth.write_model(os.path.join(d, "small.gguf"), configs.SMALL_Q4_0, seed=31)


def search(orc, prompt, W, steps, eos, penalty):
    """The search by its definition: results end with eos or have `steps` tokens."""
    live, done = [((), 0.0)], []
    for t in range(steps):
        cand = []
        for seq, s in live:
            lp = orc.logp(list(prompt) + list(seq)) + s
            cand += [(lp[v], seq + (int(v),)) for v in np.argsort(-lp, kind="stable")[:2 * W]]
        cand.sort(key=lambda c: -c[0])
        live = []
        for i, (s, seq) in enumerate(cand[:2 * W]):
            if len(live) == W:
                break
            if seq[-1] != eos:
                live.append((seq, s))
            elif i < W:
                done.append((s / len(seq) ** penalty, seq))
        if len(done) >= W and (penalty or live[0][1] <= sorted((s for s, _ in done), reverse=True)[W - 1]):
            break
    done += [(s / len(q) ** penalty, q) for q, s in live if len(q) == steps]
    return sorted(done, key=lambda d: -d[0])[:W]


@pytest.mark.parametrize("penalty", [0.0, 0.6, 1.0, 3.0, -0.5])
@pytest.mark.parametrize("prompt,W", [([5, 900, 17, 33], 4), ([7], 2), ([1, 2, 3, 4, 5, 6], 1), ([11, 1500], 8)])
def test_results_have_ended(gpu, small, penalty, prompt, W):
    steps = 10
    orc = Oracle(small)
    # of the tokens that the search meets at its second step, one that most beams can end with
    lp = sum(np.exp(orc.logp(prompt + list(t))) for _, t in search(orc, prompt, W, 1, None, 0.0))
    eos = int(np.argmax(lp))
    want = search(orc, prompt, W, steps, eos, penalty)
    with Model(small, max_ctx=128) as m:
        got = m.beam_search(prompt, W, steps, eos=eos, length_penalty=penalty)
    assert len(got) == len(want)
    for t, s in got:
        assert t[-1] == eos or len(t) == steps, f"a continuation of {len(t)} tokens has not ended"
        assert eos not in t[:-1]
        assert abs(s - orc.score(prompt, t) / len(t) ** penalty) <= TOL * steps / len(t) ** min(penalty, 0)
    assert [s for _, s in got] == sorted((s for _, s in got), reverse=True)
