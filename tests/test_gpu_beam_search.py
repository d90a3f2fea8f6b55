"""GPU: beam search on a model (fwb_beam_search) against the same search on
the oracle, token by token in 64-bit scores."""
import ctypes
import os

import numpy as np
import pytest

import pyoracle
from fwb import configs, gguf_synth, native
from fwb.model import FwbError, Model

pytestmark = pytest.mark.gpu

# A step's logits are within 1e-2 of the oracle's (parity.py), so its
# log-probabilities within twice that, and the sum over n tokens within
TOL = 2e-2


@pytest.fixture(scope="module")
def gpu(built):
    if native.product().fwb_device_count() < 1:
        pytest.skip("no CUDA device")
    return True


@pytest.fixture(scope="module")
def small(built, tmp_path_factory):
    d = tmp_path_factory.mktemp("beam")
    return gguf_synth.write_model(os.path.join(d, "small.gguf"), configs.SMALL_Q4_0, seed=31)


class Oracle:
    """Log-probabilities after any sequence: the oracle fed from the first token that differs."""

    def __init__(self, path):
        self.o = pyoracle.OracleModel(path)
        self.fed, self.last = [], None

    def logp(self, seq):
        keep = 0
        while keep < min(len(seq), len(self.fed)) - 1 and seq[keep] == self.fed[keep]:
            keep += 1
        for i in range(keep, len(seq)):
            self.last = self.o.forward(int(seq[i]), i)
        self.fed = list(seq)
        x = np.asarray(self.last, np.float64)
        x = x - x.max()
        return x - np.log(np.exp(x).sum())

    def search(self, prompt, W, steps, eos=None, penalty=0.0):
        live, done = [((), 0.0)], []
        for t in range(steps):
            cand = []
            for seq, s in live:
                lp = self.logp(list(prompt) + list(seq)) + s
                cand += [(lp[v], seq + (int(v),)) for v in np.argsort(-lp, kind="stable")[:2 * W]]
            cand.sort(key=lambda c: -c[0])
            nxt = []
            for i, (s, seq) in enumerate(cand[:2 * W]):
                if len(nxt) == W:
                    break
                if seq[-1] == eos:
                    if i < W:
                        done.append((s / len(seq) ** penalty, seq))
                else:
                    nxt.append((seq, s))
            live = nxt
            if len(done) >= W:
                best = sorted((s for s, _ in done), reverse=True)
                if penalty or live[0][1] <= best[W - 1]:
                    break
        done += [(s / len(q) ** penalty, q) for q, s in live]
        done.sort(key=lambda c: -c[0])
        return done[:W]

    def score(self, prompt, seq):
        return sum(self.logp(list(prompt) + list(seq[:i]))[int(seq[i])] for i in range(len(seq)))


@pytest.mark.parametrize("n,W,steps", [(1, 2, 3), (7, 4, 8), (40, 5, 6), (3, 16, 4), (9, 1, 12)])
def test_beam_search_matches_the_oracle(gpu, small, n, W, steps):
    prompt = np.random.default_rng(n).integers(0, 2048, n).tolist()
    orc = Oracle(small)
    want = orc.search(prompt, W, steps)
    with Model(small, max_ctx=256) as m:
        got = m.beam_search(prompt, W, steps)
        again = m.beam_search(prompt, W, steps)
    assert len(got) == W and all(len(t) == steps for t, _ in got)
    for (t, s), (t2, s2) in zip(got, again):
        assert np.array_equal(t, t2) and s == s2
    assert len({tuple(t) for t, _ in got}) == W
    scores = [s for _, s in got]
    assert scores == sorted(scores, reverse=True)
    for (t, s), (ws, wt) in zip(got, want):
        # the hypothesis's own score (its keys and values came from its own ancestors), and the search's result
        assert abs(s - orc.score(prompt, t)) <= TOL * steps
        assert abs(s - ws) <= TOL * steps
    if want[0][0] - want[min(1, W - 1)][0] > 2 * TOL * steps or W == 1:
        assert tuple(got[0][0]) == want[0][1]


@pytest.mark.parametrize("penalty", [0.0, 1.0])
def test_beam_search_ends_at_eos(gpu, small, penalty):
    prompt, W, steps = [5, 900, 17, 33], 4, 10
    orc = Oracle(small)
    eos = orc.search(prompt, W, 3)[0][1][2]     # a token that the search meets
    want = orc.search(prompt, W, steps, eos=eos, penalty=penalty)
    with Model(small, max_ctx=128) as m:
        got = m.beam_search(prompt, W, steps, eos=eos, length_penalty=penalty)
    assert any(t[-1] == eos and len(t) < steps for t, _ in got)
    for t, s in got:
        assert eos not in t[:-1]
        assert abs(s - orc.score(prompt, t) / len(t) ** penalty) <= TOL * steps
    for (t, s), (ws, wt) in zip(got, want):
        assert abs(s - ws) <= TOL * steps


def test_beam_search_leaves_the_model_usable(gpu, small):
    """Decoding after a search is decoding without it."""
    prompt = [4, 8, 15, 16, 23, 42]
    with Model(small, max_ctx=128) as m:
        m.prefill(prompt)
        want = m.generate_greedy(7, 6, 20)
        m.beam_search(prompt, 6, 10)
        assert np.array_equal(m.generate_greedy(7, 6, 20), want)


def test_beam_search_refusals(gpu, small, tmp_path):
    with Model(small, max_ctx=64) as m:
        for args in (([], 2, 4), ([1], 0, 4), ([1], 65, 4), ([1], 2, 0), ([1], 2, 64), ([5000], 2, 4), ([1] * 65, 2, 1)):
            with pytest.raises(FwbError):
                m.beam_search(*args)
        with pytest.raises(FwbError):
            m.beam_search([1], 2, 4, length_penalty=float("nan"))
        assert len(m.beam_search([1], 2, 63)) == 2
    q8 = gguf_synth.write_model(os.path.join(tmp_path, "q8.gguf"), configs.SMALL_TIED_Q8, seed=2)
    with Model(q8) as m:
        with pytest.raises(FwbError, match="Q4_0"):
            m.beam_search([1, 2], 2, 4)
    assert native.product().fwb_beam_search(None, None, 1, 1, 1, -1, 0.0, None, None, None) == -1
