"""Penalties of each row for a session's scores are held to the ranges of the single ones."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_penalties_out_of_range_are_refused():
    from detllm_amd import synth
    from detllm_amd._lib import DetllmError
    from detllm_amd.model import F32Llama

    w = synth.WORKLOADS["tiny"]
    toks = [int(t) for t in synth.tokens(w)]
    model = F32Llama.from_gguf(synth.build_model(w))
    with model.forward_workspace(len(toks), len(toks)) as s:
        s.forward_chunk(toks, 0)
        n, inf, nan = 4, float("inf"), float("nan")
        good = dict(history=[1, 2], repetition=np.full(n, 1.5), presence=np.full(n, 0.5), frequency=np.full(n, -0.25))
        want = s.token_scores(toks[:n], **dict(good, repetition=1.5, presence=0.5, frequency=-0.25))
        for name, values in (("repetition", (0.0, -0.0, -1.0, inf, -inf, nan)), ("presence", (inf, -inf, nan)),
                             ("frequency", (inf, -inf, nan))):
            for bad in values:
                for at in (0, n - 1):
                    rows = good[name].copy()
                    rows[at] = bad
                    with pytest.raises(DetllmError) as e:
                        s.token_scores(toks[:n], **dict(good, **{name: rows}))
                    assert e.value.status == 42
                    # without a history nothing is made of it, as of a single value
                    s.token_scores(toks[:n], allowed=np.ones(w.vocab, bool), **{name: rows})
        got = s.token_scores(toks[:n], **good)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
