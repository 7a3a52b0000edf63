"""The host arrays that Session.token_scores makes of its arguments."""
import numpy as np
import pytest


def by(n=2, vocab=9, history=None, prompt=None, repetition=1.0, presence=0.0, frequency=0.0, bias_ids=None, bias=None,
       allowed=None):
    from detllm_amd.model import _adjust

    return _adjust(n, vocab, history, prompt, repetition, presence, frequency, bias_ids, bias, allowed)


@pytest.mark.parametrize("history", [[1, 2, 3], [[1, 2, 3], [4, 5, 6]]])
def test_prompts_are_narrowed_to_places_of_the_history(history):
    for p in (0, 2, 3, 4, -1, -(2**31) - 1, -(2**40), -(2**63), 2**31, 2**32, 2**32 + 1, 2**63 - 1):
        want = min(max(p, 0), 3)
        for prompt in (p, [p, 1], np.array([p, 1])):
            a, keep = by(history=history, prompt=prompt)
            assert keep[1].dtype == np.int32 and keep[1].tolist() == [want, want if prompt is p else 1]
            assert a.prompt == keep[1].ctypes.data
    assert by(history=history, prompt=np.array([2**64 - 1, 1], np.uint64))[1][1].tolist() == [3, 1]
