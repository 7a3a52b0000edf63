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


def test_ids_and_places_are_whole_numbers():
    good = dict(history=[[1, 2], [3, 4]], prompt=[1, 2], bias_ids=[5, 6], bias=[0.5, 1.0])
    for name in ("history", "prompt", "bias_ids"):
        for make in (lambda x: x + 0.5, lambda x: x.astype(np.float64), lambda x: x.astype(np.float16), lambda x: x > 1,
                     lambda x: x.astype(complex), lambda x: x.astype(str), lambda x: x.astype(object) + 2**70):
            with pytest.raises(TypeError, match=name):
                by(**dict(good, **{name: make(np.array(good[name]))}))
        kinds = (np.int64, np.int32, np.int16, np.int8, np.uint64, np.uint32, np.uint8)
        arrays = [by(**dict(good, **{name: np.array(good[name], t)}))[1] for t in kinds] + [by(**good)[1]]
        assert all(np.array_equal(x, y) for keep in arrays for x, y in zip(keep, arrays[-1]))
    for one in (1.5, True, None):
        with pytest.raises(TypeError):
            by(history=[1, 2], prompt=[one])
    with pytest.raises(TypeError):
        by(history=[1, 2], prompt=1.0)
    # empty lists have no type of their own
    a, _ = by(history=[], bias_ids=[], bias=[])
    assert a.history_len == 0 == a.bias_len
    a, _ = by(history=[[], []], prompt=[3, 4], bias_ids=[[], []], bias=[[], []])
    assert a.history_len == 0 == a.bias_len
