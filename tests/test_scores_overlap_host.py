"""Where the gradient of dtl_token_scores_backward and dtl_distill* may lie: over
the logits themselves, between their rows, nowhere else near them.  Every call
here is refused on the host, for that or for its scratch, so none needs a GPU."""
import ctypes as C

import numpy as np
import pytest

INVALID, SMALL = 42, 44
P = 1 << 24  # an address that is never read
V = 70000    # a step of few rows needs scratch


def step(dtype, rows, stride, grad, grad_stride):
    """dtl_distill_step without its scratch: SMALL if the gradient may lie there."""
    from detllm_amd._lib import Logits, Teacher, lib

    z, t = Logits(P, dtype, rows, V, stride), Teacher(P, 4, P, 4, 0)
    return lib.dtl_distill_step(C.byref(z), C.byref(t), 1.0, None, P, grad, grad_stride, None, 0, None)


def others(dtype, rows, stride, grad, grad_stride):
    from detllm_amd._lib import Logits, Teacher, lib

    z, t = Logits(P, dtype, rows, V, stride), Teacher(P, 4, P, 4, 0)
    return (lib.dtl_token_scores_backward(C.byref(z), P, 8, 1.0, P, P, P, P, grad, grad_stride, None),
            lib.dtl_distill_backward(C.byref(z), C.byref(t), 1.0, P, P, grad, grad_stride, None))


@pytest.mark.parametrize("dtype,n", [(0, 4), (1, 2)])
def test_gradients_over_a_part_of_the_logits_are_refused(dtype, n):
    for rows, stride, at, grad_stride in ((2, V, 1, V), (2, V, -1, V), (2, V, V, V), (2, V, -V, V), (3, V + 5, 0, V),
                                          (3, V, 0, V + 5), (1, V, 1, V), (1, V, -V + 1, V), (2, 2 * V - 1, V, 2 * V - 1),
                                          (5, 4 * V, 1, 2 * V), (2, V, 3, 4 * V)):
        assert step(dtype, rows, stride, P + at * n, grad_stride) == INVALID, (rows, stride, at, grad_stride)
        assert set(others(dtype, rows, stride, P + at * n, grad_stride)) == {INVALID}
    for rows, stride, at, grad_stride in ((2, V, 0, V), (2, V, 2 * V, V), (2, V, -2 * V, V), (1, V, 0, 7 * V), (1, V, V, V),
                                          (1, V, -V, V), (9, 2 * V, V, 2 * V), (9, 2 * V, -V, 2 * V), (5, 4 * V, V, 2 * V),
                                          (5, 2 * V, -11 * V, 2 * V)):
        assert step(dtype, rows, stride, P + at * n, grad_stride) == SMALL, (rows, stride, at, grad_stride)


def test_every_layout_against_the_elements():
    rng = np.random.default_rng(1)
    seen = set()
    for _ in range(4000):
        rows = int(rng.integers(1, 7))
        strides = [V * int(rng.integers(1, 5)) + int(rng.integers(0, 3)) for _ in range(2)]
        if rng.random() < 0.5:
            strides[1] = strides[0]
        at = V * int(rng.integers(-12, 13)) + int(rng.integers(-2, 3))
        a = np.arange(rows) * strides[0]
        g = at + np.arange(rows) * strides[1]
        bad = bool((np.abs(a[:, None] - g[None]) < V).any())
        if at == 0 and (strides[0] == strides[1] or rows == 1):
            bad = False
        got = step(0, rows, strides[0], P + 4 * at, strides[1])
        assert got == (INVALID if bad else SMALL), (rows, strides, at)
        seen.add(bad)
    assert seen == {True, False}
