"""lists64's loss and gradient against rows64's where that holds, against
differences beyond, and against the terms written out."""
import numpy as np
import pytest

import lists64
import rows64

IDS = np.array([0, 5, 5, 39, -1, 8])
V = np.log(np.array([0.3, 0.1, 0.2, 0.1, 0.4, 0.05])).astype(np.float32)


def logits():
    z = np.random.default_rng(1).normal(0, 2, 40)
    z[3] = z[17] = -np.inf
    return z


def test_near_lists_are_rows64s():
    want = rows64.distill(logits(), IDS, V, 0.75, True, 0.7, "f32")
    got = lists64.distill_rest(logits(), IDS, V, 0.75, 0.7, "f32")
    assert abs(got[0] - want[0]) < 1e-14 and np.abs(got[2] - want[2]).max() < 1e-14


@pytest.mark.parametrize("gap", [0, 50, 95, 800, 2000])
def test_gradients_against_differences(gap):
    z = logits()
    z[IDS[IDS >= 0]] += gap
    loss, _, grad, _ = lists64.distill_rest(z, IDS, V, 1.0, 1.0, "f32")
    d = 1e-4  # the third derivative is below 1: d^2 / 6, and 1e-13 * gap / d of rounding
    for j in np.flatnonzero(np.isfinite(z)):
        a, b = z.copy(), z.copy()
        a[j] += d
        b[j] -= d
        f = lambda x: lists64.distill_rest(x, IDS, V, 1.0, 1.0, "f32")[0]
        assert abs((f(a) - f(b)) / (2 * d) - grad[j]) < 1e-8 + 1e-9 * gap
    # with nothing else left of the student's mass, what the list lacks is a
    # distribution of its own: the gradient outside sums to -rest
    rest = 1 - np.exp(V[IDS >= 0].astype(np.float64)).sum()
    if gap >= 50:
        outside = np.isfinite(z)
        outside[IDS[IDS >= 0]] = False
        assert abs(grad[outside].sum() + rest) < 1e-12
        # and the loss grows by rest for each step that the list is further away
        z[outside] -= 1
        assert abs(lists64.distill_rest(z, IDS, V, 1.0, 1.0, "f32")[0] - loss - rest) < 1e-11
