"""Scores and distillation over the whole range of logits and temperatures that
they take, through the C ABI, against the definitions in 64 bits."""
import numpy as np
import pytest

import rows64
from test_gpu_scores import (Logits, _free, check_scores, hip, make, make_teacher, near, pick_tokens,  # noqa: F401
                             run_distill, run_scores, run_scores_grad)

pytestmark = pytest.mark.gpu


# ---- logits of large size: segments of a row that hold nothing else ------------------


def far(rng, rows, vocab, value, kind):
    """Ordinary logits, but for
    tail: the end of every row, its short last segment among them, a finite mask;
    half: every second segment of 2048 such a mask, with a few others in it;
    all: every logit of that size, a few steps of float32 apart, or scaled by it."""
    z = make(rng, rows, vocab)
    if kind == "tail":
        z[:, (vocab - 1) // 2048 * 2048:] = value
    elif kind == "half":
        off = np.arange(vocab) // 2048 % 2 == 1
        z[:, off] = value
        z[:, off & (rng.random(vocab) < 0.01)] = value * 1.5
    elif kind == "all":
        z[::2] = np.float32(value) + np.spacing(np.float32(abs(value))) * rng.integers(0, 8, z[::2].shape).astype(np.float32)
        z[1::2] *= abs(np.float32(value))
    return z.astype(np.float32)


FAR = [("f32", -1e9), ("f32", -1e10), ("f32", -1e12), ("f32", -1e15), ("bf16", -1e9), ("bf16", -1e10), ("bf16", -1e15),
       ("f32", 1e10), ("f32", 1e30), ("f16", -65504.0)]


@pytest.mark.parametrize("T", [1.0, 0.1, 0.01, 1e-4, 1e4])
@pytest.mark.parametrize("dtype,value", FAR)
@pytest.mark.parametrize("rows,vocab", [(3, 70003), (130, 4100)])  # in parts and by whole rows
def test_scores_of_far_logits(hip, rows, vocab, dtype, value, T):
    rng = np.random.default_rng(31)
    for kind in ("tail", "half", "all"):
        if kind != "all" and value > 0:
            continue
        z = far(rng, rows, vocab, value, kind)
        if dtype == "f16":
            z = np.clip(z, -65504.0, 65504.0)
        lg = Logits(hip, z, dtype)
        assert np.isfinite(lg.z).all()
        print(kind, value, flush=True)
        check_scores(hip, lg, pick_tokens(rng, lg.z), T, 5, step=1 if rows < 10 else 43)


# An e below 2^-126 (t past -87.4 in natural units) is given as 0, as the header
# says.  What that takes from a gradient, on top of rows64's bounds:
def lost_score(T, g, h, H, L):
    """e |A + B t| with |A| <= (|g| + |h| (H + L)) / T, |B t| = |h t| / T, and e |t|
    falling in |t|: below 2^-126 (|g| + |h| (H + L + 88)) / T."""
    return 2.0 ** -126 * (abs(g) + abs(h) * (H + L + 88)) / T


def lost_distill(T, w, dz):
    """e share w T with share = 1 / sum of e <= 1; and the rounding of w T to
    float32, half a step of the whole gradient (none where T is a power of two)."""
    return 2.0 ** -126 * abs(w) * T + rows64.H * np.abs(dz)


@pytest.mark.parametrize("T", [1.0, 0.1, 0.01])
@pytest.mark.parametrize("dtype,value", FAR[:7])
def test_gradients_of_far_logits(hip, dtype, value, T):
    """Of scores, and of the loss without rest by the step and by the backward."""
    for rows, vocab in ((3, 70003), (130, 4100)):
        rng = np.random.default_rng(32)
        for kind in ("tail", "half"):
            z = far(rng, rows, vocab, value, kind)
            lg = Logits(hip, z, dtype)
            print(f"{kind} {value} {rows} x {vocab} {dtype} T {T}", flush=True)
            tokens = pick_tokens(rng, lg.z)
            got = run_scores(hip, lg, tokens, T, 0)
            g, h = rng.normal(0, 1, rows).astype(np.float32), rng.normal(0, 0.3, rows).astype(np.float32)
            grad = run_scores_grad(hip, lg, got, T, g, h)
            ids, v = make_teacher(rng, lg.z, 9)
            w = rng.uniform(0.1, 1, rows).astype(np.float32)
            dist = run_distill(hip, lg, ids, v, T, False, w)
            for i in range(0, rows, 1 if rows < 10 else 43):
                want, tol = rows64.scores_grad(lg.z[i], int(tokens[i]), T, float(g[i]), float(h[i]), got["h"][i], dtype)
                row = rows64.Row(lg.z[i], T)
                near(grad[i], want, tol + lost_score(T, g[i], h[i], row.H, row.L), f"gradient of row {i}")
                loss, tol, dz, dtol = rows64.distill(lg.z[i], ids[i], v[i], T, False, float(w[i]), dtype)
                near(dist[0][i], loss, tol, f"loss of row {i}")
                dtol = dtol + lost_distill(T, w[i], dz)
                near(dist[1][i], dz, dtol, f"gradient of row {i} by the step")
                near(dist[3][i], dz, dtol, f"gradient of row {i} by the backward")
