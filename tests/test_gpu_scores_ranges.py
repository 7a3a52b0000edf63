"""Scores and distillation over the whole range of logits and temperatures that
they take, through the C ABI, against the definitions in 64 bits."""
import numpy as np
import pytest

import lists64
import rows64
from rows64 import DTYPES
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


# ---- lists whose logits lie far above the others ---------------------------------------


# in parts; whole rows whose step holds all or a part of them; few rows of middle length
PHASES = [(4, 70001), (130, 9001), (133, 70001), (129, 151937), (5, 40003)]


def apart(rng, rows, vocab, k, gap, T):
    """Rows whose k listed logits lie gap * T above the largest other one."""
    z = (rng.normal(0, 1, (rows, vocab)) * T).astype(np.float32)
    z -= z.max(1, keepdims=True)
    z[:, rng.random(vocab) < 0.1] = -np.inf
    ids = np.stack([rng.permutation(vocab)[:k] for _ in range(rows)])
    np.put_along_axis(z, ids, ((gap + rng.uniform(0, 3, (rows, k))) * T).astype(np.float32), 1)
    p = rng.dirichlet(np.ones(k), rows) * rng.choice([0.5, 0.9, 0.999], (rows, 1))
    return z, ids, np.log(p).astype(np.float32)


def check_rest(hip, z, ids, v, T, dtype, loss=True, gradient=True):
    rows = len(z)
    lg = Logits(hip, z, dtype, pad=1)
    w = np.random.default_rng(33).uniform(0.1, 2, rows).astype(np.float32)
    print(f"distill with rest {rows} x {z.shape[1]} {dtype} T {T}", flush=True)
    step, grad, alone, grad2 = run_distill(hip, lg, ids, v, T, True, w)
    for i in range(0, rows, 1 if rows < 10 else 31):
        want, tol, dz, dtol = lists64.distill_rest(lg.z[i], ids[i], v[i], T, float(w[i]), dtype)
        if loss:
            near(step[i], want, tol, f"loss of row {i}")
            want, tol, _, _ = lists64.distill_rest(lg.z[i], ids[i], v[i], T, 1.0, dtype)
            near(alone[i], want, tol, f"loss of row {i} alone")
        if gradient:
            near(grad[i], dz, dtol, f"gradient of row {i} by the step")
            near(grad2[i], dz, dtol, f"gradient of row {i} by the backward")


APART = [(0.5, 1.0), (50, 1.0), (95, 1.0), (95, 0.1), (300, 1.0), (300, 0.01), (800, 1.0), (2000, 1.0), (2000, 0.01), (9e4, 1e-4)]
MASKS = [(-100.0, 1.0), (-1e4, 1.0), (-65504.0, 2.0), (-65504.0, 1e-4), (float(np.finfo(np.float32).min), 1.0),
         (float(np.finfo(np.float32).min), 1e-4)]


def masked(rng, rows, vocab, value):
    """Everything outside the list at a finite mask."""
    z = make(rng, rows, vocab)
    ids = np.stack([rng.permutation(vocab)[:20] for _ in range(rows)])
    listed = np.take_along_axis(z, ids, 1)
    z[:] = value
    np.put_along_axis(z, ids, listed, 1)
    p = rng.dirichlet(np.ones(20), rows) * 0.9
    return z, ids, np.log(p).astype(np.float32)


def far_lists(hip, rows, vocab, dtype, **what):
    rng = np.random.default_rng(34)
    every = 1 if rows * vocab < 2000000 else 3
    for gap, T in APART[::every]:
        check_rest(hip, *apart(rng, rows, vocab, 20, gap, T), T, dtype, **what)
    for value, T in MASKS[::every]:
        if dtype == "f16":
            value = max(value, -65504.0)
        check_rest(hip, *masked(rng, rows, vocab, value), T, dtype, **what)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", PHASES)
def test_losses_of_lists_far_above_the_rest(hip, rows, vocab, dtype):
    far_lists(hip, rows, vocab, dtype, gradient=False)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", PHASES)
def test_gradients_of_lists_far_above_the_rest(hip, rows, vocab, dtype):
    far_lists(hip, rows, vocab, dtype, loss=False)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,vocab", [(6, 70001), (6, 5003), (130, 70001)])
def test_rows_of_weight_0(hip, rows, vocab, rest):
    """Whatever they, their list and their stats hold: zeros, and the others as without them."""
    rng = np.random.default_rng(35)
    z = make(rng, rows, vocab)
    ids, v = make_teacher(rng, z, 7)
    w = rng.uniform(0.5, 1, rows).astype(np.float32)
    off = np.arange(rows) % 3 == 1
    w[off] = 0.0
    want = run_distill(hip, Logits(hip, z, "f32"), ids, v, 1.0, rest, w)
    z[off, ::5] = np.nan
    ids[off, 0], ids[off, 1], v[off, 2] = vocab, 1 << 30, np.nan
    got = run_distill(hip, Logits(hip, z, "f32"), ids, v, 1.0, rest, w)
    for a, b in zip(got, want):
        assert np.array_equal(a[~off], b[~off])
    assert not got[0][off].any() and not got[1][off].any() and not got[3][off].any()
    assert np.isnan(got[2][off]).all()  # the loss alone knows no weights


# ---- every temperature -----------------------------------------------------------------


EVERY_T = [1e-4, 0.1, 1.0, 1e4]
SPLIT_AND_WHOLE = [(4, 70001), (130, 5003)]
KINDS = ["text", "sure", "masked", "lowest_mask", "huge"]


def logits_of(hip, rng, rows, vocab, kind, dtype):
    z = make(rng, rows, vocab, kind)
    if dtype == "f16":
        z = np.where(np.isfinite(z), np.clip(z, -65504.0, 65504.0), z).astype(np.float32)
    return Logits(hip, z, dtype, pad=3)


@pytest.mark.parametrize("T", EVERY_T)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", SPLIT_AND_WHOLE)
def test_gradients_of_scores_at_temperatures(hip, rows, vocab, dtype, T):
    rng = np.random.default_rng(36)
    for kind in KINDS:
        lg = logits_of(hip, rng, rows, vocab, kind, dtype)
        tokens = pick_tokens(rng, lg.z)
        tokens[1] = -1
        g, h = rng.normal(0, 1, rows).astype(np.float32), rng.normal(0, 0.3, rows).astype(np.float32)
        print(f"gradient {rows} x {vocab} {dtype} {kind} T {T}", flush=True)
        got = run_scores(hip, lg, tokens, T, 0)
        grad = run_scores_grad(hip, lg, got, T, g, h, pad=1)
        for i in range(0, rows, 1 if rows < 10 else 43):
            want, tol = rows64.scores_grad(lg.z[i], int(tokens[i]), T, float(g[i]), float(h[i]), got["h"][i], dtype)
            row = rows64.Row(lg.z[i], T)
            near(grad[i], want, tol + lost_score(T, g[i], h[i], row.H, row.L), f"gradient of row {i}")


@pytest.mark.parametrize("T", EVERY_T)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", SPLIT_AND_WHOLE)
def test_distillation_at_temperatures(hip, rows, vocab, dtype, T):
    rng = np.random.default_rng(37)
    for kind in KINDS:
        lg = logits_of(hip, rng, rows, vocab, kind, dtype)
        ids, v = make_teacher(rng, lg.z, 14)
        # the teacher keeps to what is unmasked, each id once
        v = np.where(np.isfinite(np.take_along_axis(lg.z, ids, 1)), v, -np.inf)
        for i, row in enumerate(ids):
            v[i, np.setdiff1d(np.arange(row.size), np.unique(row, return_index=True)[1])] = -np.inf
        v = v.astype(np.float32)
        w = rng.uniform(0.1, 2, rows).astype(np.float32)
        for rest in (False, True):
            print(f"distill {rows} x {vocab} {dtype} {kind} T {T} rest {rest}", flush=True)
            step, grad, alone, grad2 = run_distill(hip, lg, ids, v, T, rest, w)
            for i in range(0, rows, 1 if rows < 10 else 43):
                if rest:
                    loss, tol, dz, dtol = lists64.distill_rest(lg.z[i], ids[i], v[i], T, float(w[i]), dtype)
                else:
                    loss, tol, dz, dtol = rows64.distill(lg.z[i], ids[i], v[i], T, False, float(w[i]), dtype)
                    dtol = dtol + lost_distill(T, w[i], dz)
                near(step[i], loss, tol, f"loss of row {i}")
                near(grad[i], dz, dtol, f"gradient of row {i} by the step")
                near(grad2[i], dz, dtol, f"gradient of row {i} by the backward")


@pytest.mark.parametrize("T", [1.0, 0.1, 0.01])
@pytest.mark.parametrize("dtype,value", FAR[:7])
def test_distillation_with_rest_of_far_logits(hip, dtype, value, T):
    for rows, vocab in ((3, 70003), (130, 4100)):
        rng = np.random.default_rng(38)
        for kind in ("tail", "half"):
            z = far(rng, rows, vocab, value, kind)
            ids = np.stack([rng.permutation(2048)[:9] for _ in range(rows)])  # ordinary logits
            check_rest(hip, z, ids, np.log(rng.dirichlet(np.ones(9), rows) * 0.8).astype(np.float32), T, dtype)


# ---- lists far from normalised --------------------------------------------------------


@pytest.mark.parametrize("shift", [0.0, 1e3, -1e4, -1e9, 1e12, float(np.finfo(np.float32).min)])
@pytest.mark.parametrize("rows,vocab,k", [(3, 70003, 20), (130, 5003, 256), (131, 40003, 64)])
def test_lists_of_any_size(hip, rows, vocab, k, shift):
    """Without rest a list counts up to a shift: raw logits, or nothing but masks."""
    rng = np.random.default_rng(39)
    lg = Logits(hip, make(rng, rows, vocab), "f32")
    ids, _ = make_teacher(rng, lg.z, k)
    v = rng.normal(0, 1, (rows, k)).astype(np.float32)
    if abs(shift) < 1e30:
        v = v + np.float32(shift)
        v[1] = np.float32(shift)
    else:
        v[::2] = shift     # every slot
        v[1::2, ::3] = shift  # some
    w = rng.uniform(0.1, 2, rows).astype(np.float32)
    step, grad, alone, grad2 = run_distill(hip, lg, ids, v, 1.0, False, w)
    for i in range(0, rows, 1 if rows < 10 else 43):
        loss, tol, dz, dtol = rows64.distill(lg.z[i], ids[i], v[i], 1.0, False, float(w[i]), "f32")
        dtol = dtol + lost_distill(1.0, w[i], dz)
        near(step[i], loss, tol, f"loss of row {i}")
        near(grad[i], dz, dtol, f"gradient of row {i} by the step")
        near(grad2[i], dz, dtol, f"gradient of row {i} by the backward")
