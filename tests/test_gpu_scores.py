"""Scores of given tokens and distillation (dtl_token_scores*, dtl_distill*) on
the GPU, through the C ABI, against the definitions in 64 bits (rows64.py)."""
import ctypes as C

import numpy as np
import pytest

import rows64
from rows64 import DTYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from hipmem import Hip

    h = Hip()
    yield h
    h.close()


@pytest.fixture(autouse=True)
def _free(hip):
    yield
    hip.drop()


def make(rng, rows, vocab, kind="text"):
    """Logits as a decoder leaves them, or one of the forms that go wrong."""
    z = rng.normal(0, 1, (rows, vocab)).astype(np.float32) * rng.uniform(0.5, 3, (rows, 1)).astype(np.float32)
    for row in z:
        at = rng.integers(0, vocab, min(8, vocab))
        row[at] = rng.uniform(0, 14, at.size)
    if kind == "masked":
        z[:, rng.random(vocab) < 0.4] = -np.inf
        z[:, rng.integers(0, vocab)] = 1.0
    elif kind == "equal":
        z[:] = 0.75
    elif kind == "lowest":
        z[:] = np.finfo(np.float32).min
    elif kind == "lowest_mask":
        z[:, rng.random(vocab) < 0.5] = np.finfo(np.float32).min
    elif kind == "sorted":
        z[:] = np.sort(z, 1)[:, ::-1]
    elif kind == "few":  # fewer unmasked than alternatives asked for
        keep = rng.integers(0, vocab, 3)
        v = z[:, keep].copy()
        z[:] = -np.inf
        z[:, keep] = v
    elif kind == "sure":
        z[:, rng.integers(0, vocab)] = 30.0
    elif kind == "zeros":
        z[:] = np.where(rng.random((rows, vocab)) < 0.5, np.float32(-0.0), np.float32(0.0))
    elif kind == "huge":
        z *= np.float32(1e4)
    elif kind == "mixed":
        z[0] = -np.inf
        z[1 % rows, vocab // 2] = np.nan
        z[2 % rows, vocab - 1] = np.inf
        z[3 % rows, :] = -np.inf
        z[3 % rows, vocab - 1] = -3.0
    return z


class Logits:
    def __init__(self, hip, z, dtype, pad=0, offset=0):
        from detllm_amd._lib import Logits as L

        self.dtype, self.rows, self.vocab = dtype, z.shape[0], z.shape[1]
        self.stride = self.vocab + pad
        bits = rows64.to_bits(z, dtype)
        self.z = rows64.from_bits(bits, dtype)
        wide = np.full((self.rows, self.stride), 0x7E01, bits.dtype)  # not read between the rows
        wide[:, :self.vocab] = bits
        self.addr = hip.put(wide, offset)
        self.c = L(self.addr, DTYPES[dtype][0], self.rows, self.vocab, self.stride)


def scratch(hip, n):
    return (hip.put(np.zeros(max(n, 16), np.uint8)), n)


def run_scores(hip, lg, tokens, T, top, wide=True, stats=True):
    R = lg.rows
    tok = hip.put(np.asarray(tokens, np.int64 if wide else np.int32))
    f = lambda *s: hip.put(np.full(s, 7.5, np.float32))
    lp, en, st = f(R), f(R), f(R, 2)
    ids, lps = hip.put(np.full((R, max(top, 1)), 77, np.int32)), f(R, max(top, 1))
    n = hip.dtl.dtl_token_scores_scratch(R, lg.vocab, top)
    sc, n = scratch(hip, n)
    rc = hip.dtl.dtl_token_scores(C.byref(lg.c), tok, 8 if wide else 4, T, top, lp, en, st, ids, lps, sc, n, hip.stream)
    assert rc == 0, rc
    hip.sync()
    got = dict(lp=hip.get(lp, np.float32, R), h=hip.get(en, np.float32, R), stats=hip.get(st, np.float32, (R, 2)),
               ids=hip.get(ids, np.int32, (R, max(top, 1))), lps=hip.get(lps, np.float32, (R, max(top, 1))))
    got["dev"] = dict(tok=tok, st=st, en=en)
    if not top:
        assert (got["ids"] == 77).all() and (got["lps"] == 7.5).all()
    return got


def near(got, want, tol, what):
    got, want, tol = np.asarray(got, np.float64), np.asarray(want, np.float64), np.asarray(tol, np.float64)
    # results are float32 or narrower: from 2^128 - 2^103 on, half a step past
    # the largest finite one (2^128 - 2^104), a value rounds to infinity
    want = np.where(np.abs(want) >= 2.0 ** 128 - 2.0 ** 103, np.copysign(np.inf, want), want)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        off = ~same & ~(np.abs(got - want) <= tol)
    assert not off.any(), f"{what}: {got[off][:4]} for {want[off][:4]}, tolerance {np.broadcast_to(tol, got.shape)[off][:4]}"


def check_scores(hip, lg, tokens, T, top, wide=True, step=1):
    print(f"scores {lg.rows} x {lg.vocab} {lg.dtype} top {top} T {T}", flush=True)
    got = run_scores(hip, lg, tokens, T, top, wide)
    for i in range(0, lg.rows, step):
        lp, tol_lp, h, tol_h = rows64.scores(lg.z[i], int(tokens[i]), T)
        near(got["lp"][i], lp, tol_lp, f"log_prob of row {i}")
        near(got["h"][i], h, tol_h, f"entropy of row {i}")
        if top:
            ids, lps = rows64.top(lg.z[i], top, T)
            assert got["ids"][i].tolist() == ids.tolist(), f"row {i}"
            row = rows64.Row(lg.z[i], T)
            tol = 0.0 if row.bad or row.empty else row.tol_L + 2 * rows64.H * np.where(np.isfinite(lps), np.abs(lps), 0)
            near(got["lps"][i], lps, tol + 2.0 ** -149, f"alternatives of row {i}")
    return got


def pick_tokens(rng, z):
    t = rng.integers(0, z.shape[1], z.shape[0])
    t[::2] = z[::2].argmax(1)
    return t


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_many_rows_of_middle_length(hip, dtype):
    rng = np.random.default_rng(21)
    z = make(rng, 1030, 9500)
    z[::7] = np.round(z[::7])  # ties among the alternatives
    lg = Logits(hip, z, dtype, pad=1)
    check_scores(hip, lg, pick_tokens(rng, lg.z), 1.0, 32, step=49)
    check_scores(hip, lg, pick_tokens(rng, lg.z), 2.0, 100, step=113)


SHAPES = [(1, 1), (1, 2), (3, 7), (2, 63), (1, 2047), (2, 2048), (3, 2049), (5, 32003), (2, 49152), (1, 151936),
          (1, 1 << 18)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_scores_over_vocabularies(hip, rows, vocab, dtype):
    rng = np.random.default_rng(vocab * 7 + rows)
    z = make(rng, rows, vocab)
    lg = Logits(hip, z, dtype)
    for top in sorted({0, 1, min(vocab, 20), min(vocab, 128)}):
        check_scores(hip, lg, pick_tokens(rng, lg.z), 1.0, top)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", ["masked", "equal", "lowest", "lowest_mask", "sorted", "few", "sure", "zeros", "huge",
                                  "mixed"])
@pytest.mark.parametrize("rows,vocab", [(4, 70001), (260, 5003)])  # in parts and by whole rows
def test_scores_of_logits_that_go_wrong(hip, rows, vocab, kind, dtype):
    rng = np.random.default_rng(len(kind))
    z = make(rng, rows, vocab, kind)
    if dtype == "f16" and "lowest" in kind:
        z = np.maximum(z, -65504.0)
    if dtype == "f16" and kind == "huge":
        z = np.clip(z, -65504.0, 65504.0)
    lg = Logits(hip, z, dtype, pad=5)
    tokens = pick_tokens(rng, np.nan_to_num(lg.z, nan=0.0))
    tokens[-1] = -1
    check_scores(hip, lg, tokens, 1.0, 64, step=1 if rows < 10 else 37)
    check_scores(hip, lg, tokens, 0.25, 3, step=1 if rows < 10 else 37)


@pytest.mark.parametrize("T", [1e-4, 0.1, 0.7, 1.0, 2.5, 1e4])
def test_scores_at_temperatures(hip, T):
    rng = np.random.default_rng(5)
    for dtype in DTYPES:
        lg = Logits(hip, make(rng, 3, 9001), dtype)
        check_scores(hip, lg, [5, -1, 9000], T, 8, wide=False)


def test_tokens_out_of_the_vocabulary(hip):
    rng = np.random.default_rng(6)
    lg = Logits(hip, make(rng, 5, 777), "f32")
    got = check_scores(hip, lg, np.array([777, -1, -(1 << 40), 1 << 40, 776]), 1.0, 0)
    assert np.isnan(got["lp"][[0, 3]]).all() and (got["lp"][[1, 2]] == 0).all() and got["lp"][4] < 0


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows_give_the_same_bits_alone_and_among_others(hip, dtype):
    """Row by row, in parts, whole, misaligned: a row's results depend on the row."""
    rng = np.random.default_rng(8)
    vocab, rows = 70001, 180
    z = make(rng, rows, vocab)
    tokens = pick_tokens(rng, z)
    all_ = run_scores(hip, Logits(hip, z, dtype), tokens, 0.7, 40)
    for lo, hi, pad, offset in ((0, 1, 0, 0), (7, 8, 3, 2), (100, 120, 1, 6), (12, 179, 64, 0)):
        offset = offset * 2 if dtype == "f32" else offset
        part = run_scores(hip, Logits(hip, z[lo:hi], dtype, pad, offset), tokens[lo:hi], 0.7, 40)
        for k in ("lp", "h", "stats", "lps"):
            assert np.array_equal(part[k].view(np.uint32), all_[k][lo:hi].view(np.uint32)), (k, lo, hi)
        assert np.array_equal(part["ids"], all_["ids"][lo:hi])


# ---- gradients of the scores -----------------------------------------------------


def run_scores_grad(hip, lg, got, T, g, h, wide=True, pad=0, offset=0, in_place=False):
    dt, size, _ = DTYPES[lg.dtype]
    bits = np.dtype(f"u{size}")
    stride = lg.stride if in_place else lg.vocab + pad
    out = lg.addr if in_place else hip.put(np.full((lg.rows, stride), 0x1234, bits), offset)
    dg = None if g is None else hip.put(np.asarray(g, np.float32))
    dh = None if h is None else hip.put(np.asarray(h, np.float32))
    rc = hip.dtl.dtl_token_scores_backward(C.byref(lg.c), got["dev"]["tok"], 8 if wide else 4, T, got["dev"]["st"],
                                           got["dev"]["en"], dg, dh, out, stride, hip.stream)
    assert rc == 0, rc
    hip.sync()
    raw = hip.get(out, bits, (lg.rows, stride))
    if not in_place:
        assert (raw[:, lg.vocab:] == 0x1234).all(), "written between the rows"
    return rows64.from_bits(np.ascontiguousarray(raw[:, :lg.vocab]), lg.dtype)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,kind", [(1, 1, "text"), (2, 3, "text"), (3, 2049, "text"), (5, 32003, "text"),
                                             (2, 151936, "text"), (4, 5003, "mixed"), (4, 5003, "masked"),
                                             (3, 5003, "sure"), (2, 5003, "lowest_mask"), (2, 700, "equal")])
def test_scores_gradient(hip, rows, vocab, kind, dtype):
    rng = np.random.default_rng(vocab + rows)
    z = make(rng, rows, vocab, kind)
    if dtype == "f16":
        z = np.where(np.isfinite(z), np.clip(z, -65504.0, 65504.0), z).astype(np.float32)
    tokens = pick_tokens(rng, np.nan_to_num(z))
    if rows > 2:
        tokens[2] = -1
    T = 0.75
    lg = Logits(hip, z, dtype, pad=3)
    got = run_scores(hip, lg, tokens, T, 0)
    g = rng.normal(0, 1, rows).astype(np.float32)
    h = rng.normal(0, 0.3, rows).astype(np.float32)
    none = np.zeros(rows, np.float32)
    for gg, hh in ((g, h), (g, None), (None, h), (none, none)):
        print(f"gradient {rows} x {vocab} {dtype} {kind} {gg is not None} {hh is not None}", flush=True)
        grad = run_scores_grad(hip, lg, got, T, gg, hh, pad=1, offset=2 * DTYPES[dtype][1])
        for i in range(rows):
            want, tol = rows64.scores_grad(lg.z[i], int(tokens[i]), T, 0.0 if gg is None else float(gg[i]),
                                           0.0 if hh is None else float(hh[i]), got["h"][i], dtype)
            near(grad[i], want, tol, f"gradient of row {i}")
    want = run_scores_grad(hip, lg, got, T, g, h)
    assert np.array_equal(run_scores_grad(hip, lg, got, T, g, h, in_place=True), want, equal_nan=True)


# ---- distillation ---------------------------------------------------------------


def make_teacher(rng, z, k, rest=True):
    rows, vocab = z.shape
    ids = rng.integers(0, vocab, (rows, k))
    best = np.argsort(-np.nan_to_num(z, nan=-1e30, posinf=-1e30), 1)[:, :max(1, min(k // 2, vocab))]
    ids[:, :best.shape[1]] = best
    v = np.clip(np.nan_to_num(np.take_along_axis(z, ids, 1), nan=0, posinf=0, neginf=-9), -20, 20) + rng.normal(0, 0.5, ids.shape)
    v = v - np.log(np.exp(v - v.max(1, keepdims=True)).sum(1, keepdims=True)) - v.max(1, keepdims=True)
    v = v + np.log(rng.uniform(0.5, 1.0, (rows, 1)))
    return ids, v.astype(np.float32)


def run_distill(hip, lg, ids, v, T, rest, weights, wide=True, pad=0, offset=0, in_place=False):
    """(loss, gradient by the step, loss, gradient by forward and backward)"""
    from detllm_amd._lib import Teacher

    dt, size, _ = DTYPES[lg.dtype]
    bits = np.dtype(f"u{size}")
    R = lg.rows
    dv = hip.put(v.astype(np.float32))
    t = Teacher(hip.put(ids.astype(np.int64 if wide else np.int32)), 8 if wide else 4, dv, ids.shape[1],
                int(rest))
    w = hip.put(np.asarray(weights, np.float32))
    n = hip.dtl.dtl_distill_scratch(R, lg.vocab)
    sc, n = scratch(hip, n)
    f = lambda *s: hip.put(np.full(s, 7.5, np.float32))
    loss2, stats = f(R), f(R, 5)
    assert hip.dtl.dtl_distill(C.byref(lg.c), C.byref(t), T, loss2, stats, sc, n, hip.stream) == 0
    stride = lg.vocab + pad
    out2 = hip.put(np.full((R, stride), 0x1234, bits), offset)
    assert hip.dtl.dtl_distill_backward(C.byref(lg.c), C.byref(t), T, stats, w, out2, stride, hip.stream) == 0
    loss, out = f(R), hip.put(np.full((R, stride), 0x1234, bits), offset)
    if in_place:
        out, stride = lg.addr, lg.stride
    assert hip.dtl.dtl_distill_step(C.byref(lg.c), C.byref(t), T, w, loss, out, stride, sc, n, hip.stream) == 0
    hip.sync()
    hip.get(stats, np.float32, (R, 5))
    res = []
    for l, o, s in ((loss, out, stride), (loss2, out2, lg.vocab + pad)):
        raw = hip.get(o, bits, (R, s))
        assert in_place or (raw[:, lg.vocab:] == 0x1234).all(), "written between the rows"
        res += [hip.get(l, np.float32, R), rows64.from_bits(np.ascontiguousarray(raw[:, :lg.vocab]), lg.dtype)]
    return res


def check_distill(hip, lg, ids, v, T, rest, weights, wide=True, step=1, **kw):
    print(f"distill {lg.rows} x {lg.vocab} {lg.dtype} k {ids.shape[1]} T {T} rest {rest}", flush=True)
    loss, grad, loss2, grad2 = run_distill(hip, lg, ids, v, T, rest, weights, wide, **kw)
    for i in range(0, lg.rows, step):
        w = float(np.float32(weights[i]))
        want, tol, dz, dtol = rows64.distill(lg.z[i], ids[i], v[i].astype(np.float32), T, rest, w, lg.dtype)
        near(loss[i], want, tol, f"loss of row {i}")
        near(grad[i], dz, dtol, f"gradient of row {i}")
        near(grad2[i], dz, dtol, f"backward of row {i}")
        want, tol, _, _ = rows64.distill(lg.z[i], ids[i], v[i].astype(np.float32), T, rest, 1.0, lg.dtype)
        near(loss2[i], want, tol, f"loss of row {i} alone")
    return loss, grad


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (1, 2, 1), (3, 7, 4), (2, 2048, 256), (3, 2049, 17), (5, 32003, 20),
                                          (2, 151936, 100), (1, 1 << 18, 256), (258, 4099, 31), (20, 13001, 9),
                                          (3, 30011, 64), (160, 60003, 12), (160, 151937, 40)])
def test_distillation(hip, rows, vocab, k, dtype, rest):
    rng = np.random.default_rng(vocab + k)
    z = make(rng, rows, vocab)
    lg = Logits(hip, z, dtype, pad=2)
    ids, v = make_teacher(rng, lg.z, k)
    w = rng.uniform(-1, 2, rows).astype(np.float32)
    check_distill(hip, lg, ids, v, 2.0, rest, w, wide=bool(k % 2), step=1 if rows < 10 else rows // 4, pad=1,
                  offset=2 * DTYPES[dtype][1])


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", ["masked", "equal", "lowest", "lowest_mask", "few", "sure", "mixed"])
@pytest.mark.parametrize("rows,vocab", [(6, 71001), (261, 2311)])
def test_distillation_of_logits_that_go_wrong(hip, rows, vocab, kind, dtype, rest):
    rng = np.random.default_rng(len(kind) + 1)
    k = 12
    z = make(rng, rows, vocab, kind)
    if dtype == "f16":
        z = np.where(np.isfinite(z), np.clip(z, -65504.0, 65504.0), z).astype(np.float32)
    lg = Logits(hip, z, dtype)
    ids, v = make_teacher(rng, lg.z, k)
    if kind in ("masked", "few"):  # the teacher keeps to what is unmasked, but for the last row
        on = np.isfinite(np.take_along_axis(lg.z, ids, 1))
        on[-1] = True
        v = np.where(on, v, -np.inf).astype(np.float32)
    w = rng.uniform(0.1, 2, rows).astype(np.float32)
    w[4] = 0.0
    check_distill(hip, lg, ids, v, 1.0, rest, w, step=1 if rows < 10 else 29)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,vocab", [(9, 70000), (270, 1500)])
def test_teachers_that_go_wrong(hip, rows, vocab, rest):
    """Empty slots and rows, ids twice, ids outside, broken log probabilities, lists of the whole vocabulary."""
    rng = np.random.default_rng(3)
    k = 40
    z = make(rng, rows, vocab)
    z[8] = np.nan  # an empty list: not looked at
    lg = Logits(hip, z, "f32")
    ids, v = make_teacher(rng, np.nan_to_num(lg.z), k)
    ids[0, ::2] = -1
    v[1, 1::3] = -np.inf
    ids[2] = -7
    ids[3, :20] = ids[3, 20:]          # every one twice
    ids[4, 5] = vocab                  # outside
    v[5, 7] = np.nan
    v[6, 39] = np.inf
    v[7] = v[7] + 5                    # more than all of the mass: nothing is left outside
    ids[8] = -1
    w = np.ones(rows, np.float32)
    loss, grad = check_distill(hip, lg, ids, v, 1.5, rest, w, step=1)
    assert np.isnan(loss[[4, 5, 6]]).all() and np.isnan(grad[[4, 5, 6]]).all()
    assert loss[2] == 0 and loss[8] == 0 and not grad[[2, 8]].any()
    # a list of the whole vocabulary leaves nothing outside
    lg = Logits(hip, make(rng, 3, 200), "bf16")
    ids = np.stack([rng.permutation(200) for _ in range(3)])
    _, v = make_teacher(rng, lg.z, 200)
    check_distill(hip, lg, ids, v, 1.0, rest, [1.0, 0.5, 1.0])


@pytest.mark.parametrize("rows,vocab", [(3, 70100), (280, 4100), (165, 50001), (161, 152001)])
def test_distillation_in_place_and_by_rows(hip, rows, vocab):
    """The gradient over the logits themselves, and the same bits for rows alone as among others."""
    rng = np.random.default_rng(4)
    k = 33
    z = make(rng, rows, vocab)
    ids, v = make_teacher(rng, z, k)
    w = rng.uniform(0, 1, rows).astype(np.float32)
    for dtype in DTYPES if vocab < 100000 else ("bf16",):
        for rest in (False, True):
            want = run_distill(hip, Logits(hip, z, dtype, pad=1), ids, v, 1.0, rest, w)
            got = run_distill(hip, Logits(hip, z, dtype, pad=1), ids, v, 1.0, rest, w, in_place=True)
            alone = run_distill(hip, Logits(hip, z[1:2], dtype), ids[1:2], v[1:2], 1.0, rest, w[1:2])
            for a, b, c in zip(want, got, alone):
                assert np.array_equal(a, b)
                assert np.array_equal(a[1:2], c)
            assert np.array_equal(want[1], want[3])  # the step's gradient and the backward's


# ---- together, on streams, in graphs ------------------------------------------------


def test_a_teachers_scores_into_a_students_step_in_a_graph(hip):
    """Alternatives of one model straight into the other's loss and gradient, captured and replayed."""
    from detllm_amd._lib import Teacher

    rng = np.random.default_rng(12)
    rows, vocab, k, T = 6, 68001, 24, 2.0
    zt, zs = make(rng, rows, vocab), make(rng, rows, vocab)
    teacher, student = Logits(hip, zt, "f32"), Logits(hip, zs, "bf16")
    f = lambda *s: hip.put(np.zeros(s, np.float32))
    ids, lps, loss = hip.put(np.zeros((rows, k), np.int32)), f(rows, k), f(rows)
    grad = hip.put(np.zeros((rows, vocab), np.uint16))
    s1, n1 = scratch(hip, hip.dtl.dtl_token_scores_scratch(rows, vocab, k))
    s2, n2 = scratch(hip, hip.dtl.dtl_distill_scratch(rows, vocab))
    t = Teacher(ids, 4, lps, k, 1)

    def both(stream):
        assert hip.dtl.dtl_token_scores(C.byref(teacher.c), None, 0, T, k, None, None, None, ids, lps, s1, n1, stream) == 0
        assert hip.dtl.dtl_distill_step(C.byref(student.c), C.byref(t), T, None, loss, grad, vocab, s2, n2, stream) == 0

    graph, exe = C.c_void_p(), C.c_void_p()
    print("scores and distillation under graph capture", flush=True)
    assert hip.rt.hipStreamBeginCapture(hip.stream, 0) == 0
    try:
        both(hip.stream)
    finally:
        assert hip.rt.hipStreamEndCapture(hip.stream, C.byref(graph)) == 0
    assert hip.rt.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    try:
        for replay in range(3):
            zt, zs = make(rng, rows, vocab), make(rng, rows, vocab)
            hip.fill(teacher.addr, rows64.to_bits(zt, "f32"))
            hip.fill(student.addr, rows64.to_bits(zs, "bf16"))
            z = rows64.from_bits(rows64.to_bits(zs, "bf16"), "bf16")
            print(f"graph replay {replay}", flush=True)
            assert hip.rt.hipGraphLaunch(exe, hip.stream) == 0
            hip.sync()
            got = [hip.get(loss, np.float32, rows), hip.get(grad, np.uint16, (rows, vocab)), hip.get(ids, np.int32, (rows, k))]
            both(hip.stream)
            hip.sync()
            assert np.array_equal(got[0], hip.get(loss, np.float32, rows))
            assert np.array_equal(got[1], hip.get(grad, np.uint16, (rows, vocab)))
            v = hip.get(lps, np.float32, (rows, k))
            for i in range(rows):
                want, _ = rows64.top(zt[i].astype(np.float64), k, T)
                assert got[2][i].tolist() == want.tolist()
                want, tol, dz, dtol = rows64.distill(z[i], got[2][i], v[i], T, True, 1.0, "bf16")
                near(got[0][i], want, tol, f"loss of row {i}")
                near(rows64.from_bits(got[1][i], "bf16"), dz, dtol, f"gradient of row {i}")
    finally:
        hip.rt.hipGraphExecDestroy(exe)
        hip.rt.hipGraphDestroy(graph)


# ---- a session's own logits -----------------------------------------------------------


def test_session_scores_and_a_texts():
    from detllm_amd import synth
    from detllm_amd._lib import DetllmError
    from detllm_amd.model import F32Llama

    w = synth.WORKLOADS["tiny"]
    toks = [int(t) for t in synth.tokens(w)]
    model = F32Llama.from_gguf(synth.build_model(w))
    rows = []
    model.visit_logits_for_tokens_chunked(toks, 3, lambda r: rows.append(r.copy()))
    z = np.stack(rows).astype(np.float64)
    got = model.scores_for_tokens_chunked(toks, 3, top=5, temperature=1.5)
    for i in range(len(toks)):
        y = toks[i + 1] if i + 1 < len(toks) else -1
        lp, tol, h, tol_h = rows64.scores(z[i], y, 1.5)
        near(got.log_probs[i], lp, tol, "log_prob")
        near(got.entropy[i], h, tol_h, "entropy")
        ids, _ = rows64.top(z[i], 5, 1.5)
        assert got.top_ids[i].tolist() == ids.tolist()
    with model.forward_workspace(len(toks), len(toks)) as s:
        with pytest.raises(DetllmError):  # no forward yet
            s.token_scores([1])
        s.forward_chunk(toks, 0)
        a = s.token_scores(toks[1:4], first=1, top=3, temperature=1.5)
        b = s.token_scores(toks[1:], top=128, temperature=1.5)  # grows the session's memory
        assert np.array_equal(b.log_probs, got.log_probs[:-1])
        assert np.array_equal(a.entropy, got.entropy[1:4]) and np.array_equal(a.top_ids, got.top_ids[1:4, :3])
        # the ranges that a codec would code are what they were
        c0 = s.symbol_ranges(toks[1:], 0, 256)
        s.token_scores(toks[1:], top=4)
        c1 = s.symbol_ranges(toks[1:], 0, 256)
        assert all(np.array_equal(x, y) for x, y in zip(c0, c1))
        for bad, status in (((len(toks) * [1], 1), 1), (([w.vocab], 0), 23)):
            with pytest.raises(DetllmError) as e:
                s.token_scores(bad[0], first=bad[1])
            assert e.value.status == status
        for kw, status in ((dict(top=129), 1), (dict(temperature=0.0), 42), (dict(temperature=float("nan")), 42)):
            with pytest.raises(DetllmError) as e:
                s.token_scores([1], **kw)
            assert e.value.status == status
