"""Where the gradients of scores and distillation may lie, through the C ABI."""
import ctypes as C

import numpy as np
import pytest

import rows64
from rows64 import DTYPES
from test_gpu_scores import Logits, _free, hip, make, make_teacher, pick_tokens, run_distill, run_scores, run_scores_grad, scratch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", [(3, 70001), (140, 2100)])
def test_gradients_between_the_rows_of_the_logits(hip, rows, vocab, dtype):
    """One matrix holds both: logits in its left half, the gradient in its right one."""
    from detllm_amd._lib import Logits as L, Teacher

    rng = np.random.default_rng(41)
    z = make(rng, rows, vocab)
    kind, size, _ = DTYPES[dtype]
    tokens, (ids, v) = pick_tokens(rng, z), make_teacher(rng, z, 9)
    w = rng.uniform(0.5, 1, rows).astype(np.float32)
    apart = Logits(hip, z, dtype)
    got = run_scores(hip, apart, tokens, 1.0, 0)
    want = run_scores_grad(hip, apart, got, 1.0, w, w), *run_distill(hip, apart, ids, v, 1.0, True, w)

    bits = rows64.to_bits(z, dtype)
    stride = 2 * vocab + 1
    both = np.full((rows, stride), 0x1234, bits.dtype)
    both[:, :vocab] = bits
    addr = hip.put(both)
    lg = L(addr, kind, rows, vocab, stride)
    right = addr + vocab * size
    dw, dv, dids = hip.put(w), hip.put(v), hip.put(ids.astype(np.int64))
    t = Teacher(dids, 8, dv, ids.shape[1], 1)
    loss, stats = hip.put(np.zeros(rows, np.float32)), hip.put(np.zeros((rows, 5), np.float32))
    sc, n = scratch(hip, hip.dtl.dtl_distill_scratch(rows, vocab))

    def gradient():
        hip.sync()
        raw = hip.get(addr, bits.dtype, (rows, stride))
        assert np.array_equal(raw[:, :vocab], bits) and (raw[:, -1] == 0x1234).all()
        return rows64.from_bits(np.ascontiguousarray(raw[:, vocab:-1]), dtype)

    assert hip.dtl.dtl_token_scores_backward(C.byref(lg), got["dev"]["tok"], 8, 1.0, got["dev"]["st"], got["dev"]["en"], dw,
                                             dw, right, stride, hip.stream) == 0
    assert np.array_equal(gradient(), want[0])
    assert hip.dtl.dtl_distill_step(C.byref(lg), C.byref(t), 1.0, dw, loss, right, stride, sc, n, hip.stream) == 0
    assert np.array_equal(gradient(), want[2]) and np.array_equal(hip.get(loss, np.float32, rows), want[1])
    assert hip.dtl.dtl_distill(C.byref(lg), C.byref(t), 1.0, loss, stats, sc, n, hip.stream) == 0
    assert hip.dtl.dtl_distill_backward(C.byref(lg), C.byref(t), 1.0, stats, dw, right, stride, hip.stream) == 0
    assert np.array_equal(gradient(), want[4]) and np.array_equal(hip.get(loss, np.float32, rows), want[3])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,vocab", [(129, 152001), (140, 66001), (5, 60001), (130, 33001), (3, 9001)])
def test_steps_in_place(hip, rows, vocab, dtype, rest):
    """Every shape of the step, its gradient over the logits: of rows held whole, held in part, in parts."""
    rng = np.random.default_rng(42)
    z = make(rng, rows, vocab)
    ids, v = make_teacher(rng, z, 25)
    w = rng.uniform(0.5, 1, rows).astype(np.float32)
    want = run_distill(hip, Logits(hip, z, dtype, pad=1), ids, v, 0.5, rest, w)
    got = run_distill(hip, Logits(hip, z, dtype, pad=1), ids, v, 0.5, rest, w, in_place=True)
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    assert np.array_equal(want[1], want[3])
