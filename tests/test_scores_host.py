"""What dtl_token_scores* and dtl_distill* refuse (found on the host before
anything is enqueued, so without a GPU), their oracle's gradients against
differences, and the rules that their device code keeps."""
import ctypes as C
import re
import subprocess

import numpy as np
import pytest

import rows64
from detllm_amd import build as B

OK, SHAPE, EMPTY, MANY, INVALID, SMALL = 0, 1, 20, 24, 42, 44
P = 1 << 20  # an address that is never read


def _calls(z, ids=P, id_bytes=4, v=P, k=4, T=1.0, tokens=P, token_bytes=8, top=2, out=P, stride=None, scratch=P, n=1 << 30):
    """The status of each entry point for these arguments (all refuse, or have no rows)."""
    from detllm_amd._lib import Teacher, lib

    t = Teacher(ids, id_bytes, v, k, 0)
    stride = z.vocab if stride is None else stride
    z = C.byref(z)
    return {
        "scores": lambda: lib.dtl_token_scores(z, tokens, token_bytes, T, top, out, out, out, out, out, scratch, n, None),
        "scores_backward": lambda: lib.dtl_token_scores_backward(z, tokens, token_bytes, T, out, out, out, out, out, stride, None),
        "distill": lambda: lib.dtl_distill(z, C.byref(t), T, out, out, scratch, n, None),
        "distill_backward": lambda: lib.dtl_distill_backward(z, C.byref(t), T, out, out, out, stride, None),
        "distill_step": lambda: lib.dtl_distill_step(z, C.byref(t), T, None, out, out, stride, scratch, n, None),
    }


ALL = ("scores", "scores_backward", "distill", "distill_backward", "distill_step")


def _view(data=P, dtype=0, rows=3, vocab=100, stride=100):
    from detllm_amd._lib import Logits

    return Logits(data, dtype, rows, vocab, stride)


def _expect(status, names, z, **kw):
    calls = _calls(z, **kw)
    for name in names:
        assert calls[name]() == status, (name, status, kw)


def test_refusals():
    for dtype in (-1, 3):
        _expect(INVALID, ALL, _view(dtype=dtype))
    _expect(EMPTY, ALL, _view(vocab=0))
    _expect(MANY, ALL, _view(vocab=(1 << 18) + 1, stride=1 << 19))
    _expect(SHAPE, ALL, _view(stride=99))
    _expect(SHAPE, ALL, _view(rows=(1 << 24) + 1))
    _expect(SHAPE, ALL, _view(stride=1 << 48))
    _expect(INVALID, ALL, _view(data=0))
    _expect(INVALID, ALL, _view(data=P + 2))
    _expect(INVALID, ALL, _view(data=P + 1, dtype=1))
    for T in (0.0, -1.0, 1e-5, 2e4, float("inf"), float("nan")):
        _expect(INVALID, ALL, _view(), T=T)
    grads = ("scores_backward", "distill_backward", "distill_step")
    _expect(SHAPE, grads, _view(), stride=99)
    _expect(INVALID, grads, _view(), out=0)
    _expect(INVALID, grads, _view(dtype=2), out=P + 1)
    for n in (0, 2, 16):
        _expect(INVALID, ("scores", "scores_backward"), _view(), token_bytes=n)
        _expect(INVALID, ALL[2:], _view(), id_bytes=n)
    _expect(INVALID, ("scores", "scores_backward"), _view(), tokens=0)  # log probabilities of no tokens
    _expect(SHAPE, ("scores",), _view(vocab=500, stride=500), top=129)
    _expect(SHAPE, ("scores",), _view(), top=101)
    for k in (0, 257):
        _expect(SHAPE, ALL[2:], _view(), k=k)
    _expect(INVALID, ALL[2:], _view(), ids=0)
    _expect(INVALID, ALL[2:], _view(), v=0)
    scratch = ("scores", "distill", "distill_step")
    long = _view(vocab=100000, stride=100000)
    _expect(SMALL, scratch, long, n=8)
    _expect(INVALID, scratch, long, scratch=0)
    _expect(INVALID, scratch, long, scratch=P + 8)


def test_missing_outputs_and_structs():
    from detllm_amd._lib import lib

    z = _view()
    assert lib.dtl_token_scores(None, P, 8, 1.0, 0, P, P, P, None, None, P, 1 << 20, None) == INVALID
    assert lib.dtl_token_scores(C.byref(z), P, 8, 1.0, 2, P, P, P, None, P, P, 1 << 20, None) == INVALID
    assert lib.dtl_token_scores(C.byref(z), P, 8, 1.0, 2, P, P, P, P, None, P, 1 << 20, None) == INVALID
    assert lib.dtl_token_scores_backward(C.byref(z), P, 8, 1.0, None, P, P, P, P, 100, None) == INVALID
    assert lib.dtl_token_scores_backward(C.byref(z), P, 8, 1.0, P, None, P, P, P, 100, None) == INVALID
    assert lib.dtl_distill(C.byref(z), None, 1.0, P, P, P, 1 << 20, None) == INVALID
    assert lib.dtl_session_token_scores(None, 0, 1, None, 1.0, 0, None, None, None, None) == INVALID


def test_no_rows_are_no_error():
    for data in (0, P):
        calls = _calls(_view(data=data, rows=0), ids=0, v=0, tokens=0, out=0, scratch=0, n=0)
        for name in ALL:
            assert calls[name]() == OK, name


def test_scratch_sizes():
    from detllm_amd._lib import lib

    for rows, vocab, top in ((1, 100000, 0), (8, 151936, 20), (100, 1 << 18, 128)):
        seg = -(-vocab // 2048)
        assert lib.dtl_token_scores_scratch(rows, vocab, top) >= rows * seg * (12 + (256 if top else 0))
        assert lib.dtl_distill_scratch(rows, vocab) >= rows * seg * 12 + rows * 20
    for rows, vocab in ((1, 1), (1, 32000), (4096, 151936)):
        assert lib.dtl_token_scores_scratch(rows, vocab, 1) == 0 == lib.dtl_distill_scratch(rows, vocab)


def test_oracle_gradients_against_differences():
    rng = np.random.default_rng(1)
    z = rng.normal(0, 2, 40)
    z[3] = z[17] = -np.inf
    on = np.isfinite(z)
    ids = np.array([0, 5, 5, 39, -1, 8])
    v = np.log(np.array([0.3, 0.1, 0.2, 0.1, 0.4, 0.05])).astype(np.float32)
    T, d = 0.75, 1e-5

    def slopes(f):
        out = np.zeros(z.size)
        for j in np.flatnonzero(on):
            a, b = z.copy(), z.copy()
            a[j] += d
            b[j] -= d
            out[j] = (f(a) - f(b)) / (2 * d)
        return out

    for tok in (5, -1):
        got, _ = rows64.scores_grad(z, tok, T, 1.25, -0.5, 0.0, "f32")
        want = slopes(lambda x: (1.25 * rows64.scores(x, tok, T)[0] if tok >= 0 else 0.0) - 0.5 * rows64.scores(x, tok, T)[2])
        assert np.abs(got - want).max() < 1e-8
    for rest in (False, True):
        got = rows64.distill(z, ids, v, T, rest, 0.7, "f32")[2]
        want = slopes(lambda x: rows64.distill(x, ids, v, T, rest, 0.7, "f32")[0])
        assert np.abs(got - want).max() < 1e-8


def test_oracle_scores_against_plain_sums():
    z = np.array([1.0, -2.0, 0.5, 0.5])
    p = np.exp(z / 2) / np.exp(z / 2).sum()
    lp, _, h, _ = rows64.scores(z, 2, 2.0)
    assert abs(lp - np.log(p[2])) < 1e-15 and abs(h + (p * np.log(p)).sum()) < 1e-15
    assert rows64.top(z, 3, 2.0)[0].tolist() == [0, 2, 3]


@pytest.fixture(scope="module")
def device_asm(tmp_path_factory):
    out = tmp_path_factory.mktemp("scores") / "scores.s"
    subprocess.run([B.hipcc(), f"--offload-arch={B.ARCH}", "-O3", "-std=c++17", *B.NUMERIC_FLAGS, "--cuda-device-only",
                    "-Wno-unused-result", "-S", str(B.SCORES_SRC / "dtl_scores.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    return out.read_text()


def test_device_code_keeps_its_rules(device_asm):
    """No packed float32, no write through the scalar cache, nothing spilled to
    memory, 16-byte loads and stores of the logits."""
    assert re.search(r"^\s*v_pk_(?:add|mul|fma|mov)_f32", device_asm, re.M) is None
    assert re.search(r"^\s*s_(?:store|buffer_store|atomic|dcache_(?:wb|discard))", device_asm, re.M) is None
    assert set(re.findall(r"\.vgpr_spill_count: (\d+)", device_asm)) == {"0"}
    assert "global_load_dwordx4" in device_asm and "global_store_dwordx4" in device_asm
    assert "v_exp_f32" in device_asm


def test_the_references_arithmetic_stays_apart():
    """csrc, whose rules the numeric contract checks, takes nothing of the
    scores' arithmetic but their launches."""
    for path in sorted(B.CSRC.iterdir()):
        for inc in re.findall(r'#include "(\.\./csrc_scores/[^"]+)"', path.read_text()):
            assert inc == "../csrc_scores/dtl_scores.h" and path.name == "dtl_api.hip"
