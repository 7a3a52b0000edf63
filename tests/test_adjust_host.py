"""What dtl_adjust_logits* refuse (found on the host before anything is enqueued, so
without a GPU), their oracle's gradient against differences, and the rules that
their device code keeps."""
import ctypes as C
import re
import subprocess

import numpy as np
import pytest

import adjust64
from detllm_amd import build as B

OK, SHAPE, EMPTY, MANY, INVALID = 0, 1, 20, 24, 42
P, Q, G = 1 << 20, 1 << 30, 1 << 34  # addresses that are never read, far apart


def _by(**kw):
    from detllm_amd._lib import Adjust

    full = dict(history=Q, history_bytes=8, history_len=5, history_stride=5, repetition=1.5, presence=0.0, frequency=0.0,
                bias_ids=Q, bias_bytes=4, biases=Q, bias_len=3, bias_stride=0, allowed=Q, allowed_bits=1, allowed_stride=4)
    return Adjust(**{**full, **kw})


def _status(z, by, out=G, stride=None, grad_out=P << 8, names=("forward", "backward")):
    from detllm_amd._lib import lib

    stride = z.vocab if stride is None else stride
    by = None if by is None else C.byref(by)
    got = []
    if "forward" in names:
        got.append(lib.dtl_adjust_logits(C.byref(z), by, out, stride, None))
    if "backward" in names:
        got.append(lib.dtl_adjust_logits_backward(C.byref(z), by, grad_out, z.vocab, out, stride, None))
    assert len(set(got)) == 1, got
    return got[0]


def _view(data=P, dtype=0, rows=3, vocab=100, stride=100):
    from detllm_amd._lib import Logits

    return Logits(data, dtype, rows, vocab, stride)


def test_refusals():
    z = _view()
    for bad in (_view(dtype=3), _view(data=0), _view(data=P + 2)):
        assert _status(bad, _by()) == INVALID
    assert _status(_view(vocab=0), _by()) == EMPTY
    assert _status(_view(vocab=(1 << 18) + 1, stride=1 << 19), _by()) == MANY
    for bad in (_view(stride=99), _view(rows=(1 << 24) + 1)):
        assert _status(bad, _by()) == SHAPE
    assert _status(z, None) == INVALID
    for kw in (dict(history=0), dict(history_bytes=2), dict(repetition=0.0), dict(repetition=-2.0),
               dict(repetition=float("inf")), dict(repetition=float("nan")), dict(presence=float("nan")),
               dict(frequency=float("inf")), dict(bias_ids=0), dict(biases=0), dict(bias_bytes=1), dict(allowed_bits=2),
               dict(allowed=Q + 2)):
        assert _status(z, _by(**kw)) == INVALID, kw
    for kw in (dict(history_len=(1 << 17) + 1), dict(history_stride=1 << 41), dict(bias_len=4097), dict(bias_stride=1 << 41),
               dict(allowed_stride=3), dict(allowed_stride=1 << 41), dict(allowed_bits=8, allowed_stride=99)):
        assert _status(z, _by(**kw)) == SHAPE, kw
    assert _status(z, _by(), out=0) == INVALID
    assert _status(z, _by(), out=G + 2) == INVALID
    assert _status(z, _by(), stride=99) == SHAPE
    # over a part of the logits; the gradient over the logits, or over a part of the one it is formed from
    assert _status(z, _by(), out=P + 400) == INVALID
    assert _status(z, _by(), out=P, stride=101, names=("forward",)) == INVALID
    assert _status(z, _by(), out=P, names=("backward",)) == INVALID
    assert _status(z, _by(), out=(P << 8) + 4, names=("backward",)) == INVALID
    assert _status(z, _by(), grad_out=0, names=("backward",)) == INVALID


def test_no_rows_are_no_error():
    for data in (0, P):
        assert _status(_view(data=data, rows=0), _by(), out=0, grad_out=0) == OK
        assert _status(_view(data=data, rows=0), _by(history=0, bias_ids=0, biases=0, allowed=0), out=0, grad_out=0) == OK


def test_oracle_gradient_against_differences():
    rng = np.random.default_rng(1)
    z = rng.normal(0, 2, 60)
    allowed = rng.random(60) < 0.7
    kw = dict(history=[3, 3, 7, -1, 60, 9, 11], theta=1.3, allowed=allowed)
    g, d = rng.normal(0, 1, 60), 1e-6

    def total(x):
        a, _ = adjust64.adjust(x, "f32", prompt=2, presence=0.5, frequency=0.25, bias_ids=[7, 7], bias=[1.0, -2.0], **kw)
        return (g[allowed] * a[allowed]).sum()

    want, _ = adjust64.gradient(z, g, "f32", **kw)
    for j in range(60):
        x = np.eye(60)[j] * d
        assert abs((total(z + x) - total(z - x)) / (2 * d) - want[j]) < 1e-7


def test_oracle_by_hand():
    a, _ = adjust64.adjust([2.0, -2.0, 1.0, 0.5, 3.0], "f32", history=[0, 1, 1, 1], prompt=2, theta=2.0, presence=0.5,
                           frequency=0.25, bias_ids=[2, 2, 9], bias=[8.0, 1.0, 5.0], allowed=np.array([1, 1, 1, 1, 0], bool))
    assert a.tolist() == [1.0, -4.0 - 0.5 - 0.5, 2.0, 0.5, -np.inf]


@pytest.fixture(scope="module")
def device_asm(tmp_path_factory):
    out = tmp_path_factory.mktemp("adjust") / "adjust.s"
    subprocess.run([B.hipcc(), f"--offload-arch={B.ARCH}", "-O3", "-std=c++17", *B.NUMERIC_FLAGS, "--cuda-device-only",
                    "-Wno-unused-result", "-S", str(B.SCORES_SRC / "dtl_adjust.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    return out.read_text()


def test_device_code_keeps_its_rules(device_asm):
    """No packed float32, no write through the scalar cache, nothing spilled to
    memory, 16-byte loads and stores of the logits."""
    assert re.search(r"^\s*v_pk_(?:add|mul|fma|mov)_f32", device_asm, re.M) is None
    assert re.search(r"^\s*s_(?:store|buffer_store|atomic|dcache_(?:wb|discard))", device_asm, re.M) is None
    assert set(re.findall(r"\.vgpr_spill_count: (\d+)", device_asm)) == {"0"}
    assert "global_load_dwordx4" in device_asm and "global_store_dwordx4" in device_asm
