"""What dtl_embedding*, dtl_grad_norm and dtl_clip_grads refuse (found on the host
before anything is enqueued, so without a GPU), their oracles by hand and against
differences, and the rules that their device code keeps."""
import ctypes as C
import re
import subprocess
from array import array

import numpy as np
import pytest

import train64
from detllm_amd import build as B

OK, SHAPE, EMPTY, MANY, MEMORY, INVALID, SMALL = 0, 1, 20, 24, 41, 42, 44
P, Q, G = 1 << 20, 1 << 30, 1 << 34  # addresses that are never read, far apart
MUCH = 1 << 40


def table(**kw):
    from detllm_amd._lib import Table

    return Table(**{**dict(data=P, dtype=0, vocab=50, width=8, stride=8), **kw})


def lookup(t, tokens=Q, token_bytes=8, n=10, out=G, out_stride=8):
    from detllm_amd._lib import lib

    return lib.dtl_embedding(None if t is None else C.byref(t), tokens, token_bytes, n, 1.0, out, out_stride, None)


def gradient(t, tokens=Q, token_bytes=8, n=10, grad=G, dtype=0, stride=8, add=0, scratch=1 << 36, scratch_bytes=MUCH):
    from detllm_amd._lib import lib

    return lib.dtl_embedding_backward(tokens, token_bytes, n, grad, dtype, stride, 1.0, None if t is None else C.byref(t),
                                      add, scratch, scratch_bytes, None)


def test_tables_and_tokens():
    for bad, status in ((None, INVALID), (table(dtype=3), INVALID), (table(data=0), INVALID), (table(data=P + 2), INVALID),
                        (table(data=P + 1, dtype=1), INVALID), (table(vocab=0), EMPTY), (table(vocab=(1 << 18) + 1), MANY),
                        (table(width=0), SHAPE), (table(width=(1 << 16) + 1, stride=1 << 17), SHAPE), (table(stride=7), SHAPE),
                        (table(stride=1 << 47), SHAPE)):
        assert lookup(bad) == status == gradient(bad)
    for kw, status in ((dict(tokens=0), INVALID), (dict(token_bytes=2), INVALID)):
        assert lookup(table(), **kw) == status == gradient(table(), **kw)
    assert lookup(table(), n=(1 << 24) + 1) == SHAPE == gradient(table(), n=(1 << 20) + 1)
    assert lookup(table(), out=0) == INVALID == gradient(table(), grad=0)
    assert lookup(table(), out=G + 2) == INVALID == gradient(table(), grad=G + 2)
    assert lookup(table(), out_stride=7) == SHAPE == gradient(table(), stride=7)
    assert lookup(table(), out=P + 32) == INVALID == gradient(table(), grad=P + 32)  # one over a part of the other
    assert lookup(table(), out=P - 10 * 32 + 4) == INVALID == gradient(table(), grad=P - 10 * 32 + 4)
    for dtype, of in ((1, 2), (2, 1), (0, 1), (0, 2), (3, 0)):
        assert gradient(table(dtype=of), dtype=dtype) == INVALID
    assert gradient(table(), scratch=0) == INVALID == gradient(table(), scratch=P + 8)
    assert gradient(table(), scratch_bytes=64) == SMALL
    assert lookup(table(), n=0, tokens=0, out=0) == OK == gradient(table(), n=0, tokens=0, grad=0, add=1)


def test_embedding_scratch():
    from detllm_amd._lib import lib

    f = lib.dtl_embedding_backward_scratch
    for n, width in ((1, 1), (1000, 896), (65536, 2048), (1 << 20, 8), (5000, 65536)):
        assert f(n, 1000, width) >= 16 * n + n // 16384 * 2 * width * 4
        assert f(n, 5, width) <= 256 + 16 * (n + 1024) + 128 * 512 * 4 + (n // 8 + 1) * 2 * (width + 8) * 4
    assert f((1 << 20) + 1, 10, 8) == 0


def tensors(*entries):
    return array("Q", [v for e in entries for v in e])


def clip(t, n=None, out=None, max_norm=1.0, norm=P, scratch=1 << 36, scratch_bytes=MUCH, names=("norm", "clip")):
    from detllm_amd._lib import lib

    at, n = t.buffer_info()[0], len(t) // 3 if n is None else n
    got = []
    if "norm" in names:
        got.append(lib.dtl_grad_norm(at, n, 0, 1.0, None, norm, scratch, scratch_bytes, None))
    if "clip" in names:
        to = None if out is None else out.buffer_info()[0]
        got.append(lib.dtl_clip_grads(at, n, 0, 1.0, None, max_norm, to, norm, scratch, scratch_bytes, None))
    assert len(set(got)) == 1, got
    return got[0]


def test_tensor_lists():
    good = (G, 100, 0)
    for bad, status in (((G, 100, 3), INVALID), ((0, 100, 0), INVALID), ((G + 2, 100, 0), INVALID), ((G + 1, 100, 1), INVALID),
                        ((G, (1 << 36) + 1, 0), SHAPE)):
        assert clip(tensors((Q, 5, 0), bad)) == status
    assert clip(tensors(good), n=(1 << 16) + 1) == SHAPE
    assert clip(tensors(good), norm=0) == INVALID
    assert clip(tensors(good), scratch=0) == INVALID == clip(tensors(good), scratch=P + 8)
    assert clip(tensors(good), scratch_bytes=16) == SMALL
    only = ("clip",)
    for max_norm in (-1.0, float("nan")):
        assert clip(tensors(good), max_norm=max_norm, names=only) == INVALID
    for out, status in (((Q, 99, 0), SHAPE), ((Q, 100, 1), INVALID), ((0, 100, 0), INVALID), ((G + 4, 100, 0), INVALID),
                        ((G - 400 + 4, 100, 0), INVALID)):
        assert clip(tensors(good), out=tensors(out), names=only) == status, out
    a, b = (G, 100, 1), (G + 200, 100, 1)
    for grads, out in (((a, a), None), ((a, (G + 198, 100, 1)), None),
                       ((a, b), (b, a)), ((a, b), ((Q, 100, 1), (Q + 100, 100, 1))),
                       ((a, b), ((G, 100, 0), (Q, 100, 0)))):  # wider, over itself
        assert clip(tensors(*grads), out=None if out is None else tensors(*out), names=only) == INVALID


def test_norm_scratch():
    from detllm_amd._lib import lib

    t = tensors((G, 1 << 30, 0), (Q, 0, 1), (Q, 1, 2))
    assert lib.dtl_grad_norm_scratch(t.buffer_info()[0], 3) >= ((1 << 30) // 65536) * 8
    assert lib.dtl_grad_norm_scratch(tensors((G, 1 << 37, 0)).buffer_info()[0], 1) == 0
    assert lib.dtl_grad_norm_scratch(None, 0) >= 4


def test_oracles():
    rows, _ = train64.embedding([[1.0, 2.0], [3.0, 4.0]], [1, -1, 2], 2.0, "f32")
    assert rows[0].tolist() == [6.0, 8.0] and rows[1].tolist() == [0.0, 0.0] and np.isnan(rows[2]).all()
    tokens, g = np.array([1, 3, -1, 1, 9]), np.arange(10.0).reshape(5, 2)
    want, _ = train64.gradient(tokens, g, 4, 0.5, "f32")
    assert want.tolist() == [[0, 0], [3.0, 4.0], [0, 0], [1.0, 1.5]]
    # against differences of sum(g * embedding(w))
    w, d = np.random.default_rng(1).normal(size=(4, 2)), 1e-6
    real = tokens < 4
    for v in range(4):
        for j in range(2):
            a, b = w.copy(), w.copy()
            a[v, j] += d
            b[v, j] -= d
            f = [(g[real] * train64.embedding(x, tokens[real], 0.5, "f32")[0]).sum() for x in (a, b)]
            assert abs((f[0] - f[1]) / (2 * d) - want[v, j]) < 1e-6
    assert train64.norm([[3.0], [[4.0, -12.0]]])[0] == 13.0 and train64.norm([[3.0], [-4.0]], -2.0, True)[0] == 8.0
    assert abs(train64.clipped([2.0], 4.0, 1.0, 1.0, "f32")[0][0] - 0.5) < 1e-6 and train64.clipped([2.0], 0.5, 1.0, 1.0, "f32")[0] == 2.0


@pytest.mark.parametrize("name", ["dtl_embedding.hip", "dtl_clip.hip"])
def test_device_code_keeps_its_rules(name, tmp_path):
    """No packed float32, no write through the scalar cache, nothing spilled to
    memory, 16-byte loads and stores."""
    out = tmp_path / "device.s"
    subprocess.run([B.hipcc(), f"--offload-arch={B.ARCH}", "-O3", "-std=c++17", *B.NUMERIC_FLAGS, "--cuda-device-only",
                    "-Wno-unused-result", "-S", str(B.SCORES_SRC / name), "-o", str(out)], check=True, capture_output=True)
    asm = out.read_text()
    assert re.search(r"^\s*v_pk_(?:add|mul|fma|mov)_f32", asm, re.M) is None
    assert re.search(r"^\s*s_(?:store|buffer_store|atomic|dcache_(?:wb|discard))", asm, re.M) is None
    assert set(re.findall(r"\.vgpr_spill_count: (\d+)", asm)) == {"0"}
    assert set(re.findall(r"\.private_segment_fixed_size: (\d+)", asm)) == {"0"}
    assert "global_load_dwordx4" in asm and "global_store_dwordx4" in asm
