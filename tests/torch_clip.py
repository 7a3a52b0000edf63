"""detllm_amd.train's gradient norm and clipping.  Run by test_gpu_train.py in a process
of its own, where torch's HIP runtime is the one the library takes."""
import math

import torch  # first: the library shares its HIP runtime

import numpy as np
import pytest

import train64
from adjust64 import same
from detllm_amd import train
from detllm_amd._lib import DetllmError

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NAME = {v: k for k, v in TYPES.items()}


def host(t):
    return t.detach().double().cpu().numpy()


def tensors(seed, sizes, dtypes, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(size * torch.randn(n, generator=g)).to(TYPES[d]).to(DEV) for n, d in zip(sizes, dtypes)]


def check(grads, got, max_norm, scale, outs, kind=2.0):
    want, tol = train64.norm([host(t) for t in grads], scale, kind == math.inf)
    assert same(host(got), want, tol)
    for t, o in zip(grads, outs):
        w, tol = train64.clipped(host(t), want, max_norm, scale, NAME[o.dtype])
        assert same(host(o), w, tol).all()


LISTS = [  # sizes
    [1], [7], [8, 1, 3], [0, 5, 0], [255, 256, 257], [32768], [32769, 32767, 3], [100003, 2, 70001],
    [17] * 400, [1000, 2000] * 100, [3_000_001],
]


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clipping(sizes, dtype, kind):
    kinds = [dtype if dtype != "mixed" else ("f16", "f32", "bf16")[i % 3] for i in range(len(sizes))]
    grads = tensors(len(sizes), sizes, kinds)
    for scale, max_norm in ((1.0, 0.5), (0.25, 1e6), (-2.0, 3.0)):
        norm = train.grad_norm(grads, norm_type=kind, scale=scale)
        check(grads, norm, max_norm, scale, [], kind)
        one = torch.tensor(scale, device=DEV)
        outs = [torch.full_like(t, 9.0) for t in grads]
        assert torch.equal(train.clip_grad_norm(grads, max_norm, norm_type=kind, scale=scale, out=outs), norm)
        check(grads, norm, max_norm, scale, outs, kind)
        wide = [torch.empty(t.shape, device=DEV) for t in grads]
        assert torch.equal(train.clip_grad_norm(grads, max_norm, norm_type=kind, scale=one, out=wide), norm)
        check(grads, norm, max_norm, scale, wide, kind)
        mine = [t.clone() for t in grads]
        assert torch.equal(train.clip_grad_norm(mine, max_norm, norm_type=kind, scale=scale), norm)
        assert all(torch.equal(a, b) for a, b in zip(mine, outs))


def test_pieces_of_one_buffer_not_aligned():
    """Tensors cut from one buffer at odd places: what lies between them stays."""
    for dtype in TYPES.values():
        flat = torch.randn(200_000, device=DEV).to(dtype)
        cuts = [(1, 30_000), (30_003, 30_004), (30_007, 130_000), (130_011, 199_999)]
        before = flat.clone()
        grads = [before[a:b] for a, b in cuts]
        mine = [flat[a:b] for a, b in cuts]
        norm = train.clip_grad_norm(mine, 2.0)
        check(grads, norm, 2.0, 1.0, mine)
        between = torch.ones(200_000, dtype=torch.bool, device=DEV)
        for a, b in cuts:
            between[a:b] = False
        assert torch.equal(flat[between], before[between])


def test_large_and_small_magnitudes():
    for size, n in ((1e30, 1000), (1e-30, 1000), (3e-44, 70000), (1e19, 3)):
        g = [torch.full((n,), size, device=DEV), torch.full((n,), size, device=DEV)]
        assert same(host(train.grad_norm(g)), *train64.norm([host(t) for t in g]))
        norm = train.clip_grad_norm(g, 1.0)
        if size > 1:
            assert abs(float(train.grad_norm(g)) - 1) < 1e-5 and float(norm) > 1
        else:
            assert (g[0] == size).all()


def test_infinities_and_no_numbers():
    for kind in (2.0, math.inf):
        for bad, dtype in ((math.inf, "f32"), (-math.inf, "bf16"), (math.nan, "f16"), (math.nan, "f32")):
            grads = tensors(3, [70000, 5, 300], [dtype] * 3)
            for at in ((0, 0), (0, 69999), (2, 299)):
                mine = [t.clone() for t in grads]
                mine[at[0]][at[1]] = bad
                norm = train.grad_norm(mine, norm_type=kind)
                assert norm.isnan() if math.isnan(bad) else norm == math.inf
                assert torch.equal(train.clip_grad_norm(mine, 1.0, norm_type=kind).nan_to_num(7.0), norm.nan_to_num(7.0))
                for i, t in enumerate(mine):
                    nan = t.isnan()
                    if math.isnan(bad):
                        assert nan.all()
                    else:
                        assert nan.sum() == (i == at[0]) and (t[~nan] == 0).all()


def test_lists_shapes_and_layouts():
    assert float(train.grad_norm([])) == 0.0 == float(train.clip_grad_norm([None], 1.0))
    a = torch.randn(30, 40, device=DEV)
    t = a.t()  # dense, in another order
    assert torch.equal(train.grad_norm(a), train.grad_norm([None, t]))
    want = a * (1.0 / (float(train.grad_norm(a)) + 1e-6))
    train.clip_grad_norm((x for x in (t, None)), 1.0)
    assert torch.allclose(a, want, rtol=1e-6)
    out = torch.empty(40, 30, device=DEV)
    with pytest.raises(ValueError):
        train.clip_grad_norm([t], 1.0, out=[out])  # other strides
    train.clip_grad_norm([t], 1.0, out=[torch.empty_like(t)])
    w = torch.randn(20, 30, device=DEV, requires_grad=True)
    (w * 3).square().sum().backward()
    before = w.grad.clone()
    norm = train.clip_grad_norm([w.grad], 1.0)
    check([before], norm, 1.0, 1.0, [w.grad])
    assert float(train.clip_grad_norm([w.grad.clone()], 0.0)) > 0


def test_in_a_graph():
    grads = tensors(5, [50_000, 3, 1000], ["bf16", "f32", "f16"])
    outs = [torch.empty(t.shape, device=DEV) for t in grads]

    def work():
        return train.grad_norm(grads, norm_type=math.inf), train.clip_grad_norm(grads, 1.0, out=outs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for i in range(3):
        for t in grads:
            t.copy_(torch.randn(t.shape, device=DEV) * (i + 0.5))
        want = [x.clone() for x in (*work(), *outs)]
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*got, *outs), want))


def test_on_two_streams():
    lists = [tensors(6 + i, [300_000, 17, 90_001], ["f32", "bf16", "f16"]) for i in range(2)]
    want = [train.grad_norm(g) for g in lists]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in lists], [[] for _ in lists]
    for _ in range(10):
        for g, s, o in zip(lists, streams, got):
            with torch.cuda.stream(s):
                o.append(train.grad_norm(g))
    torch.cuda.synchronize()
    assert all(torch.equal(w, x) for w, o in zip(want, got) for x in o)


def test_a_tensor_past_32_bits():
    n = (1 << 32) + 77
    t = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    t[-1], t[n // 2], t[5] = 3.0, 4.0, 12.0
    assert float(train.clip_grad_norm(t, 6.5)) == 13.0
    assert t[-1] == 1.5 and t[n // 2] == 2.0 and t[5] == 6.0 and int(torch.count_nonzero(t)) == 3


def test_refusals():
    a, b = torch.randn(10, device=DEV), torch.randn(10, device=DEV)
    for bad, err in (([a.double()], TypeError), ([a, a.cpu()], ValueError), ([a.cpu()], ValueError), ([a, 3.0], TypeError),
                     ([a[::2]], ValueError), ([a.to_sparse()], TypeError), ([a.clone().requires_grad_()], ValueError)):
        for call in (train.grad_norm, lambda t: train.clip_grad_norm(t, 1.0)):
            with pytest.raises(err):
                call(bad)
    for kw, err in ((dict(norm_type=1.0), ValueError), (dict(scale=torch.ones(2, device=DEV)), ValueError),
                    (dict(scale=torch.ones((), device=DEV).double()), ValueError), (dict(scale=torch.ones(())), ValueError)):
        with pytest.raises(err):
            train.grad_norm([a], **kw)
    for max_norm in (-1.0, math.nan):
        with pytest.raises(DetllmError):
            train.clip_grad_norm([a], max_norm)
    for grads, out, err in (([a], [], ValueError), ([a], [b[:9]], ValueError), ([a], [b.bfloat16()], TypeError),
                            ([a], [b.cpu()], ValueError), ([a.bfloat16()], [b.half()], TypeError),
                            ([a, b], [b, a], DetllmError),  # each over what the other is read from
                            ([a, b], [torch.empty(10, device=DEV)] * 2, DetllmError), ([a[:9]], [a[1:]], DetllmError)):
        with pytest.raises(err):
            train.clip_grad_norm(grads, 1.0, out=out)
    for grads in ([a, a], [a[:6], a[5:]]):
        with pytest.raises(DetllmError):
            train.clip_grad_norm(grads, 1.0)
    assert torch.equal(train.grad_norm([a, a]), train.grad_norm([torch.cat([a, a])]))
    leaf = torch.randn(5, device=DEV, requires_grad=True)
    x = leaf * 1
    y = (x * x).sum()
    with torch.no_grad():
        train.clip_grad_norm([x], 1e-3)
    with pytest.raises(RuntimeError):
        y.backward()
