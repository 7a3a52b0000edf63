"""detllm_amd.train's embeddings.  Run by test_gpu_train.py in a process of its own,
where torch's HIP runtime is the one the library takes."""
import torch  # first: the library shares its HIP runtime

import numpy as np
import pytest

import train64
from adjust64 import same
from detllm_amd import train
from detllm_amd._lib import DetllmError

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def host(t):
    return t.detach().double().cpu().numpy()


def inputs(seed, n, V, D, dtype, wide=True, kind="text"):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g).to(TYPES[dtype]).to(DEV)
    if kind == "text":  # a few tokens often, some padding, some that are none
        t = (V * torch.rand(n, generator=g) ** 6).long().clamp(max=V - 1)
        t = torch.where(torch.rand(n, generator=g) < 0.1, -1, t)
        t = torch.where(torch.rand(n, generator=g) < 0.02, V + 3, t)
    elif kind == "one":
        t = torch.full((n,), V // 2)
    elif kind == "none":
        t = torch.full((n,), -5)
    else:  # each in turn, from the last
        t = V - 1 - torch.arange(n) % V
    grad = torch.randn(n, D, generator=g).to(TYPES[dtype]).to(DEV)
    return w, t.to(torch.int64 if wide else torch.int32).to(DEV), grad


def check_gradient(tokens, grad, got, scale, dtype, old=None):
    want, tol = train64.gradient(tokens.cpu().numpy(), host(grad), got.shape[0], scale, dtype, old)
    assert same(host(got), want, tol).all()


SHAPES = [  # tokens, vocabulary, width, kind
    (1, 1, 1, "one"), (1, 300, 17, "text"), (7, 50, 8, "turn"), (65, 513, 100, "text"), (1000, 49, 33, "text"),
    (1024, 262144, 3, "turn"), (1025, 1000, 24, "text"), (4096, 5000, 40, "text"), (4097, 5000, 40, "text"),
    (5000, 262144, 5, "text"), (3000, 700, 64, "one"), (2000, 700, 9, "none"), (20000, 32000, 7, "text"),
    (70001, 1200, 18, "text"), (200000, 500, 2, "one"), (300, 90, 2050, "text"), (300000, 3000, 4, "turn"),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_lookup_and_gradient(shape, dtype):
    n, V, D, kind = shape
    scale = 1.0 if D % 2 else 1.7
    w, tokens, g = inputs(n + V, n, V, D, dtype, wide=n % 2 == 0, kind=kind)
    leaf = w.requires_grad_()
    rows = train.embedding(leaf, tokens, scale=scale)
    few = torch.randperm(n, generator=torch.Generator().manual_seed(1))[:2000]
    want, tol = train64.embedding(host(w), tokens.cpu().numpy()[few], scale, dtype)
    assert same(host(rows)[few], want, tol).all()
    grad, = torch.autograd.grad(rows, leaf, g)
    check_gradient(tokens, g, grad, scale, dtype)
    again = train.embedding_grad(tokens, g, V, scale=scale)
    assert torch.equal(again, grad)
    # on top of what is there, of the rows' type and in 32 bits; other rows are left as they are
    for out in (torch.randn(V, D, device=DEV).to(w.dtype), torch.randn(V, D + 3, device=DEV)[:, :D]):
        old = out.clone()
        assert train.embedding_grad(tokens, g, scale=scale, out=out, add=True) is out
        check_gradient(tokens, g, out, scale, "f32" if out.dtype == torch.float32 else dtype, host(old))
        absent = torch.ones(V, dtype=torch.bool, device=DEV)
        absent[tokens[(tokens >= 0) & (tokens < V)].long()] = False
        assert torch.equal(out[absent], old[absent])


def test_leading_shapes_and_strides():
    w, tokens, g = inputs(1, 24, 100, 20, "bf16")
    for lead in ((24,), (4, 6), (2, 3, 1, 4)):
        rows = train.embedding(w, tokens.view(lead))
        assert rows.shape == (*lead, 20) and torch.equal(rows.view(24, 20), train.embedding(w, tokens))
        assert torch.equal(train.embedding_grad(tokens.view(lead), g.view(*lead, 20), 100), train.embedding_grad(tokens, g, 100))
    assert train.embedding(w, tokens[0]).shape == (20,)
    wide = torch.randn(100, 33, device=DEV).bfloat16()
    part = wide[:, 5:25]  # rows further apart than they are long, not aligned
    assert torch.equal(train.embedding(part, tokens).nan_to_num(3.0), train.embedding(part.contiguous(), tokens).nan_to_num(3.0))
    out = torch.full((100, 33), 9.0, device=DEV).bfloat16()
    train.embedding_grad(tokens, g, out=out[:, 5:25])
    assert torch.equal(out[:, 5:25], train.embedding_grad(tokens, g, 100)) and (out[:, :5] == 9).all() and (out[:, 25:] == 9).all()
    wider = torch.randn(24, 31, device=DEV).bfloat16()
    leaf = w.clone().requires_grad_()
    for x in (wider[:, 3:23], wider[:, :20], wider[:1, 5:25].expand(24, 20)):
        want = train.embedding_grad(tokens, x.contiguous(), 100)
        assert torch.equal(train.embedding_grad(tokens, x, 100), want)
        assert torch.equal(torch.autograd.grad(train.embedding(leaf, tokens), leaf, x)[0], want)
    every_other = torch.randn(24, 40, device=DEV).bfloat16()[:, ::2]
    assert torch.equal(train.embedding_grad(tokens, every_other, 100), train.embedding_grad(tokens, every_other.contiguous(), 100))


def test_rows_that_are_no_number_stay_with_their_tokens():
    w, tokens, g = inputs(2, 3000, 400, 24, "f32")
    bad = torch.tensor([5, 700, 2999], device=DEV)
    tokens[bad] = torch.tensor([11, -1, 399], device=DEV)
    g[bad] = float("nan")
    got = train.embedding_grad(tokens, g, 400)
    assert got.isnan().any(1).nonzero().flatten().tolist() == [11, 399]
    w[7] = float("inf")
    rows = train.embedding(w, torch.tensor([7, -1, 400, 8], device=DEV), scale=0.0)
    assert rows[0].isnan().all() and (rows[1] == 0).all() and rows[2].isnan().all() and (rows[3] == 0).all()


def test_no_tokens():
    w = torch.randn(10, 6, device=DEV, requires_grad=True)
    none = torch.empty(0, 3, dtype=torch.long, device=DEV)
    rows = train.embedding(w, none)
    rows.sum().backward()
    assert rows.shape == (0, 3, 6) and (w.grad == 0).all()
    out = torch.ones(10, 6, device=DEV)
    train.embedding_grad(none, rows.detach(), out=out, add=True)
    assert (out == 1).all()


@pytest.mark.parametrize("n", [3000, 9000])
def test_in_a_graph_and_on_two_streams(n):
    V, D = 6000, 70
    w, tokens, g = inputs(3, n, V, D, "bf16")
    static_t, static_g = tokens.clone(), g.clone()

    def work(t, x):
        leaf = w.detach().requires_grad_()
        rows = train.embedding(leaf, t, scale=2.0)
        grad, = torch.autograd.grad(rows, leaf, x)
        return rows.detach(), grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(static_t, static_g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(static_t, static_g)
    wants = []
    for i in range(3):
        _, t, x = inputs(30 + i, n, V, D, "bf16")
        wants.append((t, x, want := work(t, x)))
        static_t.copy_(t)
        static_g.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))
    streams, got = [torch.cuda.Stream() for _ in wants], [[] for _ in wants]
    torch.cuda.synchronize()
    for _ in range(5):
        for (t, x, _), s, o in zip(wants, streams, got):
            with torch.cuda.stream(s):
                o.append(work(t, x))
    torch.cuda.synchronize()
    for (_, _, want), o in zip(wants, got):
        for r in o:
            assert all(torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) for a, b in zip(r, want))


def test_tables_past_32_bits():
    V, D = 1 << 17, 1 << 14  # 2^31 elements
    w = torch.zeros(V, D, dtype=torch.bfloat16, device=DEV)
    w[-1], w[1] = 2.0, 3.0
    tokens = torch.tensor([V - 1, 0, 1, V - 1], device=DEV)
    rows = train.embedding(w, tokens)
    assert (rows == torch.tensor([2.0, 0.0, 3.0, 2.0], device=DEV)[:, None]).all()
    w.fill_(7.0)
    train.embedding_grad(tokens, rows, out=w)
    assert (w[-1] == 4).all() and (w[1] == 3).all() and (w[0] == 0).all() and not w[2:-1].any()


def test_as_many_tokens_as_a_gradient_takes():
    n, V = 1 << 20, 70000
    g = torch.Generator(device=DEV).manual_seed(4)
    tokens = torch.randint(0, V, (n,), generator=g, device=DEV)
    tokens[: n // 4] = 69999
    x = torch.randint(-3, 4, (n, 8), generator=g, device=DEV).float()  # sums of whole numbers are exact
    got = train.embedding_grad(tokens, x, V)
    assert torch.equal(got, torch.zeros(V, 8, dtype=torch.float64, device=DEV).index_add_(0, tokens, x.double()).float())
    with pytest.raises(DetllmError):
        train.embedding_grad(torch.zeros(n + 1, dtype=torch.int32, device=DEV), torch.zeros(n + 1, 1, device=DEV), 5)
    with pytest.raises(DetllmError):
        train.embedding(torch.zeros(3, 1, device=DEV, requires_grad=True), torch.zeros(n + 1, dtype=torch.int32, device=DEV))
    assert train.embedding(torch.ones(3, 1, device=DEV), torch.zeros(n + 1, dtype=torch.int32, device=DEV)).all()


def test_refusals():
    w, tokens, g = inputs(5, 12, 30, 8, "f32")
    for bad, err in ((w.double(), TypeError), (w.cpu(), ValueError), (w[0], ValueError), (w.t(), ValueError),
                     (w[:0], ValueError), (w[:1].expand(30, 8), ValueError), (w.tolist(), TypeError)):
        with pytest.raises(err):
            train.embedding(bad, tokens)
    for bad, err in ((tokens.float(), TypeError), (tokens.cpu(), ValueError), (tokens.tolist(), TypeError)):
        with pytest.raises(err):
            train.embedding(w, bad)
        with pytest.raises(err):
            train.embedding_grad(bad, g, 30)
    for args, kw, err in (((tokens, g), {}, ValueError), ((tokens, g, 30), dict(add=True), ValueError),
                          ((tokens, g[:5], 30), {}, ValueError), ((tokens, g.double(), 30), {}, TypeError),
                          ((tokens, g, 31), dict(out=w), ValueError), ((tokens, g[:, :7]), dict(out=w), ValueError),
                          ((tokens, g), dict(out=w.bfloat16()), TypeError), ((tokens, g), dict(out=w.cpu()), ValueError),
                          ((tokens, g), dict(out=w.clone().requires_grad_()), ValueError),
                          ((tokens, g), dict(out=torch.zeros(8, 30, device=DEV).t()), ValueError),
                          ((tokens[:8], w[:8]), dict(out=w), DetllmError),
                          ((tokens, g, (1 << 18) + 1), {}, DetllmError)):
        with pytest.raises(err):
            train.embedding_grad(*args, **kw)
    with pytest.raises(DetllmError):
        train.embedding(torch.zeros(2, (1 << 16) + 1, device=DEV), tokens)
    leaf = w.clone().requires_grad_()
    x, = torch.autograd.grad(train.embedding(leaf, tokens).exp().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        x.sum().backward()
    changed = tokens.clone()
    rows = train.embedding(leaf, changed)
    changed.zero_()
    with pytest.raises(RuntimeError):
        rows.sum().backward()
