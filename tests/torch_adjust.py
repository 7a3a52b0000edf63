"""detllm_amd.scores.adjust_logits.  Run by test_gpu_adjust.py in a process of its
own, where torch's HIP runtime is the one the library takes."""
import torch  # first: the library shares its HIP runtime

import numpy as np
import pytest

import adjust64
from detllm_amd import scores
from detllm_amd._lib import DetllmError

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def words_of(on):
    """bool[..., vocab] as 32-bit words, with noise behind the last logit."""
    V = on.shape[-1]
    pad = torch.rand(*on.shape[:-1], -V % 32, device=on.device) < 0.5
    bits = torch.cat([on, pad], -1).view(*on.shape[:-1], -1, 32).int()
    return (bits << torch.arange(32, device=on.device, dtype=torch.int32)).sum(-1, dtype=torch.int32)


def case(seed, R, V, dtype, H=0, K=0, mask="", wide=True, shared=False, per_row=False, stride=None, wild=False):
    """Logits, arguments, and the same on the host for each row."""
    g = torch.Generator().manual_seed(seed)
    z = torch.empty(R, stride or V, dtype=TYPES[dtype], device=DEV)[:, :V]
    x = 4 * torch.randn(R, V, generator=g)
    if wild:  # infinities, no numbers, the type's lowest, both zeros
        odd = torch.tensor([float("inf"), float("-inf"), float("nan"), torch.finfo(TYPES[dtype]).min, 0.0, -0.0])
        x = torch.where(torch.rand(R, V, generator=g) < 0.3, odd[torch.randint(0, 6, (R, V), generator=g)], x)
    z.copy_(x)
    kw, rows = {}, [{} for _ in range(R)]
    index = torch.int64 if wide else torch.int32

    def lead(t):
        return t.expand(R, -1) if shared else t

    if H:
        # a third of the places are no token, or one that is not in the vocabulary
        h = torch.randint(-V // 3 - 1, V + V // 6 + 1, ((H,) if shared else (R, H)), generator=g)
        h = torch.where(torch.rand(h.shape, generator=g) < 0.3, h.clamp(0, min(3, V - 1)), h)  # some often
        prompt = torch.randint(-2, H + 3, (R,), generator=g)
        theta, presence, frequency = 0.5 + torch.rand(R, generator=g), torch.randn(R, generator=g), torch.randn(R, generator=g)
        if not per_row:
            theta, presence, frequency = (t[:1].expand(R) for t in (theta, presence, frequency))
        for i in range(R):
            rows[i].update(history=lead(h)[i].tolist(), prompt=int(prompt[i]), theta=float(theta[i]),
                           presence=float(presence[i]), frequency=float(frequency[i]))
        kw.update(history=h.to(index).to(DEV), prompt=prompt.to(index).to(DEV))
        for name, t in (("repetition", theta), ("presence", presence), ("frequency", frequency)):
            kw[name] = t.to(DEV) if per_row else float(t[0])
    if K:
        ids = torch.randint(-2, V + 2, ((K,) if shared else (R, K)), generator=g)
        bias = 3 * torch.randn(ids.shape, generator=g)
        bias[..., 0] = float("-inf")
        for i in range(R):
            rows[i].update(bias_ids=lead(ids)[i].tolist(), bias=lead(bias)[i].tolist())
        kw.update(bias_ids=ids.to(index).to(DEV), bias=bias.to(DEV))
    if mask:
        on = torch.rand((V,) if shared else (R, V), generator=g) < 0.6
        if not shared and R > 1:
            on[1] = False  # nothing is left
        if not shared and R > 2:
            on[2] = True
        for i in range(R):
            rows[i]["allowed"] = lead(on)[i].numpy()
        kw["allowed"] = on.to(DEV) if mask == "bytes" else words_of(on.to(DEV))
    return z, kw, rows


def host(t):
    return t.detach().double().cpu().numpy()


def check(z, kw, rows, dtype, got, before=None):
    for i, (x, y) in enumerate(zip(host(z if before is None else before), host(got))):
        want, tol = adjust64.adjust(x, dtype, **rows[i])
        ok = adjust64.same(y, want, tol)
        assert ok.all(), (i, np.flatnonzero(~ok)[:5], y[~ok][:5], want[~ok][:5], x[~ok][:5])


SHAPES = [  # rows, vocabulary, history, biases, mask, 64-bit ids, one for all rows, numbers for each row, stride
    (1, 1, 1, 1, "bits", True, False, False, None),
    (3, 7, 5, 3, "bytes", False, False, True, 9),
    (4, 256, 40, 0, "", True, False, True, None),
    (3, 1001, 0, 17, "bits", False, True, False, 1003),
    (5, 2047, 300, 300, "bytes", True, True, True, 2051),
    (3, 2049, 2500, 1, "bits", False, False, False, 2050),
    (2, 8191, 64, 5, "bytes", True, False, False, None),
    (3, 8192, 129, 33, "bits", True, False, True, None),
    (3, 8193, 7000, 4096, "bits", True, False, True, 8195),
    (2, 32003, 20000, 100, "bytes", False, True, False, 32003),
    (1, 151936, 131072, 16, "bits", False, False, False, None),
    (9, 262144, 50, 2, "bits", True, False, True, None),
]


@pytest.mark.parametrize("wild", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:5])))
def test_adjusted_logits(shape, dtype, wild):
    R, V, H, K, mask, wide, shared, per_row, stride = shape
    z, kw, rows = case(sum(shape[:4]), R, V, dtype, H, K, mask, wide, shared, per_row, stride, wild)
    got = scores.adjust_logits(z, **kw)
    check(z, kw, rows, dtype, got)
    # in place, at the logits' own stride; what lies between the rows stays
    mine = torch.full((R, (stride or V) + 3), 7.0, dtype=z.dtype, device=DEV)
    part = mine[:, :V]
    part.copy_(z)
    out = scores.adjust_logits(part, **kw, out=part)
    assert out is part and torch.equal(part.nan_to_num(1.5), got.nan_to_num(1.5)) and torch.equal(part.isnan(), got.isnan())
    assert (mine[:, V:] == 7.0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("parts", ["h", "hm", "m", "k", "hkm"])
def test_gradient(parts, dtype):
    R, V = 4, 9001
    z, kw, rows = case(5, R, V, dtype, 700 if "h" in parts else 0, 9 if "k" in parts else 0, "bits" if "m" in parts else "",
                       per_row="k" in parts, stride=9011)
    leaf = z.requires_grad_()
    got = scores.adjust_logits(leaf, **kw)
    assert torch.equal(got.detach(), scores.adjust_logits(z.detach(), **kw))
    g = torch.randn(R, V, device=DEV).to(z.dtype)
    if "m" in parts:  # whatever is there where nothing is allowed
        on = torch.stack([torch.from_numpy(r["allowed"]) for r in rows]).to(DEV)
        g = torch.where(~on & (torch.rand(R, V, device=DEV) < 0.5), float("nan"), g)
    grad, = torch.autograd.grad(got, leaf, g)
    for i in range(R):
        r = rows[i]
        want, tol = adjust64.gradient(host(z)[i], host(g)[i], dtype, r.get("history", ()), r.get("theta", 1.0), r.get("allowed"))
        assert adjust64.same(host(grad)[i], want, tol).all()


def test_gradient_of_a_sum_of_one_row_and_of_a_shared_history():
    z, kw, rows = case(6, 3, 500, "f32", 50, shared=True)
    for x, n in ((z[1], 1), (z.view(3, 1, 500), 3)):
        args = dict(kw, prompt=kw["prompt"][1] if n == 1 else kw["prompt"][:, None])
        leaf = x.clone().requires_grad_()
        scores.adjust_logits(leaf, **args).sum().backward()
        for i, row in enumerate(host(leaf).reshape(-1, 500)):
            want, tol = adjust64.gradient(row, np.ones(500), "f32", rows[0]["history"], rows[0]["theta"])
            assert adjust64.same(host(leaf.grad).reshape(-1, 500)[i], want, tol).all()
    # an intermediate tensor, written in place under no_grad, is noticed
    leaf = z.clone().requires_grad_()
    x = leaf * 1
    y = scores.adjust_logits(x, **kw).sum()
    with torch.no_grad():
        scores.adjust_logits(x, **kw, out=x)
    with pytest.raises(RuntimeError):
        y.backward()


def test_rows_alone_and_among_others():
    z, kw, rows = case(7, 40, 40000, "bf16", 500, 20, "bits", per_row=True)
    got = scores.adjust_logits(z, **kw)
    for i in (0, 17, 39):
        one = {k: v if not isinstance(v, torch.Tensor) else v[i:i + 1] for k, v in kw.items()}
        assert torch.equal(scores.adjust_logits(z[i:i + 1], **one), got[i:i + 1])


def test_out_between_the_rows_and_into_another_tensor():
    both = torch.randn(6, 2, 3001, device=DEV)
    z, out = both[:, 0], both[:, 1]
    _, kw, rows = case(8, 6, 3001, "f32", 60, 4, "bytes")
    before = z.clone()
    got = scores.adjust_logits(z, **kw, out=out)
    assert got is out and torch.equal(z, before)
    check(z, kw, rows, "f32", out)
    with pytest.raises(DetllmError):
        scores.adjust_logits(both.view(12, 3001)[:6], **kw, out=both.view(12, 3001)[3:9])


def test_parts_of_longer_buffers():
    """The first places of a history that grows, masks and biases cut from wider ones,
    one row for all by expand: as their copies, forward and backward."""
    z, kw, rows = case(12, 6, 3000, "bf16", 500, 20, "bits", per_row=True)

    def wider(t, n):
        buf = torch.full((*t.shape[:-1], t.shape[-1] + n), 1, dtype=t.dtype, device=DEV)
        buf[..., n // 2:n // 2 + t.shape[-1]] = t
        return buf[..., n // 2:n // 2 + t.shape[-1]]

    cut = {k: wider(v, 14) if v.dim() == 2 else torch.stack([v, v], 1)[:, 1] for k, v in kw.items()}
    assert not any(v.is_contiguous() for v in cut.values())
    first = {k: v[:1] for k, v in kw.items()}
    alike = {k: v.expand(6, *v.shape[1:]) for k, v in first.items()}
    copied = {k: v.contiguous() for k, v in alike.items()}
    for a, b in ((cut, kw), (alike, copied)):
        leaf = z.clone().requires_grad_()
        got = [scores.adjust_logits(leaf, **x) for x in (a, b)]
        assert torch.equal(*got)
        g = torch.randn_like(got[0])
        assert torch.equal(*(torch.autograd.grad(x, leaf, g)[0] for x in got))
        with torch.autograd.graph.save_on_cpu():
            moved = scores.adjust_logits(leaf, **a)
        assert torch.equal(torch.autograd.grad(moved, leaf, g)[0], torch.autograd.grad(scores.adjust_logits(leaf, **b), leaf, g)[0])
    three = {k: v[:, None].expand(6, 2, *v.shape[1:]) for k, v in kw.items()}
    got = scores.adjust_logits(z[:, None].expand(6, 2, 3000).contiguous(), **three)
    assert torch.equal(got[:, 0], got[:, 1]) and torch.equal(got[:, 0], scores.adjust_logits(z, **kw))
    assert torch.equal(scores.adjust_logits(z, history=kw["history"], repetition=np.float32(1.5)),
                       scores.adjust_logits(z, history=kw["history"], repetition=1.5))


def test_nothing_to_do_copies():
    z = torch.randn(3, 100, device=DEV)
    for kw in ({}, dict(history=torch.zeros(3, 5, dtype=torch.long, device=DEV)),
               dict(history=torch.zeros(3, 0, dtype=torch.long, device=DEV), repetition=2.0)):
        got = scores.adjust_logits(z, **kw)
        assert torch.equal(got, z) and got.data_ptr() != z.data_ptr()
        assert torch.equal(scores.adjust_logits(z, **kw, out=z), got)
    leaf = z.clone().requires_grad_()
    grad, = torch.autograd.grad(scores.adjust_logits(leaf), leaf, z)
    assert torch.equal(grad, z)


def test_no_rows():
    z = torch.empty(0, 100, device=DEV, requires_grad=True)
    h = torch.empty(0, 4, dtype=torch.long, device=DEV)
    got = scores.adjust_logits(z, history=h, repetition=2.0)
    got.sum().backward()
    assert got.shape == (0, 100) == z.grad.shape


def test_in_a_graph_and_on_another_stream():
    z, kw, rows = case(9, 50, 33000, "bf16", 400, 20, "bits", per_row=True)
    static = z.clone()

    def work(x):
        leaf = x.detach().requires_grad_()
        got = scores.adjust_logits(leaf, **kw)
        grad, = torch.autograd.grad(got, leaf, torch.ones_like(got))
        mine = x.clone()
        scores.adjust_logits(mine, **kw, out=mine)
        return got.detach(), grad, mine, scores.token_scores(mine, top=5).top_ids

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(static)
    for i in range(3):
        fresh = torch.randn(z.shape, device=DEV).to(z.dtype)
        want = work(fresh)
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_more_rows_than_a_launch_and_past_32_bits():
    R, V = (1 << 18) + 5, 64
    z, kw, rows = case(10, 16, V, "f16", 9, 2, "bits")
    big = {k: v.repeat(R // 16 + 1, 1)[:R] if isinstance(v, torch.Tensor) and v.dim() > 1 else
           v.repeat(R // 16 + 1)[:R] if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    got = scores.adjust_logits(z.repeat(R // 16 + 1, 1)[:R], **big)
    want = scores.adjust_logits(z, **kw)
    assert torch.equal(got[:16], want) and torch.equal(got[16:], got[:-16])
    V, R = 1 << 18, (1 << 13) + 3
    z = torch.empty(R, V, dtype=torch.bfloat16, device=DEV).fill_(1.0)
    history = torch.full((R, 3), V - 1, device=DEV)
    on = words_of(torch.arange(V, device=DEV) > 0)
    scores.adjust_logits(z, history=history, repetition=2.0, presence=0.25, allowed=on, out=z)
    assert (z[:, 0] == float("-inf")).all() and (z[:, -1] == 0.25).all() and (z[-1, 1:-1] == 1.0).all()
    assert bool((z[:, 1:-1] == 1.0).all())


def test_masks_and_scores_together():
    """What a constrained decoder asks: the alternatives among what is allowed."""
    z = torch.randn(8, 32000, device=DEV)
    on = torch.rand(8, 32000, device=DEV) < 0.001
    on[3] = False
    got = scores.token_scores(scores.adjust_logits(z, allowed=words_of(on)), top=8)
    for i in range(8):
        ids = [t for t in torch.where(on[i], z[i], -1e9).topk(8).indices.tolist() if on[i, t]]
        assert [t for t in got.top_ids[i].tolist() if t >= 0] == ids
    assert (got.top_ids[3] == -1).all() and got.entropy[3] == 0


def test_refusals():
    z, kw, _ = case(11, 4, 300, "f32", 6, 3, "bits")
    bad = lambda **k: scores.adjust_logits(z, **dict(kw, **k))  # noqa: E731
    dev = dict(device=DEV)
    for k, err in ((dict(history=kw["history"].float()), TypeError), (dict(history=kw["history"].cpu()), ValueError),
                   (dict(history=kw["history"][:3]), ValueError), (dict(prompt=kw["prompt"][:3]), ValueError),
                   (dict(history=None), ValueError), (dict(bias=None), ValueError), (dict(bias_ids=None), ValueError),
                   (dict(bias=kw["bias"].double()), TypeError), (dict(bias=kw["bias"][:, :2]), ValueError),
                   (dict(bias=kw["bias"].clone().requires_grad_()), ValueError),
                   (dict(repetition=torch.ones(4, **dev).requires_grad_()), ValueError),
                   (dict(repetition=torch.ones(3, **dev)), ValueError), (dict(presence=torch.ones(4, **dev).double()), TypeError),
                   (dict(allowed=kw["allowed"][:, :-1]), ValueError), (dict(allowed=kw["allowed"].float()), TypeError),
                   (dict(allowed=torch.ones(4, 299, dtype=torch.bool, **dev)), ValueError),
                   (dict(out=torch.empty(4, 299, **dev)), ValueError), (dict(out=torch.empty(4, 300)), ValueError),
                   (dict(out=torch.empty(300, 4, **dev).t()), ValueError),
                   (dict(repetition=0.0), DetllmError), (dict(repetition=-1.0), DetllmError),
                   (dict(repetition=float("inf")), DetllmError), (dict(presence=float("nan")), DetllmError),
                   (dict(frequency=float("inf")), DetllmError),
                   (dict(history=torch.zeros(4, (1 << 17) + 1, dtype=torch.int32, **dev)), DetllmError),
                   (dict(bias_ids=torch.zeros(4097, dtype=torch.long, **dev), bias=torch.zeros(4097, **dev)), DetllmError)):
        with pytest.raises(err):
            bad(**k)
    for t in (z.double(), z.cpu(), z[0, 0], z.t(), z.tolist()):
        with pytest.raises((TypeError, ValueError)):
            scores.adjust_logits(t)
    leaf = z.clone().requires_grad_()
    with pytest.raises(ValueError):
        scores.adjust_logits(leaf, **kw, out=torch.empty_like(z))
    with pytest.raises(ValueError):
        scores.adjust_logits(z, **kw, out=leaf)
    g, = torch.autograd.grad(scores.adjust_logits(leaf, **kw).exp().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
