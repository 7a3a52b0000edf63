"""detllm_amd.scores on torch tensors.  Run by test_gpu_scores_torch.py in a
process of its own, where torch's HIP runtime is the one the library takes."""
import torch  # first: the library shares its HIP runtime

import numpy as np
import pytest

import rows64
from detllm_amd import scores
from detllm_amd._lib import DetllmError

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def logits(seed, *shape, dtype="f32"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * 2 + 6 * (torch.rand(*shape, generator=g) > 0.99)).to(TYPES[dtype]).to(DEV)


def rows_of(t):
    return t.detach().double().cpu().reshape(-1, t.shape[-1]).numpy()


def near(got, want, tol, what):
    got = np.asarray(got.detach().double().cpu().reshape(-1)) if isinstance(got, torch.Tensor) else np.asarray(got)
    off = np.abs(got - want)
    assert (off <= tol).all(), (what, off.max())


def check_scores(z, tokens, got, T, top):
    rows, tok = rows_of(z), tokens.cpu().reshape(-1)
    for i, r in enumerate(rows):
        lp, tol, h, tol_h = rows64.scores(r, int(tok[i]), T)
        near(got.log_probs.reshape(-1)[i], lp, tol, "log_prob")
        near(got.entropy.reshape(-1)[i], h, tol_h, "entropy")
        if top:
            assert got.top_ids.reshape(-1, top)[i].tolist() == rows64.top(r, top, T)[0].tolist()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lead", [(), (1,), (5,), (2, 3), (2, 1, 4)])
def test_scores_of_any_leading_shape(lead, dtype):
    z = logits(1, *lead, 3001, dtype=dtype)
    tokens = torch.randint(0, 3001, lead, device=DEV)
    got = scores.token_scores(z, tokens, top=7, temperature=2.0)
    assert got.log_probs.shape == lead == got.entropy.shape and got.top_ids.shape == (*lead, 7) == got.top_log_probs.shape
    check_scores(z, tokens, got, 2.0, 7)
    same = scores.token_scores(z, tokens.int(), top=7, temperature=2.0)
    assert all(torch.equal(a, b) for a, b in zip(got, same))
    none = scores.token_scores(z, top=2)
    assert none.log_probs is None and torch.equal(none.top_ids, got.top_ids[..., :2])


def test_scores_of_views():
    wide = logits(2, 6, 4, 2100, dtype="bf16")
    for z in (wide[:, :, :2001], wide[1:3, :, 7:2000], wide[:, 2, 1:], wide[::2, 1, :500]):
        tokens = torch.randint(0, z.shape[-1], z.shape[:-1], device=DEV)
        check_scores(z, tokens, scores.token_scores(z, tokens, top=3), 1.0, 3)
    for bad in (wide[:, :2], wide.transpose(1, 2), wide[..., ::2], wide[:1, 0].expand(5, 2100)):
        with pytest.raises(ValueError):
            scores.token_scores(bad)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gradients_through_autograd(dtype):
    T = 0.75
    z = logits(3, 2, 4, 5001, dtype=dtype)[..., :4999].requires_grad_()
    tokens = torch.randint(0, 4999, (2, 4), device=DEV)
    tokens[1, 2] = -1
    g, h = torch.randn(2, 4, device=DEV), torch.randn(2, 4, device=DEV)
    for gg, hh in ((g, h), (g, None), (None, h)):
        got = scores.token_scores(z, tokens, top=2, temperature=T)
        assert not got.top_log_probs.requires_grad
        loss = (0 if gg is None else (got.log_probs * gg).sum()) + (0 if hh is None else (got.entropy * hh).sum())
        grad, = torch.autograd.grad(loss, z)
        for i, r in enumerate(rows_of(z)):
            want, tol = rows64.scores_grad(r, int(tokens.reshape(-1)[i]), T, 0.0 if gg is None else float(gg.reshape(-1)[i]),
                                           0.0 if hh is None else float(hh.reshape(-1)[i]), float(got.entropy.reshape(-1)[i]),
                                           dtype)
            near(grad.reshape(-1, 4999)[i], want, tol, "gradient")


def teacher_of(z, k, T, seed=5):
    t = logits(seed, *z.shape)
    got = scores.token_scores(t, top=k, temperature=T)
    return got.top_ids, got.top_log_probs


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_training_step(dtype, rest):
    """A teacher's alternatives, the student's loss and gradient by autograd and by the step."""
    T, k = 2.0, 16
    hidden = logits(6, 2, 3, 64, dtype="f32")
    head = (logits(7, 64, 2500) * 0.05).requires_grad_()
    z = (hidden @ head).to(TYPES[dtype])
    z.retain_grad()
    ids, v = teacher_of(z, k, T)
    w = torch.tensor([[0.5, 0.0, 1.0], [0.25, 0.1, 0.0]], device=DEV)
    loss = scores.distill_loss(z, ids, v, temperature=T, rest=rest)
    (loss * w).sum().backward()
    step, grad = scores.distill_loss_and_grad(z, ids.long(), v, w, temperature=T, rest=rest)
    assert torch.equal(grad, z.grad) and torch.equal(step, loss.detach() * w)
    for i, r in enumerate(rows_of(z)):
        wi = float(w.reshape(-1)[i])
        args = (r, ids.reshape(-1, k)[i].cpu().numpy(), v.reshape(-1, k)[i].cpu().numpy(), T, rest)
        want, tol, _, _ = rows64.distill(*args, 1.0, dtype)
        near(loss.reshape(-1)[i], want, tol, "loss")
        _, _, dz, dtol = rows64.distill(*args, wi, dtype)
        near(z.grad.reshape(-1, 2500)[i], dz, dtol, "gradient")
    before = head.grad.clone()
    head.grad = None
    z = (hidden @ head).to(TYPES[dtype])
    z.backward(scores.distill_loss_and_grad(z, ids, v, w, temperature=T, rest=rest)[1])
    assert torch.equal(head.grad, before)
    assert float(before.abs().sum()) > 0
    mine = z.detach().clone()
    _, out = scores.distill_loss_and_grad(mine, ids, v, w, temperature=T, rest=rest, out=mine)
    assert out is mine and torch.equal(mine, grad)


def test_no_rows():
    z = torch.empty(0, 100, device=DEV, requires_grad=True)
    got = scores.token_scores(z, torch.empty(0, dtype=torch.long, device=DEV), top=3)
    assert got.log_probs.shape == (0,) and got.top_ids.shape == (0, 3)
    (got.log_probs.sum() + got.entropy.sum()).backward()
    assert z.grad.shape == (0, 100)
    ids, v = torch.empty(0, 4, dtype=torch.int32, device=DEV), torch.empty(0, 4, device=DEV)
    assert scores.distill_loss(z, ids, v).shape == (0,)
    loss, grad = scores.distill_loss_and_grad(z.detach(), ids, v)
    assert loss.shape == (0,) and grad.shape == (0, 100)


def test_on_another_stream_and_two_at_once():
    z = [logits(8 + i, 200, 30000, dtype="bf16") for i in range(2)]
    tokens = torch.randint(0, 30000, (200,), device=DEV)
    want = [scores.token_scores(x, tokens, top=20) for x in z]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in z]
    got = [[] for _ in z]
    for _ in range(10):
        for x, s, o in zip(z, streams, got):
            with torch.cuda.stream(s):
                o.append(scores.token_scores(x, tokens, top=20))
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        for r in o:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


def test_forward_and_backward_in_a_graph():
    """Captured together, replayed with new logits between eager calls, on a leaf of its own."""
    T, k = 1.0, 8
    static = logits(10, 40, 6001, dtype="bf16")
    ids, v = teacher_of(static, k, T)
    tokens = torch.randint(0, 6001, (40,), device=DEV)
    w = torch.rand(40, device=DEV)

    def work(z):
        leaf = z.detach().requires_grad_()
        got = scores.token_scores(leaf, tokens, top=4)
        loss = scores.distill_loss(leaf, ids, v, rest=True)
        grad, = torch.autograd.grad([got.log_probs, got.entropy, loss], [leaf], [w, w, w])
        return got.log_probs, got.entropy, got.top_ids, loss, grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(static)
    for i in range(4):
        fresh = logits(20 + i, 40, 6001, dtype="bf16")
        want = work(fresh)
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_refusals():
    z = logits(11, 4, 300)
    tok = torch.zeros(4, dtype=torch.long, device=DEV)
    ids, v = teacher_of(z, 8, 1.0)
    for bad, err in ((z.double(), TypeError), (z.cpu(), ValueError), (z[0, 0], ValueError), (z[:, :0], ValueError),
                     (z.tolist(), TypeError)):
        with pytest.raises(err):
            scores.token_scores(bad)
    for bad, err in ((tok.float(), TypeError), (tok.cpu(), ValueError), (tok[:3], ValueError), (tok[:, None], ValueError)):
        with pytest.raises(err):
            scores.token_scores(z, bad)
    for bad_ids, bad_v, err in ((ids.float(), v, TypeError), (ids, v.double(), TypeError), (ids[:3], v[:3], ValueError),
                                (ids, v[:, :7], ValueError), (ids.cpu(), v, ValueError), (ids, v.cpu(), ValueError)):
        for f in (scores.distill_loss, scores.distill_loss_and_grad):
            with pytest.raises(err):
                f(z, bad_ids, bad_v)
    with pytest.raises(ValueError):
        scores.distill_loss_and_grad(z, ids, v, torch.ones(3, device=DEV))
    for out in (torch.empty(4, 299, device=DEV), torch.empty(4, 300, device=DEV, dtype=torch.bfloat16), torch.empty(4, 300),
                torch.empty(300, 4, device=DEV).t()):
        with pytest.raises(ValueError):
            scores.distill_loss_and_grad(z, ids, v, out=out)
    for kw, status in ((dict(top=129), 1), (dict(top=301), 1), (dict(top=-1), 1), (dict(temperature=0.0), 42)):
        with pytest.raises(DetllmError) as e:
            scores.token_scores(z, tok, **kw)
        assert e.value.status == status
    with pytest.raises(DetllmError):
        scores.distill_loss(z, torch.zeros(4, 257, dtype=torch.long, device=DEV), torch.zeros(4, 257, device=DEV))
    # a changed input is noticed, a second derivative refused
    leaf = z.clone().requires_grad_()
    x = leaf * 1
    s = scores.token_scores(x, tok).log_probs.sum()
    with torch.no_grad():
        x.zero_()
    with pytest.raises(RuntimeError):
        s.backward()
    x = leaf * 1
    s = (x * x).sum()
    scores.distill_loss_and_grad(x, ids, v, out=x)  # over what s needs
    with pytest.raises(RuntimeError):
        s.backward()
    g, = torch.autograd.grad(scores.distill_loss(leaf, ids, v).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_logits_larger_than_the_cache():
    """Beyond 256 MB, rows of odd length: read and written past the caches, the same bits."""
    R, V, k = 900, 151937, 5
    z = torch.empty(R, V, dtype=torch.bfloat16, device=DEV).normal_()
    few = [slice(0, 3), slice(449, 451), slice(R - 2, R)]
    tokens = torch.randint(0, V, (R,), device=DEV)
    leaf = z.requires_grad_()
    w = torch.rand(R, device=DEV)

    def work(rows):
        x = leaf[rows]
        got = scores.token_scores(x, tokens[rows], top=k)
        loss = scores.distill_loss(x, got.top_ids, got.top_log_probs - 0.2, rest=True)
        g, = torch.autograd.grad([got.log_probs, got.entropy], [x], [w[rows], -w[rows]], retain_graph=True)
        d, = torch.autograd.grad([loss], [x], [w[rows]])
        step = scores.distill_loss_and_grad(x.detach(), got.top_ids, got.top_log_probs - 0.2, w[rows], rest=True)
        return [t.detach() for t in (*got, loss, g, d, *step)]

    whole = work(slice(None))
    for rows in few:
        for a, b in zip(whole, work(rows)):
            assert torch.equal(a[rows], b)
    i = 450
    want, tol = rows64.scores_grad(rows_of(z[i:i + 1])[0], int(tokens[i]), 1.0, float(w[i]), -float(w[i]),
                                   float(whole[1][i]), "bf16")
    near(whole[5][i], want, tol, "gradient")


def test_more_rows_than_a_launch():
    R, V = (1 << 18) + 5, 70
    z = logits(40, 64, V, dtype="f16").repeat(R // 64 + 1, 1)[:R].contiguous().requires_grad_()
    tokens = (torch.arange(R, device=DEV) % 64) % V
    got = scores.token_scores(z, tokens, top=2)
    loss = scores.distill_loss(z, got.top_ids, got.top_log_probs)
    ones = torch.ones(R, device=DEV)
    grad, = torch.autograd.grad([got.log_probs, got.entropy, loss], [z], [ones, ones, ones])
    step = scores.distill_loss_and_grad(z.detach(), got.top_ids, got.top_log_probs)
    for t in (*got, loss, grad, *step):
        t = t.detach().reshape(R, -1)
        assert torch.equal(t[64:], t[:-64])
    check_scores(z[:3], tokens[:3], type(got)(*(t[:3] for t in got)), 1.0, 2)


def test_rows_past_32_bits():
    """More than 2^31 logits: the last rows are read and written where they are."""
    V, R = 1 << 18, (1 << 13) + 3
    z = torch.empty(R, V, dtype=torch.bfloat16, device=DEV)
    z.fill_(-1.0)
    z[-1] = logits(30, V, dtype="bf16")
    z[-2, 77] = 9.0
    tokens = torch.full((R,), 77, device=DEV)
    got = scores.token_scores(z, tokens, top=2)
    last = scores.token_scores(z[-2:].clone(), tokens[-2:], top=2)
    assert all(torch.equal(a[-2:], b) for a, b in zip(got, last))
    ids, v = got.top_ids, got.top_log_probs
    w = torch.ones(R, device=DEV)
    want = scores.distill_loss_and_grad(z[-2:].clone(), ids[-2:], v[-2:] - 0.1, w[-2:], rest=True)
    loss, grad = scores.distill_loss_and_grad(z, ids, v - 0.1, w, rest=True, out=z)
    assert torch.equal(loss[-2:], want[0]) and torch.equal(grad[-2:], want[1])
