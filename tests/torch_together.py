"""The operators together, as programs use them: a student's distillation step, and a
constrained decoder's.  Run by test_gpu_train.py in a process of its own."""
import torch  # first: the library shares its HIP runtime

import pytest

from detllm_amd import scores, train
from words import words_of

DEV = "cuda"


def student(seed, V, D, dtype):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * k).to(dtype).to(DEV).requires_grad_()
            for s, k in (((V, D), 1.0), ((D, D), D**-0.5), ((V, D), 0.5))]


def steps(params, tokens, history, on, ids, v, w, T, manual):
    table, mix, head = params
    hidden = train.embedding(table, tokens, scale=2.0)
    z = torch.tanh(hidden @ mix) @ head.t()
    x = scores.adjust_logits(z, history=history, repetition=1.3, allowed=on)
    if manual:
        loss, grad = scores.distill_loss_and_grad(x.detach(), ids, v, w, temperature=T, rest=True)
        x.backward(grad)
        return loss
    loss = scores.distill_loss(x, ids, v, temperature=T, rest=True) * w
    loss.sum().backward()
    return loss.detach()


def in_64_bits(params, tokens, history, on, ids, v, w, T):
    """The same with elementary operations in float64 on the CPU."""
    table, mix, head = ps = [p.detach().double().cpu().requires_grad_() for p in params]
    tokens, history, on, ids, v, w = (t.cpu() for t in (tokens, history, on, ids, v, w))
    hidden = torch.where(tokens[:, None] < 0, 0.0, table[tokens.clamp(min=0)]) * 2.0
    z = torch.tanh(hidden @ mix) @ head.t()
    theta = float(torch.tensor(1.3))
    seen = torch.zeros(z.shape, dtype=torch.bool).scatter_(1, history, True)
    z = torch.where(seen, torch.where(z > 0, z / theta, z * theta), z).masked_fill(~on, -torch.inf)
    lq = torch.log_softmax(z / T, 1)
    p = v.double().exp()
    loss = (p * (v.double() - lq.gather(1, ids.long()))).sum(1)
    rest = 1 - p.sum(1)
    inside = torch.zeros(z.shape, dtype=torch.bool).scatter_(1, ids.long(), True)
    left = torch.where(inside | ~on, 0.0, lq.exp()).sum(1)
    loss = (loss + rest * (rest.log() - left.log())) * T * T * w.double()
    loss.sum().backward()
    return loss.detach(), [q.grad for q in ps]


@pytest.mark.parametrize("manual", [False, True])
@pytest.mark.parametrize("tied", [False, True])
def test_a_distillation_step(tied, manual):
    N, V, D, T, k = 60, 700, 48, 2.0, 12
    g = torch.Generator().manual_seed(3)
    params = student(1, V, D, torch.float32)
    tokens = torch.randint(0, 40, (N,), generator=g).to(DEV)
    tokens[5] = tokens[50] = -1
    history = torch.randint(0, V, (N, 30), generator=g).to(DEV)
    on = (torch.rand(N, V, generator=g) < 0.8).to(DEV)
    teacher = scores.token_scores(scores.adjust_logits(4 * torch.randn(N, V, generator=g).to(DEV), allowed=on), top=k, temperature=T)
    w = torch.rand(N, generator=g).to(DEV) / N
    w[9] = 0.0
    args = (tokens, history, words_of(on), teacher.top_ids, teacher.top_log_probs, w, T)
    loss = steps(params, *args, manual)
    want, grads = in_64_bits(params, tokens, history, on, *args[3:])
    # float32 matrix products of D or V terms: errors of some 1e-6 of the values' size
    assert torch.allclose(loss.double().cpu(), want, rtol=2e-5, atol=1e-7)
    mine = [p.grad for p in params]
    if tied:  # one matrix at both ends: the embedding's gradient goes on top of the output's
        rows = torch.autograd.grad(train.embedding(params[0], tokens, scale=2.0), params[0],
                                   torch.ones(N, D, device=DEV))[0]
        both = mine[2].clone()
        train.embedding_grad(tokens, torch.ones(N, D, device=DEV), scale=2.0, out=both, add=True)
        assert torch.allclose(both, mine[2] + rows, rtol=1e-6, atol=1e-9)
    for a, b in zip(mine, grads):
        assert torch.allclose(a.double().cpu(), b, rtol=1e-4, atol=2e-5 * float(b.abs().max()))
    before = [x.double().cpu() for x in mine]
    norm = train.clip_grad_norm(mine, 0.01)
    size = torch.sqrt(sum((b * b).sum() for b in before))
    assert abs(float(norm) - float(size)) <= 1e-6 * float(size)
    for a, b in zip(mine, before):
        assert torch.allclose(a.double().cpu(), b * min(1.0, 0.01 / (float(size) + 1e-6)), rtol=1e-6, atol=0)


def test_a_step_in_a_graph():
    """A whole step with its gradients, captured, replayed with new tokens between eager ones."""
    N, V, D, k = 40, 300, 32, 6
    g = torch.Generator().manual_seed(4)
    params = student(2, V, D, torch.bfloat16)
    teacher = scores.token_scores(torch.randn(N, V, generator=g).to(DEV), top=k)
    on = words_of((torch.rand(V, generator=g) < 0.9).to(DEV))
    w = torch.full((N,), 1.0 / N, device=DEV)
    static = torch.randint(0, V, (N,), generator=g).to(DEV)

    def work(tokens):
        leaves = [p.detach().requires_grad_() for p in params]
        hidden = train.embedding(leaves[0], tokens)
        z = torch.tanh(hidden @ leaves[1]) @ leaves[2].t()
        x = scores.adjust_logits(z, history=tokens[:, None].expand(N, 3), repetition=1.2, presence=0.5, allowed=on)
        loss, grad = scores.distill_loss_and_grad(x.detach(), teacher.top_ids, teacher.top_log_probs, w)
        grads = torch.autograd.grad([x], leaves, [grad])
        norm = train.clip_grad_norm(grads, 0.05)
        return loss, norm, *grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(static)
    for i in range(3):
        fresh = torch.randint(0, V, (N,), generator=g).to(DEV)
        want = work(fresh)
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_a_constrained_decoder():
    """Greedy steps of several streams: what was said is penalised, what the grammar
    forbids is never taken."""
    R, V, H = 5, 1000, 20
    g = torch.Generator().manual_seed(6)
    rows = 2 * torch.randn(H, R, V, generator=g).to(DEV)
    history = torch.full((R, H), -1, device=DEV)
    for t in range(H):
        on = torch.rand(R, V, generator=g).to(DEV) < 0.02
        z = rows[t].clone()
        scores.adjust_logits(z, history=history, repetition=1.5, frequency=5.0, allowed=words_of(on), out=z)
        got = scores.token_scores(z, top=1)
        want = rows[t].double()
        for i in range(R):
            for j in set(history[i, :t].tolist()):
                x = want[i, j]
                want[i, j] = (x / 1.5 if x > 0 else x * 1.5) - 5.0 * int((history[i, :t] == j).sum())
        want[~on] = -torch.inf
        assert torch.equal(got.top_ids[:, 0].long(), want.argmax(1))
        history[:, t] = got.top_ids[:, 0]
