"""adjust_logits and detllm_amd.train under torch's other ways to differentiate,
transform, record and checkpoint: refused, or right.  Run by test_gpu_train.py in a
process of its own."""
import pytest
import torch  # first: the library shares its HIP runtime
from torch.autograd import forward_ad

from detllm_amd import scores, train

GPU, CPU = torch.device("cuda"), torch.device("cpu")


def calls(dev):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 50, generator=g).to(dev)
    h = torch.randint(0, 50, (6, 9), generator=g).to(dev)
    tokens = torch.randint(0, 6, (11,), generator=g).to(dev)
    return x, {"adjust": lambda t: scores.adjust_logits(t, history=h, repetition=1.5),
               "embed": lambda t: train.embedding(t, tokens),
               "embed_grad": lambda t: train.embedding_grad(tokens[:6], t, 7),
               "norm": lambda t: train.grad_norm([t.detach() if not forward_ad._current_level >= 0 else t])}


def tangents(dev):
    x, fs = calls(dev)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for f in fs.values():
            with pytest.raises(NotImplementedError):
                f(dual)


def traced(dev):
    x, fs = calls(dev)
    for f in fs.values():
        with pytest.raises(RuntimeError, match="torch.jit.trace"):
            torch.jit.trace(f, (x,), check_trace=False)


def test_tangents_and_traces_are_refused_before_the_device_is_looked_at():
    tangents(CPU)
    traced(CPU)


@pytest.mark.gpu
def test_tangents_and_traces():
    tangents(GPU)
    traced(GPU)
    x, fs = calls(GPU)
    with forward_ad.dual_level():  # of the other tensors, and of a backward's gradient
        one = forward_ad.make_dual(torch.ones(6, device=GPU), torch.ones(6, device=GPU))
        with pytest.raises(NotImplementedError):
            scores.adjust_logits(x, history=torch.zeros(6, 1, dtype=torch.long, device=GPU), presence=one)
        leaf = x.clone().requires_grad_()
        for name in ("adjust", "embed"):
            out = fs[name](leaf)
            dual = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(out, leaf, dual)


@pytest.mark.gpu
def test_transforms_are_refused():
    x, fs = calls(GPU)
    for name in ("adjust", "embed"):
        f = fs[name]
        for transformed in (lambda: torch.func.vmap(f)(x.expand(2, 6, 50)), lambda: torch.func.jvp(f, (x,), (x,)),
                            lambda: torch.func.grad(lambda t: f(t).sum())(x)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                transformed()


@pytest.mark.gpu
def test_checkpoints_and_saved_tensors_that_move():
    from torch.utils.checkpoint import checkpoint

    x, fs = calls(GPU)
    for name in ("adjust", "embed"):
        leaf = x.clone().requires_grad_()
        want, = torch.autograd.grad(fs[name](leaf).square().sum(), leaf)
        got, = torch.autograd.grad(checkpoint(lambda t: fs[name](t).square().sum(), leaf, use_reentrant=False), leaf)
        assert torch.equal(got, want)
        with torch.autograd.graph.save_on_cpu():
            out = fs[name](leaf).square().sum()
        got, = torch.autograd.grad(out, leaf)
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_where_the_caller_stands():
    """Under inference_mode and no_grad, accumulated twice, and a graph kept for a second pass."""
    x, fs = calls(GPU)
    want = {k: f(x) for k, f in fs.items()}
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            for k, f in fs.items():
                assert torch.equal(f(x), want[k])
    for name in ("adjust", "embed"):
        leaf = x.clone().requires_grad_()
        out = fs[name](leaf)
        g = torch.randn_like(out)
        once, = torch.autograd.grad(out, leaf, g, retain_graph=True)
        out.backward(g, retain_graph=True)
        out.backward(g)
        assert torch.equal(leaf.grad, once + once)


@pytest.mark.gpu
def test_beside_a_compiled_function():
    x, fs = calls(GPU)
    for name in ("adjust", "embed"):
        f = torch.compiler.disable(fs[name])

        @torch.compile(backend="eager")
        def run(t):
            return f(t * 2).sum()

        leaf = x.clone().requires_grad_()
        got, = torch.autograd.grad(run(leaf), leaf)
        want, = torch.autograd.grad(fs[name](leaf * 2).sum(), leaf)
        assert torch.equal(got, want)
