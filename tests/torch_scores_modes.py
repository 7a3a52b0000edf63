"""detllm_amd.scores under torch's other ways to differentiate, transform and
record: refused, or right.  Run by test_scores_torch_modes.py in a process of its
own, where torch's HIP runtime is the one the library takes."""
import pytest
import torch  # first: the library shares its HIP runtime
from torch.autograd import forward_ad

from detllm_amd import scores

GPU = torch.device("cuda")
CPU = torch.device("cpu")


def inputs(dev):
    z = torch.randn(3, 50, generator=torch.Generator().manual_seed(1)).to(dev)
    ids = torch.arange(6, dtype=torch.int32, device=dev).repeat(3, 1)
    return z, ids, torch.full((3, 6), -2.0, device=dev)


def calls(z, ids, v):
    return (lambda x: scores.token_scores(x, top=1).entropy, lambda x: scores.distill_loss(x, ids, v),
            lambda x: scores.distill_loss_and_grad(x, ids, v)[0])


def tangents(dev):
    z, ids, v = inputs(dev)
    with forward_ad.dual_level():
        for leaf in (z, z.clone().requires_grad_()):
            dual = forward_ad.make_dual(leaf, torch.ones_like(z))
            for x in (dual, dual[1:], dual * 2):
                for f in calls(x, ids[:x.shape[0]], v[:x.shape[0]]):
                    with pytest.raises(NotImplementedError):
                        f(x)
                    with torch.no_grad(), pytest.raises(NotImplementedError):
                        f(x)


def traced(dev):
    z, ids, v = inputs(dev)
    for leaf in (z, z.clone().requires_grad_()):
        for f in calls(z, ids, v):
            with pytest.raises(RuntimeError, match="torch.jit.trace"):
                torch.jit.trace(f, (leaf,), check_trace=False)


def test_tangents_and_traces_are_refused_before_the_device_is_looked_at():
    tangents(CPU)
    traced(CPU)


@pytest.mark.gpu
def test_tangents_and_traces():
    tangents(GPU)
    traced(GPU)
    z, ids, v = inputs(GPU)
    with forward_ad.dual_level():  # of the other tensors, and of a backward's gradients
        dual = forward_ad.make_dual(v, v)
        w = forward_ad.make_dual(torch.ones(3, device=GPU), torch.ones(3, device=GPU))
        for call in (lambda: scores.distill_loss(z, ids, dual), lambda: scores.distill_loss_and_grad(z, ids, v, w)):
            with pytest.raises(NotImplementedError):
                call()
        leaf = z.clone().requires_grad_()
        for out in (scores.token_scores(leaf).entropy, scores.distill_loss(leaf, ids, v)):
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(out, leaf, w)
        # tensors without a tangent are what they always are
        assert torch.equal(scores.token_scores(z).entropy, scores.token_scores(leaf).entropy.detach())
    assert scores.token_scores(z).entropy.isfinite().all()


@pytest.mark.gpu
def test_transforms_are_refused():
    z, ids, v = inputs(GPU)
    for f in calls(z, ids, v):
        for transformed in (lambda: torch.func.vmap(f)(z.expand(2, 3, 50)), lambda: torch.func.jvp(f, (z,), (z,)),
                            lambda: torch.func.grad(lambda x: f(x).sum())(z)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                transformed()
    leaf = z.clone().requires_grad_()
    for out in (scores.token_scores(leaf).entropy, scores.distill_loss(leaf, ids, v)):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, leaf, torch.eye(3, device=GPU), is_grads_batched=True)


@pytest.mark.gpu
def test_saved_tensors_through_hooks():
    """Kept on the host between forward and backward, and made again by checkpointing."""
    from torch.utils.checkpoint import checkpoint

    z, ids, v = inputs(GPU)
    tokens = torch.arange(3, device=GPU)

    def loss(x):
        got = scores.token_scores(x, tokens, top=2)
        return got.log_probs.sum() + 0.5 * got.entropy.sum() + scores.distill_loss(x * 1, ids, v, rest=True).sum()

    leaf = z.clone().requires_grad_()
    want, = torch.autograd.grad(loss(leaf), leaf)
    with torch.autograd.graph.save_on_cpu():
        out = loss(leaf)
    got, = torch.autograd.grad(out, leaf)
    assert torch.equal(got, want)
    got, = torch.autograd.grad(checkpoint(loss, leaf, use_reentrant=False), leaf)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_out_over_a_part_of_the_logits_is_refused():
    from detllm_amd._lib import DetllmError

    wide = torch.randn(4, 100, device=GPU)
    ids, v = torch.arange(6, dtype=torch.int32, device=GPU).repeat(3, 1), torch.full((3, 6), -2.0, device=GPU)
    for z, out in ((wide[:3, :50], wide[:3, 1:51]), (wide[:3], wide[1:]), (wide[:3, :50], wide.view(-1)[:150].view(3, 50))):
        with pytest.raises(DetllmError) as e:
            scores.distill_loss_and_grad(z, ids, v, out=out)
        assert e.value.status == 42
    want = scores.distill_loss_and_grad(wide[:3, :50], ids, v)[1]
    _, got = scores.distill_loss_and_grad(wide[:3, :50], ids, v, out=wide[:3, 50:])
    assert torch.equal(got, want) and torch.equal(wide[:3, 50:], want)
    scores.distill_loss_and_grad(wide[:3, :50], ids, v, out=wide[:3, :50])
    assert torch.equal(wide[:3, :50], want)


@pytest.mark.gpu
def test_inside_a_compiled_function():
    z, ids, v = inputs(GPU)

    @torch.compiler.disable
    def calls_of_the_library(x):
        return scores.token_scores(x, top=2).entropy.sum() + scores.distill_loss(x, ids, v, rest=True).sum()

    def loss(x):
        return calls_of_the_library(x * 2) + x.sum()

    leaf = z.clone().requires_grad_()
    want = loss(leaf)
    got = torch.compile(loss, backend="eager")(leaf)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got, leaf)[0], torch.autograd.grad(want, leaf)[0])
