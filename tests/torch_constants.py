"""Calls of detllm_amd.train that autograd does not see refuse what needs a gradient,
whose result would be cut off without a word.  Run by test_gpu_train_forms.py in a
process of its own."""
import pytest
import torch  # first: the library shares its HIP runtime

from detllm_amd import train

pytestmark = pytest.mark.gpu


def test_rows_of_an_embedding_gradient():
    g = torch.randn(5, 6, device="cuda")
    tokens = torch.tensor([1, 0, 3, 1, -1], device="cuda")
    want = train.embedding_grad(tokens, g, 4)
    leaf = g.clone().requires_grad_()
    for x in (leaf, leaf * 1):
        for kw in ({}, dict(out=torch.zeros(4, 6, device="cuda")), dict(out=torch.zeros(4, 6, device="cuda"), add=True)):
            with pytest.raises(ValueError, match="grad is a constant"):
                train.embedding_grad(tokens, x, 4, **kw)
        assert torch.equal(train.embedding_grad(tokens, x.detach(), 4), want)
        for mode in (torch.no_grad, torch.inference_mode):  # where nothing is recorded
            with mode():
                assert torch.equal(train.embedding_grad(tokens, x, 4), want)


def test_a_scale():
    grads = [torch.randn(50, device="cuda"), torch.randn(7, device="cuda").bfloat16()]
    scale = torch.tensor(0.25, device="cuda")
    leaf = scale.clone().requires_grad_()
    calls = (lambda s: train.grad_norm(grads, scale=s),
             lambda s: train.clip_grad_norm(grads, 0.5, scale=s, out=[torch.empty_like(t) for t in grads]))
    for call in calls:
        want = call(scale)
        for s in (leaf, leaf * 1):
            with pytest.raises(ValueError, match="scale is a constant"):
                call(s)
            assert torch.equal(call(s.detach()), want)
            with torch.no_grad():
                assert torch.equal(call(s), want)
    before = [t.clone() for t in grads]
    with pytest.raises(ValueError):
        train.clip_grad_norm(grads, 0.5, scale=leaf)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_a_vocabulary_beside_out():
    g, tokens, out = torch.randn(3, 6, device="cuda"), torch.tensor([1, 0, 3], device="cuda"), torch.ones(4, 6, device="cuda")
    for vocab in (0, 3, 5, -4):
        with pytest.raises(ValueError):
            train.embedding_grad(tokens, g, vocab, out=out)
    assert (out == 1).all()
    assert torch.equal(train.embedding_grad(tokens, g, 4, out=out.clone()), train.embedding_grad(tokens, g, out=out.clone()))
