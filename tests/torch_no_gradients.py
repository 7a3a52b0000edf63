"""The norm and clipping of lists that hold no tensor, or none with elements.  Run by
test_gpu_train_forms.py in a process of its own."""
import math

import pytest
import torch  # first: the library shares its HIP runtime

from detllm_amd import train
from detllm_amd._lib import DetllmError

pytestmark = pytest.mark.gpu
EMPTY = ([], [None], (None for _ in range(3)), [torch.empty(0)], [torch.empty(0, 5), None, torch.empty(0).half()])


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("which", range(len(EMPTY)))
def test_norms_are_zeros_on_the_device(which, kind):
    def grads():
        return [t if t is None else t.cuda() for t in EMPTY[which]]

    scale = torch.tensor(-3.0, device="cuda")
    got = [train.grad_norm(grads(), norm_type=kind), train.grad_norm(grads(), norm_type=kind, scale=scale),
           train.clip_grad_norm(grads(), 1.0, norm_type=kind), train.clip_grad_norm(grads(), 0.0, scale=scale),
           train.clip_grad_norm(grads(), 1.0, out=[t for t in grads() if t is not None])]
    some = train.grad_norm(torch.ones(4, device="cuda"))
    assert torch.stack([*got, some]).tolist() == [0.0] * len(got) + [2.0]
    assert all(n.device == some.device and n.dtype == torch.float32 for n in got)


def test_what_is_refused_of_other_lists_is_refused_here():
    one = torch.ones(1, device="cuda")
    for kw, err in ((dict(norm_type=1.0), ValueError), (dict(scale=torch.ones(())), ValueError), (dict(scale=one.double()), ValueError),
                    (dict(scale=one.expand(2)), ValueError)):
        with pytest.raises(err):
            train.grad_norm([], **kw)
        with pytest.raises(err):
            train.clip_grad_norm([None], 1.0, **kw)
    with pytest.raises(ValueError):
        train.clip_grad_norm([], 1.0, out=[one])
    for max_norm in (-1.0, math.nan):
        with pytest.raises(DetllmError):
            train.clip_grad_norm([], max_norm)


def test_in_a_graph():
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train.clip_grad_norm([], 1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = train.clip_grad_norm([], 1.0)
    for i in range(3):
        got.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert float(got) == 0.0
