"""Where adjust_logits' prompt ends, over the whole range of its types.  Run by
test_gpu_adjust_forms.py in a process of its own."""
import pytest
import torch  # first: the library shares its HIP runtime

import adjust64
from detllm_amd import scores

# before the history, in it, at its end, and past what 32 bits hold on both sides
PLACES = [0, 3, 5, 6, -1, -(2**31), -(2**31) - 1, -(2**40), -(2**63), 2**31 - 1, 2**31, 2**32, 2**32 + 2, 2**40, 2**63 - 1]


def test_places_are_narrowed_to_those_of_the_history():
    z = torch.zeros(len(PLACES), 9)
    for index in (torch.int64, torch.int32):
        for history in (torch.zeros(len(PLACES), 5, dtype=index), torch.zeros(5, dtype=index)):
            by = scores._By(z, 9, history, torch.tensor(PLACES), 1.0, 0.0, 0.0, None, None, None)
            held = by.tensors[1]
            assert held.dtype == torch.int32 and held.tolist() == [min(max(p, 0), 5) for p in PLACES]


@pytest.mark.gpu
def test_prompts_of_any_size():
    g = torch.Generator().manual_seed(1)
    R, V = len(PLACES), 40
    z = torch.randn(R, V, generator=g)
    history = torch.randint(0, V, (R, 5), generator=g)
    for which in (slice(0, R), slice(9, 10)):  # 2^31 - 1 is in both types
        for index in (torch.int64, torch.int32):
            at = torch.tensor(PLACES)[which]
            if index == torch.int32:
                at = at.clamp(-(2**31), 2**31 - 1)
            got = scores.adjust_logits(z[which].cuda(), history=history[which].cuda(), prompt=at.to(index).cuda(), repetition=1.5,
                                       presence=0.5, frequency=0.25)
            for i, p in enumerate(at.tolist()):
                want, tol = adjust64.adjust(z[which][i], "f32", history[which][i], p, 1.5, 0.5, 0.25)
                assert adjust64.same(got[i].cpu(), want, tol).all(), p
    # every second of a longer list, one row alone
    longer = torch.tensor(PLACES).repeat_interleave(2).cuda()
    assert torch.equal(scores.adjust_logits(z.cuda(), history=history.cuda(), prompt=longer[::2], presence=0.5),
                       scores.adjust_logits(z.cuda(), history=history.cuda(), prompt=torch.tensor(PLACES).cuda(), presence=0.5))
    assert torch.equal(scores.adjust_logits(z[0].cuda(), history=history[0].cuda(), prompt=torch.tensor(2**40).cuda(), presence=0.5),
                       z[0].cuda())
