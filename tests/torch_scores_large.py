"""Logits and gradients beyond the memory-side cache of 256 MB, which are read and
written past it, in the types that torch_scores.py does not have there.  Run by
test_scores_torch_modes.py."""
import pytest
import torch  # first: the library shares its HIP runtime

from detllm_amd import scores

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype,R", [(torch.float32, 460), (torch.float16, 900)])
def test_rows_are_the_same_bits_past_the_cache(dtype, R, rest):
    V, k = 151937, 5
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.empty(R, V, dtype=dtype, device="cuda").normal_(generator=g).requires_grad_()
    assert z.nbytes > 256 << 20
    tokens = torch.randint(0, V, (R,), device="cuda", generator=g)
    w = torch.rand(R, device="cuda", generator=g)

    def work(rows):
        x = z[rows]
        got = scores.token_scores(x, tokens[rows], top=k)
        plain = scores.token_scores(x, tokens[rows])
        loss = scores.distill_loss(x, got.top_ids, got.top_log_probs - 0.2, rest=rest)
        d, = torch.autograd.grad([plain.log_probs, plain.entropy], [x], [w[rows], -w[rows]], retain_graph=True)
        e, = torch.autograd.grad([loss], [x], [w[rows]])
        step = scores.distill_loss_and_grad(x.detach(), got.top_ids, got.top_log_probs - 0.2, w[rows], rest=rest)
        assert torch.equal(step[1], e)
        return [t.detach() for t in (*got, plain.log_probs, plain.entropy, loss, d, e, *step)]

    whole = work(slice(None))
    for rows in (slice(0, 3), slice(R // 2, R // 2 + 130), slice(R - 2, R)):  # in parts and by whole rows
        for a, b in zip(whole, work(rows)):
            assert torch.equal(a[rows], b)
