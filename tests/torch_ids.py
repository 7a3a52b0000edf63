"""Ids over the whole range of their types, in histories, biases and embeddings: those of
the vocabulary count, whatever the others have in common with them in 32 bits.  Run by
test_gpu_adjust_forms.py in a process of its own."""
import numpy as np
import pytest
import torch  # first: the library shares its HIP runtime

import adjust64
from detllm_amd import scores, train

pytestmark = pytest.mark.gpu
V = 5000
NONE = [-1, V, -(2**63), 2**63 - 1, -(2**63) + 7, 2**63 - V, 2**32, 2**32 + 3, -(2**32) + 3, 2**31, -(2**31), 2**31 + 2048,
        -(2**63) + 4096, 2**62 + 2048]
NONE_32 = [-1, V, -(2**31), 2**31 - 1, -(2**31) + 7, 2**31 - V]


@pytest.mark.parametrize("index", [torch.int64, torch.int32], ids=str)
def test_histories_and_biases(index):
    none = NONE if index == torch.int64 else NONE_32
    ids = torch.tensor([*none, 0, 3, 7, 2048, 4096, V - 1, 3], dtype=index)
    z = torch.randn(2, V, generator=torch.Generator().manual_seed(1))
    for rows in (2, 700):  # segments of 2048, and of 8192
        x = z.repeat(rows // 2, 1).cuda()
        got = scores.adjust_logits(x, history=ids.cuda(), repetition=1.5, frequency=0.25, bias_ids=ids.cuda(),
                                   bias=torch.arange(1.0, ids.numel() + 1).cuda())
        for i in range(2):
            want, tol = adjust64.adjust(z[i], "f32", ids, 0, 1.5, 0.0, 0.25, ids, np.arange(1.0, ids.numel() + 1))
            assert adjust64.same(got[i].cpu(), want, tol).all() and (want != z[i].numpy()).sum() == 6
            assert torch.equal(got[i::2], got[i].expand(rows // 2, V))


@pytest.mark.parametrize("n", [30, 3000, 9000])
def test_embeddings(n):
    real = torch.tensor([0, 3, V - 1, 7, 511, 512, 2048]).repeat(n // 7)
    tokens = torch.cat([torch.tensor(NONE), real])
    tokens = tokens[torch.randperm(tokens.numel(), generator=torch.Generator().manual_seed(n))].cuda()
    w = torch.arange(V, device="cuda").float()[:, None].expand(V, 5).contiguous()
    rows = train.embedding(w, tokens)
    inside = (tokens >= 0) & (tokens < V)
    assert torch.equal(rows[inside], tokens[inside, None].float().expand(-1, 5))
    assert (rows[tokens < 0] == 0).all() and rows[tokens >= V].isnan().all()
    g = torch.full((tokens.numel(), 5), float("nan"), device="cuda")
    g[inside] = 1.0
    got = train.embedding_grad(tokens, g, V)
    assert torch.equal(got[:, 0], torch.bincount(tokens[inside], minlength=V).float()) and torch.equal(got, got[:, :1].expand(V, 5))
