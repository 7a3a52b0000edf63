"""The norm and clipping of lists that do not fit the memory-side cache, and of norms at
the end of 32 bits.  Run by test_gpu_train_forms.py in a process of its own."""
import math

import pytest
import torch  # first: the library shares its HIP runtime

from adjust64 import ROUND
from detllm_amd import train

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NAME = {v: k for k, v in TYPES.items()}
LISTS = {  # element counts and types, more than 256 MB each
    "one": [(150_000_001, "bf16")],  # in place more pieces than workgroups
    "mixed": [(40_000_003, "bf16"), (3, "f32"), (30_000_001, "f32"), (0, "f16"), (70_000_007, "f16"), (1, "bf16")],
    "many": [(300_007 + k, ("f16", "f32", "bf16")[k % 3]) for k in range(500)],  # several launches, the last 192 MB cached
    "small_last": [(140_000_000, "f16"), *[(5, "f32")] * 300],
}


def lists(name):
    g = torch.Generator(device=DEV).manual_seed(len(name))
    return [torch.randn(n, generator=g, device=DEV).mul_(0.01 * (1 + k % 5)).to(TYPES[d]) for k, (n, d) in enumerate(LISTS[name])]


def norm_of(tensors, largest):
    if largest:
        return max(float(t.abs().max()) for t in tensors if t.numel())
    return math.sqrt(math.fsum(float(p.double().square().sum()) for t in tensors for p in t.split(1 << 25)))


def scaled(t, out, c):
    """out = t c: c's rounding to 32 bits, the product's, and the type's."""
    half, least = ROUND[NAME[out.dtype]]
    for a, b in zip(t.split(1 << 25), out.split(1 << 25)):
        want = a.double() * c
        assert bool(((b.double() - want).abs() <= want.abs() * (1.01 * 2.0**-23 + half) + least + 2.0**-149).all())


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("name", list(LISTS))
def test_past_the_cache(name, kind):
    grads = lists(name)
    assert sum(t.numel() * t.element_size() for t in grads) > 256 << 20
    scale = -0.5
    want = 0.5 * norm_of(grads, kind == math.inf)
    norm = train.grad_norm(grads, norm_type=kind, scale=scale)
    assert abs(float(norm) - want) <= 1.01 * 2.0**-24 * want
    for max_norm in (want / 3, 2 * want):
        c = scale * min(1.0, max_norm / (want + 1e-6))
        outs = [torch.full_like(t, 9.0) for t in grads]
        assert torch.equal(train.clip_grad_norm(grads, max_norm, norm_type=kind, scale=scale, out=outs), norm)
        [scaled(t, o, c) for t, o in zip(grads, outs)]
        wide = [torch.full(t.shape, 9.0, device=DEV) for t in grads]
        assert torch.equal(train.clip_grad_norm(grads, max_norm, norm_type=kind, scale=scale, out=wide), norm)
        [scaled(t, o, c) for t, o in zip(grads, wide)]
        mine = [t.clone() for t in grads]
        assert torch.equal(train.clip_grad_norm(mine, max_norm, norm_type=kind, scale=scale), norm)
        assert all(torch.equal(a, b) for a, b in zip(mine, outs))
        same = [t.clone() for t in grads]  # a list given as its own output
        assert torch.equal(train.clip_grad_norm(same, max_norm, norm_type=kind, scale=scale, out=same), norm)
        assert all(torch.equal(a, b) for a, b in zip(same, outs))
    mine = [t.clone() for t in grads]  # nothing to clip
    train.clip_grad_norm(mine, 4 * want, norm_type=kind)
    assert all(torch.equal(a, b) for a, b in zip(mine, grads))
    outs = [torch.full_like(t, 9.0) for t in grads]
    train.clip_grad_norm(grads, 4 * want, norm_type=kind, out=outs)
    assert all(torch.equal(a, b) for a, b in zip(outs, grads))


def test_a_norm_past_32_bits():
    """Finite gradients whose norm is not: it is given as infinity, the factor is that of
    the norm in 64 bits."""
    n = 10000
    g = [torch.full((n,), 3e38, device=DEV), torch.full((7,), -3e38, device=DEV)]
    want = norm_of(g, False)
    assert want > torch.finfo(torch.float32).max
    assert float(train.grad_norm(g)) == math.inf
    mine = [t.clone() for t in g]
    assert float(train.clip_grad_norm(mine, 1e5)) == math.inf
    c = 1e5 / want
    assert c > 2.0**-126
    [scaled(t, o, c) for t, o in zip(g, mine)]
    mine = [t.clone() for t in g]  # a factor among the smallest numbers is off by half a step of theirs
    train.clip_grad_norm(mine, 1.0)
    assert all(torch.allclose(o.double(), t.double() / want, rtol=2.0**-150 * want + 1e-7, atol=0) for t, o in zip(g, mine))
    assert float(train.grad_norm(g, scale=1e-10)) == pytest.approx(1e-10 * want, rel=1e-6)
