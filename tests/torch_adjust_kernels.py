"""Every kernel that adjust_logits and its gradient choose among: copied, in place or a
gradient; with lists or a mask alone; segments of 2048, 8192 and 16384 logits; results
within the memory-side cache and past it.  Run by test_gpu_adjust_forms.py in a process
of its own."""
import numpy as np
import pytest
import torch  # first: the library shares its HIP runtime

import adjust64
from detllm_amd import scores
from torch_adjust import TYPES, case, check, host, words_of

DEV = "cuda"


def same_bits(a, b):
    bits = torch.int32 if a.dtype == torch.float32 else torch.int16
    return torch.equal(a.contiguous().view(bits), b.contiguous().view(bits))


LISTS = [  # rows, vocabulary, history, biases, stride: segments of 2048 twice, 8192 twice, 16384 twice
    (5, 4095, 6000, 7, 4097), (3, 20001, 300, 0, 20005),
    (66, 33003, 300, 5, 33005), (130, 16411, 4096, 0, 16411),
    (3, 20001, 5000, 9, 20003), (2, 40007, 4097, 0, 40007),
]


@pytest.mark.parametrize("mask", ["", "bits", "bytes"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", LISTS, ids=lambda s: "x".join(map(str, s)))
def test_lists(shape, dtype, mask):
    R, V, H, K, stride = shape
    z, kw, rows = case(R + V, R, V, dtype, H, K, mask, per_row=R % 2 == 1, stride=stride)
    leaf = z.detach().requires_grad_()
    got = scores.adjust_logits(leaf, **kw)
    check(z, kw, rows, dtype, got)
    g = torch.randn(R, V, generator=torch.Generator(device=DEV).manual_seed(V), device=DEV).to(z.dtype)
    if mask:  # whatever is there where nothing is allowed
        on = torch.stack([torch.from_numpy(r["allowed"]) for r in rows]).to(DEV)
        g = torch.where(~on & (torch.arange(V, device=DEV) % 3 == 0), float("nan"), g)
    grad, = torch.autograd.grad(got, leaf, g)
    for i, r in enumerate(rows):
        want, tol = adjust64.gradient(host(z)[i], host(g)[i], dtype, r["history"], r["theta"], r.get("allowed"))
        got_i = host(grad[i])
        ok = adjust64.same(got_i, want, tol)
        assert ok.all(), (i, np.flatnonzero(~ok)[:5], got_i[~ok][:5], want[~ok][:5])
    wide = torch.full((R, stride + 3), 7.0, dtype=z.dtype, device=DEV)
    mine = wide[:, :V]
    mine.copy_(z)
    scores.adjust_logits(mine, **kw, out=mine)
    assert same_bits(mine, got.detach()) and (wide[:, V:] == 7.0).all()


@pytest.mark.parametrize("form", ["bits", "bytes", "shared"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(3, 1, 5), (7, 31, 33), (4, 4093, 4099), (2, 30011, 30011), (70, 30011, 30013), (9, 262141, 262144)],
                         ids=lambda s: "x".join(map(str, s)))
def test_a_mask_alone(shape, dtype, form):
    """Bits are kept or become -inf (0 in a gradient), whatever they are."""
    R, V, stride = shape
    g = torch.Generator(device=DEV).manual_seed(R * V)
    buf = torch.randint(-(2**15), 2**15, (R, stride * (2 if dtype == "f32" else 1)), generator=g, device=DEV).short()
    whole = buf.view(TYPES[dtype])  # every kind of number, no number among them
    z = whole[:, :V]
    # rows with next to nothing, half and nearly everything allowed; none, all
    share = torch.tensor([0.01, 0.5, 0.97, 0.8, 0.0, 1.0], device=DEV)[torch.arange(R, device=DEV) % 6]
    on = torch.rand(R, V, generator=g, device=DEV) < share[:, None]
    if form == "shared":
        on = on[-1:].expand(R, V)
    allowed = on[0] if form == "shared" else on
    allowed = words_of(allowed) if form != "bytes" else allowed.contiguous()
    want = torch.where(on, z, -torch.inf)
    between = whole[:, V:].clone()
    leaf = z.clone().requires_grad_()
    got = scores.adjust_logits(leaf, allowed=allowed)
    assert same_bits(got.detach(), want)
    grad, = torch.autograd.grad(got, leaf, z.contiguous())
    assert same_bits(grad, torch.where(on, z, 0.0))
    scores.adjust_logits(z, allowed=allowed, out=z)
    assert same_bits(z, want) and same_bits(whole[:, V:], between)


def rounds_within(got, want, tol, dtype):
    """|got - want| <= tol and the type's rounding, in 64 bits on the device."""
    half, least = adjust64.ROUND[dtype]
    return bool(((got.double() - want).abs() <= tol + want.abs() * half + least).all())


@pytest.mark.parametrize("shape", [("f32", 1030, 65543, 200), ("bf16", 600, 262143, 300), ("f16", 520, 261001, 5000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_past_the_cache(shape):
    """More than 256 MB of results."""
    dtype, R, V, H = shape
    g = torch.Generator(device=DEV).manual_seed(V)
    z = (4 * torch.randn(R, V, generator=g, device=DEV)).to(TYPES[dtype])
    assert z.numel() * z.element_size() > 256 << 20
    history = torch.randint(-1, V, (R, H), generator=g, device=DEV)
    history[:, ::7] = history[:, :1]
    on = torch.rand(V, generator=g, device=DEV) < 0.7
    theta, presence, frequency = 1.5, 0.25, 0.5  # exact in 32 bits
    kw = dict(history=history, repetition=theta, presence=presence, frequency=frequency, allowed=words_of(on))
    leaf = z.requires_grad_()
    out = scores.adjust_logits(leaf, **kw)
    gr = torch.randn(R, V, generator=g, device=DEV).to(z.dtype)
    grad, = torch.autograd.grad(out, leaf, gr)
    z, out = z.detach(), out.detach()
    for part in torch.arange(R).split(64):
        x, h = z[part].double(), history[part]
        at = torch.where(h < 0, V, h)
        n = torch.zeros(len(part), V + 1, dtype=torch.float64, device=DEV)
        n.scatter_add_(1, at, torch.ones(h.shape, dtype=torch.float64, device=DEV))
        n = n[:, :V]
        a = torch.where(n > 0, torch.where(x > 0, x / theta, x * theta), x)
        less = torch.where(n > 0, presence + frequency * n, 0.0)
        off = torch.where(n > 0, 1.01 * 2.0**-24 * (a.abs() + (a - less).abs()), 0.0)  # counts and their terms are exact
        got = out[part]
        assert (got[:, ~on] == -torch.inf).all()
        assert rounds_within(got[:, on], (a - less)[:, on], off[:, on], dtype)
        d = torch.where(n > 0, torch.where(x > 0, gr[part].double() / theta, gr[part].double() * theta), gr[part].double())
        d = torch.where(on, d, 0.0)
        assert rounds_within(grad[part], d, 1.01 * 2.0**-24 * d.abs(), dtype)
    scores.adjust_logits(z, **kw, out=z)
    assert same_bits(z, out)
