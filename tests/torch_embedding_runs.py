"""Embedding gradients whose tokens' runs cross the stretches and groups of the sorted
list: stretches of 8 to 64 positions, runs through hundreds of groups.  Run by
test_gpu_train_forms.py in a process of its own."""
import pytest
import torch  # first: the library shares its HIP runtime

from detllm_amd import train

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}


def runs(n, V, long, seed):
    """n tokens of a vocabulary of V, shuffled.  In order: single tokens, runs of every
    length up to 150 so that they begin and end at every place of a stretch, then one of
    `long` between two more of them, and what is left shared by a few; about 1 % are
    padding or no tokens."""
    none = n // 100 + 3
    lengths, left, k = [], n - none - long, 0
    while left > 0 and len(lengths) < V - 4:
        k += 1
        lengths.append(min(left, 1 if k % 3 else (7 * k) % 150 + 1))
        left -= lengths[-1]
    lengths.insert(len(lengths) // 2, long)
    lengths += [left - left // 3, left // 3]
    tokens = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
    odd = torch.tensor([-1, V, -7, V + 100])[torch.arange(none) % 4]
    tokens = torch.cat([tokens, odd])
    assert tokens.numel() == n and int(tokens.max()) >= V and len(lengths) <= V
    return tokens[torch.randperm(n, generator=torch.Generator().manual_seed(seed))].to(DEV)


def summed(tokens, g, V):
    """The sums of each token's rows in 64 bits, and of their magnitudes, and how many."""
    real = (tokens >= 0) & (tokens < V)
    at = torch.where(real, tokens, V).long()
    times = torch.bincount(at, minlength=V + 1)[:-1]
    often = (times > 200).nonzero().flatten().tolist()
    few = ~torch.isin(at, torch.tensor([*often, V], device=DEV))
    both = []
    for x in (g.double(), g.double().abs()):
        out = torch.zeros(V, g.shape[1], dtype=torch.float64, device=DEV).index_add_(0, at[few], x[few])
        for t in often:  # many additions to one place take long
            out[t] = x[at == t].sum(0)
        both.append(out)
    return *both, times


CASES = [  # tokens, vocabulary, the type's 16-byte packets of a row, longest run
    (20011, 3000, 40, 5003),  # stretches of 8, groups of 128
    (60013, 900, 5, 40009),  # of 8 and 256
    (300007, 5000, 1, 290003),  # of 8 and 2048
    (70003, 2000, 128, 36007),  # of 16 and 256
    (1000003, 4000, 9, 200003),  # of 16 and 256
    (140001, 3000, 127, 60001),  # of 32 and 512
    (280003, 3000, 125, 150001),  # of 64 and 1024
    (1 << 20, 200000, 33, 100003),  # of 64 and 1024
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", CASES, ids=lambda s: "x".join(map(str, s)))
def test_whole_numbers(shape, dtype):
    """Sums of small whole numbers are exact in any order: only the type's rounding is left."""
    n, V, packets, long = shape
    D = packets * (4 if dtype == "f32" else 8) - (1 if packets > 1 else 0)
    tokens = runs(n, V, long, n)
    g = torch.randint(-3, 5, (n, D), generator=torch.Generator(device=DEV).manual_seed(n), device=DEV).to(TYPES[dtype])
    want, size, times = summed(tokens, g, V)
    assert float(size.max()) < 2**24 and int(times.max()) >= long
    got = train.embedding_grad(tokens, g, V)
    assert torch.equal(got, want.float().to(TYPES[dtype]))
    old = torch.randint(-9, 10, (V, D + 3), device=DEV).float()[:, :D]
    out = old.clone()
    train.embedding_grad(tokens.int(), g, scale=0.5, out=out, add=True)
    assert torch.equal(out, (old.double() + 0.5 * want).float())
    leaf = torch.zeros(V, D, dtype=TYPES[dtype], device=DEV, requires_grad=True)
    grad, = torch.autograd.grad(train.embedding(leaf, tokens, scale=2.0), leaf, g)
    assert torch.equal(grad, (2.0 * want).float().to(TYPES[dtype]))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", CASES[:6] + [(200000, 500, 1, 190000)], ids=lambda s: "x".join(map(str, s)))
def test_roundings_of_a_long_run(shape, dtype):
    """A token's rows are added in 32 bits within a stretch (at most 64) and along a group's
    stretches (at most 256), then in 64: at most 320 roundings of the magnitudes' sum, one of
    the joined sum, one of the product.  That is far from what a sum without some rows is."""
    n, V, packets, long = shape
    D = packets * (4 if dtype == "f32" else 8)
    tokens = runs(n, V, long, n + 1)
    g = (0.3 + torch.randn(n, D, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)).to(TYPES[dtype])
    want, size, times = summed(tokens, g, V)
    want, size = want * 0.7, size * 0.7
    tol = 1.01 * 2.0**-24 * (times.clamp(max=320) + 2)[:, None] * size + 1.01 * 2.0**-24 * want.abs()  # 0.7 in 32 bits
    most = times.argmax()
    assert float((tol / want.abs())[most].max()) < 2e-4
    for out in (None, torch.zeros(V, D, device=DEV)):
        got = train.embedding_grad(tokens, g, V, scale=0.7, out=out)
        half = HALF["f32" if out is not None else dtype]
        over = 65504.0 if got.dtype == torch.float16 else float("inf")
        fits = want.abs() < over
        assert bool((((got.double() - want).abs() <= tol + want.abs() * half + 2.0**-25) | ~fits).all())
        assert bool((got[~fits].isinf() | (got[~fits].abs() == over)).all())
