"""The operators around the scores and losses as cases that can be timed and
compared: what is done to rows of logits before they are scored, drawn from or
trained on, and the two ends of a student's training step.

  adjust   per row of logits z[rows][vocab]: tokens of the row's history are
           penalised (a repetition factor, a presence and a frequency term; the
           prompt counts for the first alone), biases are added to listed tokens
           (of an id that is listed twice the later place counts), and what the
           row's mask does not allow becomes -inf.  Its gradient passes through.
  embed    out[i] = s W[token[i]] (token -1: padding, zeros), and the gradient
           dW[v] = s sum of the rows i of token v.
  norm     the 2-norm (or largest magnitude) over all of a model's gradients,
  clip     and the gradients times min(1, max_norm / (norm + 1e-6)), divided by
           the loss scale where there is one.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INDEX_BITS = 18  # vocabularies of up to 2^18 entries
LARGEST_BYTES = 2048 * 151936 * 4  # of the largest case's logits
# Shapes of decoders: layers, width, FFN width, key/value width, vocabulary, tied output
MODELS = {"tiny": (2, 64, 128, 32, 256, False), "smollm2": (30, 576, 1536, 192, 49152, True),
          "qwen05": (24, 896, 4864, 128, 151936, True), "tinyllama": (22, 2048, 5632, 256, 32000, False)}


def _adjust(name, rows, vocab, dtype, *, history=0, biases=0, shared_biases=False, mask="", per_row=False, in_place=False,
            stride=0, grad=False):
    c = dict(call="adjust_grad" if grad else "adjust", rows=rows, vocab=vocab, dtype=dtype, history=history,
             biases=biases, shared_biases=shared_biases, mask=mask, per_row=per_row, in_place=in_place,
             stride=stride or vocab)
    return dict(c, name=name) if name else c


def _embed(name, tokens, vocab, width, dtype, *, scale=1.0, grad=False, direct=False):
    c = dict(call="embed_grad" if grad else "embed", tokens=tokens, vocab=vocab, width=width, dtype=dtype, scale=scale,
             direct=direct)  # direct: a loop of its own asks for the gradient, not autograd
    return dict(c, name=name) if name else c


def _clip(name, model, dtype, *, layers=0, scale=1.0, out="", inf=False, norm=False):
    c = dict(call="norm" if norm else "clip", model=model, dtype=dtype, layers=layers or MODELS[model][0], scale=scale,
             out=out or dtype, inf=inf)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One stream's next token: f32 logits of one position, a short history,
        # a handful of biases.  Nothing but latency.
        _adjust("adjust-1x32000-f32-h200-b16", 1, 32000, "f32", history=200, biases=16, shared_biases=True),
        # A serving step of 64 requests, each with penalties, biases and a grammar of its own.
        _adjust("adjust-64x151936-bf16-h2048-b100-mask", 64, 151936, "bf16", history=2048, biases=100, mask="rows",
                per_row=True),
        # The same step where only the grammar masks, in the logits' own memory.
        _adjust("mask-256x151936-bf16", 256, 151936, "bf16", mask="rows", in_place=True),
        # A teacher's window of 2048 positions before it is scored: every position with
        # the tokens so far and what its grammar allows.
        _adjust("adjust-2048x151936-f32-h1024-mask", 2048, 151936, "f32", history=1024, mask="rows"),
        # Training on penalised logits: a small batch, rows of odd length further apart
        # than they are long,
        _adjust("adjust_grad-300x49155-f16-h100-mask", 300, 49155, "f16", history=100, mask="shared", stride=49216, grad=True),
        # and a full one of the largest vocabulary.
        _adjust("adjust_grad-4096x151936-bf16-h512", 4096, 151936, "bf16", history=512, grad=True),
        # The embeddings of a serving step of 64 streams.
        _embed("embed-64-151936x896-bf16", 64, 151936, 896, "bf16"),
        # A training batch of 2048 tokens: lookup and dense gradient, mostly the gradient's zeros;
        _embed("embed_grad-2048-49152x576-f32", 2048, 49152, 576, "f32", scale=24.0, grad=True, direct=True),
        # one of 65536 tokens, where the rows themselves count, through autograd.
        _embed("embed_grad-65536-32000x2048-bf16", 65536, 32000, 2048, "bf16", grad=True),
        # The gradients' norm alone, watched every step: 272 tensors.
        _clip("norm-smollm2-f32", "smollm2", "f32", norm=True),
        # A small student's gradients, scaled for f16, to the optimizer's f32.
        _clip("clip-qwen05-4layers-f16-scaled", "qwen05", "f16", layers=4, scale=1.0 / 4096, out="f32"),
        # A whole model's gradients: 201 tensors, 1.1e9 elements.
        _clip("clip-tinyllama-bf16", "tinyllama", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    call = rng.choice(["adjust", "adjust", "adjust_grad", "embed", "embed_grad", "embed_grad", "norm", "clip"])
    dtype = rng.choice(sorted(DTYPES))
    if call.startswith("adjust"):
        vocab = rng.choice([32000, 49152, 151936]) if rng.random() < 0.4 else _log_int(rng, 256, 1 << INDEX_BITS)
        rows = _log_int(rng, 1, max(1, min(16384, LARGEST_BYTES // (4 if dtype == "f32" else 2) // (vocab + 64))))
        history = rng.choice([0, _log_int(rng, 1, 256), _log_int(rng, 16, 8192)])
        history = min(history, (1 << 22) // rows)
        mask = rng.choice(["", "rows", "shared"])
        in_place = call == "adjust" and mask != "" and rng.random() < 0.4
        biases = 0 if in_place else rng.choice([0, 0, _log_int(rng, 1, 300)])
        return _adjust("", rows, vocab, dtype, history=0 if in_place else history, biases=min(biases, vocab),
                       shared_biases=rng.random() < 0.5, mask=mask, per_row=rng.random() < 0.5, in_place=in_place,
                       stride=vocab + rng.choice([0, 0, 1, -vocab % 64, 64]), grad=call == "adjust_grad")
    if call.startswith("embed"):
        vocab = rng.choice([32000, 49152, 151936]) if rng.random() < 0.4 else _log_int(rng, 256, 1 << INDEX_BITS)
        width = rng.choice([576, 896, 2048]) if rng.random() < 0.5 else _log_int(rng, 16, 8192)
        most = LARGEST_BYTES // (4 if dtype == "f32" else 2)
        vocab = min(vocab, most // width)
        tokens = _log_int(rng, 1, max(1, min(1 << 17, most // width)))
        return _embed("", tokens, vocab, width, dtype, scale=rng.choice([1.0, 1.0, math.sqrt(width)]),
                      grad=call == "embed_grad", direct=call == "embed_grad" and rng.random() < 0.5)
    model = rng.choice(sorted(MODELS))
    scale = rng.choice([1.0, 1.0, 1.0 / 1024]) if dtype != "bf16" else 1.0
    layers = _log_int(rng, 1, max(1, MODELS[model][0] // (4 if dtype == "f32" else 2)))
    return _clip("", model, dtype, layers=layers, scale=scale, out=rng.choice([dtype, "f32"]), inf=rng.random() < 0.3,
                 norm=call == "norm")


# ---- what a program has in hand ---------------------------------------------------


def _text(g, shape, vocab, dev):
    """Token ids as they come in text: few are frequent (rank r with a share of about 1 / r)."""
    u = torch.rand(shape, generator=g, device=dev)
    rank = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp(max=vocab - 1)
    return torch.randperm(vocab, generator=g, device=dev)[rank]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 29)
    call = case["call"]
    if call.startswith("adjust"):
        return _prepare_adjust(case, g, dev)
    if call.startswith("embed"):
        N, V, D = case["tokens"], case["vocab"], case["width"]
        w = torch.empty(V, D, dtype=DTYPES[case["dtype"]], device=dev).normal_(std=0.05, generator=g)
        tokens = _text(g, (N,), V, dev)
        if N > 16:  # padded sequences
            tokens[torch.rand(N, generator=g, device=dev) < 0.05] = -1
        state = {"case": case, "weight": w.requires_grad_(call == "embed_grad" and not case["direct"]), "tokens": tokens}
        if call == "embed_grad":
            state["grad"] = torch.empty(N, D, dtype=w.dtype, device=dev).normal_(std=0.01, generator=g)
        return state
    sizes = _shapes(case)
    n = sum(math.prod(s) for s in sizes)
    flat = torch.empty(n, dtype=DTYPES[case["dtype"]], device=dev).normal_(std=0.01 / case["scale"], generator=g)
    parts = flat.split([math.prod(s) for s in sizes])
    size = [0.2 + k % 7 for k in range(len(sizes))]
    torch._foreach_mul_(list(parts), size)  # layers differ
    state = {"case": case, "grads": [p.view(s) for p, s in zip(parts, sizes)], "max_norm": 1.0}
    if call == "clip":
        state["flat"] = torch.empty(n, dtype=DTYPES[case["out"]], device=dev)
        state["out"] = [p.view(s) for p, s in zip(state["flat"].split([p.numel() for p in parts]), sizes)]
    return state


def _shapes(case):
    _, d, ff, kv, vocab, tied = MODELS[case["model"]]
    layer = [(d,), (d, d), (kv, d), (kv, d), (d, d), (d,), (ff, d), (ff, d), (d, ff)]
    return [(vocab, d)] + layer * case["layers"] + [(d,)] + ([] if tied else [(vocab, d)])


def _prepare_adjust(case, g, dev):
    R, V, H, K = case["rows"], case["vocab"], case["history"], case["biases"]
    z = torch.empty(R, case["stride"], dtype=DTYPES[case["dtype"]], device=dev).normal_(std=3.0, generator=g)[:, :V]
    state = {"case": case, "logits": z.requires_grad_(case["call"] == "adjust_grad")}
    if case["call"] == "adjust_grad":
        state["grad"] = torch.empty(R, V, dtype=z.dtype, device=dev).normal_(std=0.01, generator=g)
    kw = state["adjust"] = {}
    if H:
        length = torch.randint(H // 2, H + 1, (R,), generator=g, device=dev)  # ragged: -1 behind a row's tokens
        prompt = (length * torch.rand(R, generator=g, device=dev) * 0.8).int()
        history = _text(g, (R, H), V, dev)
        history[torch.arange(H, device=dev) >= length[:, None]] = -1
        kw.update(history=history, prompt=prompt, repetition=1.1, presence=0.25, frequency=0.0625)
        if case["per_row"]:
            kw.update(repetition=1.0 + 0.5 * torch.rand(R, generator=g, device=dev),
                      presence=torch.rand(R, generator=g, device=dev),
                      frequency=0.2 * torch.rand(R, generator=g, device=dev))
    if K:
        lead = () if case["shared_biases"] else (R,)
        kw["bias_ids"] = torch.randint(0, V, (*lead, K), generator=g, device=dev)
        kw["bias"] = 4.0 * torch.randn(*lead, K, generator=g, device=dev)
    if case["mask"]:
        rows = R if case["mask"] == "rows" else 1
        words = torch.empty(rows, -(-V // 32), dtype=torch.int32, device=dev)
        # a grammar allows nearly everything (inside a string) or next to nothing
        share = torch.where(torch.rand(rows, 1, generator=g, device=dev) < 0.5, 0.97, 0.01)
        step = max(1, (1 << 26) // V)
        bit = torch.arange(32, device=dev, dtype=torch.int32)
        for r in range(0, rows, step):
            w = words[r:r + step]
            on = torch.rand(*w.shape, 32, generator=g, device=dev) < share[r:r + step, :, None]
            w.copy_((on.int() << bit).sum(2, dtype=torch.int32))
        kw["allowed"] = words if rows == R and case["mask"] == "rows" else words[0]
    return state


# ---- one pass -----------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    with torch.no_grad():
        if case["call"].startswith("adjust"):
            return _plain_adjust(case, state)
        if case["call"].startswith("embed"):
            return _plain_embed(case, state)
        return _plain_clip(case, state)


def _own(case, s):
    from detllm_amd import scores, train

    call = case["call"]
    if call == "adjust":
        return {"logits": scores.adjust_logits(s["logits"], **s["adjust"], out=s["logits"] if case["in_place"] else None)}
    if call == "adjust_grad":
        out = scores.adjust_logits(s["logits"], **s["adjust"])
        grad, = torch.autograd.grad([out], [s["logits"]], [s["grad"]])
        return {"logits": out.detach(), "grad": grad}
    if call == "embed":
        return {"rows": train.embedding(s["weight"], s["tokens"], scale=case["scale"])}
    if call == "embed_grad":
        out = train.embedding(s["weight"], s["tokens"], scale=case["scale"])
        if case["direct"]:
            return {"rows": out, "grad": train.embedding_grad(s["tokens"], s["grad"], case["vocab"], scale=case["scale"])}
        grad, = torch.autograd.grad([out], [s["weight"]], [s["grad"]])
        return {"rows": out.detach(), "grad": grad}
    kind = math.inf if case["inf"] else 2.0
    if call == "norm":
        return {"norm": train.grad_norm(s["grads"], norm_type=kind, scale=case["scale"])}
    norm = train.clip_grad_norm(s["grads"], s["max_norm"], norm_type=kind, scale=case["scale"], out=s["out"])
    return {"norm": norm, "grads": s["flat"]}


def _plain_adjust(case, s):
    kw, z = s["adjust"], s["logits"].detach()
    R, V = z.shape
    a = z.float()
    factor = None
    column = lambda p: p[:, None] if isinstance(p, torch.Tensor) else p  # noqa: E731
    if "history" in kw:
        h = kw["history"]
        at = torch.where((h < 0) | (h >= V), V, h)  # a column for what is no token
        answer = (torch.arange(h.shape[1], device=h.device) >= kw["prompt"][:, None]).int()
        seen = torch.zeros(R, V + 1, dtype=torch.bool, device=z.device).scatter_(1, at, True)[:, :V]
        count = torch.zeros(R, V + 1, dtype=torch.int32, device=z.device).scatter_add_(1, at, answer)[:, :V]
        theta = column(kw["repetition"])
        if case["call"] == "adjust_grad":
            factor = torch.where(seen, torch.where(a > 0, 1.0 / theta, theta), 1.0)
        a = torch.where(seen, torch.where(a > 0, a / theta, a * theta), a)
        a = a - torch.where(count > 0, column(kw["presence"]) + column(kw["frequency"]) * count, 0.0)
    if "bias" in kw:
        ids, bias = (kw[k].expand(R, -1) for k in ("bias_ids", "bias"))
        place = torch.arange(1, ids.shape[1] + 1, device=ids.device).expand(R, -1)
        last = torch.zeros(R, V, dtype=torch.int64, device=z.device).scatter_reduce_(1, ids, place, "amax")
        a = a + torch.where(last > 0, bias.gather(1, (last - 1).clamp(min=0)), 0.0)
    allowed = None
    if "allowed" in kw:
        bit = torch.arange(32, device=z.device, dtype=torch.int32)
        allowed = ((kw["allowed"][..., None] >> bit) & 1).bool().flatten(-2)[..., :V]
        a = torch.where(allowed, a, -math.inf)
    a = a.to(z.dtype)
    if case["in_place"]:
        z.copy_(a)
        return {"logits": z}
    if case["call"] == "adjust":
        return {"logits": a}
    grad = s["grad"].float()
    grad = grad if factor is None else grad * factor
    return {"logits": a, "grad": (grad if allowed is None else torch.where(allowed, grad, 0.0)).to(z.dtype)}


def _plain_embed(case, s):
    w, tokens, scale = s["weight"].detach(), s["tokens"], case["scale"]
    real = tokens >= 0
    at = tokens.clamp(min=0)
    rows = torch.where(real[:, None], w[at].float() * scale, 0.0).to(w.dtype)
    if case["call"] == "embed":
        return {"rows": rows}
    grad = torch.zeros(w.shape, device=w.device)
    grad.index_add_(0, at, torch.where(real[:, None], s["grad"].float(), 0.0))
    return {"rows": rows, "grad": (grad * scale).to(w.dtype)}


def _plain_clip(case, s):
    scale = case["scale"]
    if case["inf"]:
        norm = torch.stack([t.float().abs().amax() for t in s["grads"]]).amax() * scale
    else:
        norm = torch.stack([t.float().square().sum(dtype=torch.float64) for t in s["grads"]]).sum().sqrt().mul(scale).float()
    if case["call"] == "norm":
        return {"norm": norm}
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0) * scale
    [o.copy_(t.float() * factor) for t, o in zip(s["grads"], s["out"])]
    return {"norm": norm, "grads": s["flat"]}


# ---- the same in 64 bits ------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    call = case["call"]
    if call.startswith("embed"):
        w, t = s["weight"].detach().double(), s["tokens"]
        rows = torch.cat([w, torch.zeros_like(w[:1])])[t] * case["scale"]  # -1: the row of zeros at the end
        if call == "embed":
            return {"rows": rows}
        grad = torch.zeros(w.shape[0] + 1, w.shape[1], dtype=torch.float64, device=w.device)
        order = torch.argsort(t, stable=True)
        grad.index_put_((torch.where(t < 0, w.shape[0], t)[order],), s["grad"].double()[order], accumulate=True)
        return {"rows": rows, "grad": grad[:-1] * case["scale"]}
    if call in ("norm", "clip"):
        parts = [torch.linalg.vector_norm(t.double(), math.inf if case["inf"] else 2) for t in s["grads"]]
        norm = torch.linalg.vector_norm(torch.stack(parts), math.inf if case["inf"] else 2) * case["scale"]
        if call == "norm":
            return {"norm": norm}
        c = min(1.0, s["max_norm"] / (float(norm) + 1e-6)) * case["scale"]
        return {"norm": norm, "grads": torch.cat([t.double().flatten() for t in s["grads"]]).mul_(c)}
    step = max(1, (1 << 26) // case["vocab"])
    parts = [_exact_rows(case, s, slice(r, min(case["rows"], r + step))) for r in range(0, case["rows"], step)]
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_rows(case, s, rows):
    kw = s["adjust"]
    z = s["logits"].detach()[rows].double()
    R, V = z.shape
    slope = torch.ones_like(z)

    def per_row(name):
        p = kw[name]
        return p[rows].double()[:, None] if isinstance(p, torch.Tensor) else torch.full((R, 1), p, dtype=torch.float64, device=z.device)

    if "history" in kw:
        h = kw["history"][rows]
        row = torch.arange(R, device=z.device)[:, None].expand_as(h)
        is_token = (h >= 0) & (h < V)
        behind = is_token & (torch.arange(h.shape[1], device=h.device) >= kw["prompt"][rows][:, None])
        n_all, n = (torch.bincount((row * V + h)[m], minlength=R * V).view(R, V).double() for m in (is_token, behind))
        # as the parameters are held: 32 bits
        theta, presence, frequency = (per_row(k).float().double() for k in ("repetition", "presence", "frequency"))
        slope = torch.where(n_all > 0, torch.where(z > 0, theta.reciprocal(), theta), slope)
        z = z * slope - frequency * n - presence * n.clamp(max=1.0)
    if "bias" in kw:
        ids, bias = kw["bias_ids"], kw["bias"].double()
        ids, bias = (ids, bias) if case["shared_biases"] else (ids[rows], bias[rows])
        ids, bias = ids.expand(R, -1), bias.expand(R, -1)
        # of two places with one id the later one counts
        k = ids.shape[1]
        again = torch.triu(torch.ones(k, k, dtype=torch.bool, device=z.device), 1)
        per = max(1, (1 << 24) // (k * k))
        dead = torch.cat([((i[:, :, None] == i[:, None, :]) & again).any(2) for i in ids.split(per)])
        z = z.scatter_add(1, ids, torch.where(dead, 0.0, bias))
    if "allowed" in kw:
        words = kw["allowed"] if case["mask"] == "shared" else kw["allowed"][rows]
        j = torch.arange(V, device=z.device)
        off = (words[..., j // 32] >> (j % 32).int()) & 1 == 0
        z = z.masked_fill(off, -math.inf)
        slope = slope.masked_fill(off, 0.0)
    if case["call"] == "adjust":
        return {"logits": z}
    return {"logits": z, "grad": s["grad"][rows].double() * slope}


def work(case):
    call, e = case["call"], 4 if case["dtype"] == "f32" else 2
    if call.startswith("adjust"):
        R, n = case["rows"], case["rows"] * case["vocab"]
        small = R * case["history"] * 8 + case["biases"] * 12 * (1 if case["shared_biases"] else R)
        small += {"": 0, "rows": R, "shared": 1}[case["mask"]] * case["vocab"] // 8
        if case["in_place"]:  # masked logits are written, the others stay: half of them as these masks go
            return {"bytes": n * e // 2 + small, "flops": n}
        return {"bytes": n * e * (4 if call == "adjust_grad" else 2) + small, "flops": 4 * n}
    if call.startswith("embed"):
        N, V, D = case["tokens"], case["vocab"], case["width"]
        b = N * 8 + (min(N, V) + N) * D * e
        return {"bytes": b + ((N + V) * D * e if call == "embed_grad" else 0), "flops": N * D * (2 if call == "embed_grad" else 1)}
    n = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": n * (e + (0 if call == "norm" else 4 if case["out"] == "f32" else 2)), "flops": n * (2 if call == "norm" else 3)}
