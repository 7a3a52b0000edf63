"""The operators on rows of logits as cases that can be timed and compared:
what the rows say of given tokens (log probability, entropy, top alternatives)
and distillation from a teacher's top alternatives, with their gradients.

logits[rows][vocab] are what a decoder's output projection leaves on the
device: f32 from this library's sessions, 16-bit floats in training programs.
With z a row, T the temperature, m = max z and p = softmax(z / T):

  scores   log p[token], the entropy -sum p log p, and the `top` largest z
           (ties to the lowest index) with their log p.  A token of -1 is
           padding: 0.  Logits of -inf are masked and no alternatives: id -1.
  distill  per row, from a list of ids with log probabilities v at the same
           temperature (id -1: an empty slot):
             loss = w T^2 sum_k p_k (log p_k - log q[id_k]),  q = softmax(z / T)
           with p = softmax(v) over the list, or, where `rest` is set, p = exp(v)
           and one more term for what lies outside the list on either side.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INDEX_BITS = 18  # vocabularies of up to 2^18 entries
LARGEST = 4096 * 151936  # logits of the largest case
LARGEST_BYTES = 2048 * 151936 * 4


def _case(name, call, rows, vocab, dtype, k, *, stride=0, temperature=1.0, rest=False, masked=False):
    c = dict(call=call, rows=rows, vocab=vocab, dtype=dtype, k=k, stride=stride or vocab, temperature=temperature,
             rest=rest, masked=masked)
    return dict(c, name=name) if name else c


def listed():
    return [
        # The token a decoder just produced, with its best alternative: f32
        # logits of one position, nothing but latency.
        _case("score-1x32000-f32-top1", "score", 1, 32000, "f32", 1),
        # A serving step for eight streams, each with 20 alternatives; some
        # tokens are masked by what the caller allows.
        _case("score-8x151936-bf16-top20", "score", 8, 151936, "bf16", 20, masked=True),
        # A document's code length and entropy per token, no alternatives; the
        # output matrix is padded, so rows are further apart than they are long.
        _case("score-300x49155-f16", "score", 300, 49155, "f16", 0, stride=49216),
        # A teacher's targets for a whole window of 2048 positions.
        _case("score-2048x151936-f32-top64", "score", 2048, 151936, "f32", 64),
        # Log probabilities and entropy with their gradient, rows of odd length
        # (no row but the first is aligned), below the usual temperature.
        _case("score_grad-512x32003-bf16", "score_grad", 512, 32003, "bf16", 0, temperature=0.75),
        # The same for a training batch of the largest vocabulary.
        _case("score_grad-4096x151936-bf16", "score_grad", 4096, 151936, "bf16", 0),
        # The loss of a handful of positions, watched while decoding.
        _case("distill-4x32000-f32-k8", "distill", 4, 32000, "f32", 8),
        # Evaluating a student on held-out targets.
        _case("distill-1024x49152-f16-k32", "distill", 1024, 49152, "f16", 32, rest=True),
        # The loss inside a larger graph: forward, then backward with the
        # gradient of each row's loss, softened targets, masked logits.
        _case("distill_grad-333x49152-f32-k128", "distill_grad", 333, 49152, "f32", 128, temperature=2.0, rest=True,
              masked=True),
        # Training steps with known row weights: a small batch,
        _case("distill_step-256x32000-bf16-k20", "distill_step", 256, 32000, "bf16", 20),
        # a ragged one of the largest vocabulary,
        _case("distill_step-1021x151936-bf16-k64", "distill_step", 1021, 151936, "bf16", 64, rest=True),
        # and a full one.
        _case("distill_step-4096x151936-bf16-k100", "distill_step", 4096, 151936, "bf16", 100, temperature=2.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    call = rng.choice(["score", "score", "score_grad", "distill", "distill_grad", "distill_step"])
    dtype = rng.choice(sorted(DTYPES))
    vocab = rng.choice([32000, 49152, 151936]) if rng.random() < 0.4 else _log_int(rng, 256, 1 << INDEX_BITS)
    most = min(LARGEST, LARGEST_BYTES // (4 if dtype == "f32" else 2))
    rows = _log_int(rng, 1, max(1, min(16384, most // vocab)))
    k = rng.choice([0, 1, _log_int(rng, 2, 128)]) if call == "score" else 0 if call == "score_grad" else _log_int(rng, 1, 256)
    stride = vocab + (rng.choice([0, 0, 1, -vocab % 64, 64]))
    if rows * stride > most:
        stride = vocab
    return _case("", call, rows, vocab, dtype, min(k, vocab), stride=stride, temperature=rng.choice([1.0, 1.0, 0.7, 2.0, 4.0]),
                 rest=call.startswith("distill") and rng.random() < 0.5, masked=rng.random() < 0.3)


# ---- what a program has in hand ---------------------------------------------------


def prepare(case, seed):
    """Logits of a decoder over text: a few tokens of every row stand out, common tokens are
    likelier everywhere, rows differ in how sure they are; some rows are padding."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    R, V, K, T = case["rows"], case["vocab"], case["k"], case["temperature"]
    z = torch.empty(R, case["stride"], dtype=DTYPES[case["dtype"]], device=dev).normal_(generator=g)[:, :V]
    common = -0.5 * torch.log1p(torch.randperm(V, generator=g, device=dev).float())
    z.mul_((0.5 + 2.0 * torch.rand(R, 1, generator=g, device=dev)).to(z.dtype)).add_(common.to(z.dtype))
    tokens = torch.randint(0, V, (R,), generator=g, device=dev)
    at = torch.randint(0, V, (R, 12), generator=g, device=dev)
    at[:, 0] = tokens
    z.scatter_(1, at, (14.0 * torch.rand(R, 12, generator=g, device=dev)).to(z.dtype))
    if case["masked"]:
        off = torch.rand(V, generator=g, device=dev) < 0.3
        z.masked_fill_(off, -math.inf)
        z.scatter_(1, tokens[:, None], 3.0)
    padding = torch.rand(R, generator=g, device=dev) < (0.1 if R > 1 else 0.0)
    state = {"case": case, "logits": z.requires_grad_(case["call"].endswith("_grad")),
             "tokens": torch.where(padding, -1, tokens)}
    if case["call"] == "score_grad":
        state["grads"] = [torch.where(padding, 0.0, torch.randn(R, generator=g, device=dev)) / R, torch.full((R,), 0.01 / R, device=dev)]
    if case["call"].startswith("distill"):
        z = z.detach()
        # the teacher's list: mostly tokens that the student rates too, the target first
        ids = torch.randint(0, V, (R, K), generator=g, device=dev)
        few = min(K, 12)
        ids[:, :few] = at[:, :few]
        ids = ids.sort(1).values
        ids[:, 1:].masked_fill_(ids[:, 1:] == ids[:, :-1], -1)  # each token once; empty slots in between
        v = torch.gather(z, 1, ids.clamp(min=0)).float().clamp(min=-8.0) / T + 0.5 * torch.randn(R, K, generator=g, device=dev)
        v = torch.where(ids < 0, -math.inf, v)
        v = torch.log_softmax(v, 1) + torch.log1p(-0.3 * torch.rand(R, 1, generator=g, device=dev))
        void = padding[:, None].expand(R, K)
        state["teacher_ids"] = torch.where(void, -1, ids).int()
        state["teacher_log_probs"] = torch.where(void, -math.inf, v).contiguous()
        state["weights"] = torch.where(padding, 0.0, 1.0 / R)
    return state


# ---- one pass -----------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    with torch.no_grad():
        if case["call"].startswith("score"):
            return _plain_scores(case, state)
        return _plain_distill(case, state)


def _own(case, s):
    from detllm_amd import scores

    call, T = case["call"], case["temperature"]
    if call in ("score", "score_grad"):
        got = scores.token_scores(s["logits"], s["tokens"], top=case["k"], temperature=T)
        out = {"log_probs": got.log_probs, "entropy": got.entropy}
        if case["k"]:
            out |= {"top_ids": got.top_ids, "top_log_probs": got.top_log_probs}
        if call == "score_grad":
            out["grad"], = torch.autograd.grad([got.log_probs, got.entropy], [s["logits"]], s["grads"])
        return {k: v.detach() for k, v in out.items()}
    if call == "distill_step":
        loss, grad = scores.distill_loss_and_grad(s["logits"], s["teacher_ids"], s["teacher_log_probs"], s["weights"],
                                                  temperature=T, rest=case["rest"])
        return {"loss": loss, "grad": grad}
    loss = scores.distill_loss(s["logits"], s["teacher_ids"], s["teacher_log_probs"], temperature=T, rest=case["rest"])
    if call == "distill":
        return {"loss": loss}
    grad, = torch.autograd.grad([loss], [s["logits"]], [s["weights"]])
    return {"loss": loss.detach(), "grad": grad}


def _plain_scores(case, s):
    T, K, tokens = case["temperature"], case["k"], s["tokens"]
    x = s["logits"].detach().float()
    m = x.amax(1, keepdim=True)
    t = (x - m) / T
    e = torch.exp(t)
    # long sums in 64 bits: a sure row's log probability is log(1 + something tiny)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    log_total = torch.log(total)
    p = (e / total.float())
    logp = torch.where(t == -math.inf, 0.0, t - log_total.float())
    entropy = -(p * logp).sum(1, dtype=torch.float64)
    picked = torch.gather(t, 1, tokens.clamp(min=0)[:, None]).double() - log_total
    out = {"log_probs": torch.where(tokens < 0, 0.0, picked[:, 0]).float(), "entropy": entropy.float()}
    if K:
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        last = (1 << INDEX_BITS) - 1
        key = order * (1 << INDEX_BITS) + (last - torch.arange(x.shape[1], device=x.device))
        ids = last - (torch.topk(key, K, dim=1, sorted=True).values & last)
        v = torch.gather(t, 1, ids)
        out |= {"top_ids": torch.where(v == -math.inf, -1, ids).int(), "top_log_probs": (v.double() - log_total).float()}
    if case["call"] == "score_grad":
        a, b = s["grads"]
        a = torch.where(tokens < 0, 0.0, a)[:, None]
        grad = -p * (a + b[:, None] * (logp + entropy.float()[:, None]))
        grad.scatter_add_(1, tokens.clamp(min=0)[:, None], a)
        out["grad"] = (grad / T).to(s["logits"].dtype)
    return out


def _plain_distill(case, s):
    T, ids, v = case["temperature"], s["teacher_ids"].long(), s["teacher_log_probs"]
    x = s["logits"].detach().float()
    m = x.amax(1, keepdim=True)
    e = torch.exp((x - m) / T)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    log_total = torch.log(total)
    void = (ids < 0) | (v == -math.inf)
    at = ids.clamp(min=0)
    top = torch.where(void, -math.inf, v).double()  # the loss is a small difference of large terms
    if not case["rest"]:
        most = top.amax(1, keepdim=True).clamp(min=-1e30)
        top = top - most - torch.log(torch.exp(top - most).sum(1, keepdim=True).clamp(min=1e-30))
    p = torch.exp(top)
    logq = (torch.gather(x, 1, at) - m).double() / T - log_total
    loss = torch.where(void | (p == 0), 0.0, p * (top - logq)).sum(1)
    mass = p.sum(1, keepdim=True)
    share = mass / total
    outside = None
    if case["rest"]:
        listed_ = torch.zeros_like(x, dtype=torch.bool).scatter_(1, at, ~void)
        # an empty slot must not clear the entry 0 that another one lists
        listed_[:, 0] = ((at == 0) & ~void).any(1)
        left = e.masked_fill(listed_, 0.0).sum(1, keepdim=True, dtype=torch.float64)
        rest = torch.where(void.all(1, keepdim=True) | (left == 0), 0.0, (1.0 - mass).clamp(min=0.0))
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - torch.log(left / total)), 0.0)[:, 0]
        share = (mass + rest) / total
        outside = torch.where(left > 0, rest / left, 0.0)
    w = s["weights"][:, None].double()
    scale = T * T * (w if case["call"] == "distill_step" else 1.0)
    out = {"loss": (scale * loss[:, None])[:, 0].float() if case["call"] == "distill_step" else (T * T * loss).float()}
    if case["call"] != "distill":
        grad = e * share.float()
        if outside is not None:
            grad -= (e * outside.float()).masked_fill(listed_, 0.0)
        grad.scatter_add_(1, at, torch.where(void, 0.0, -p).float())
        out["grad"] = (grad * (w * T).float()).to(s["logits"].dtype)
    return out


# ---- the same in 64 bits ------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    step = max(1, (1 << 26) // case["vocab"])
    parts = [_exact_rows(case, {k: v[r:r + step] for k, v in _rows_of(s).items()}) for r in range(0, case["rows"], step)]
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _rows_of(s):
    rows = {k: v.detach() for k, v in s.items() if isinstance(v, torch.Tensor)}
    return rows | ({"a": s["grads"][0], "b": s["grads"][1]} if "grads" in s else {})


def _exact_rows(case, s):
    T = case["temperature"]
    z = s["logits"].double() / T
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    p = lp.exp()
    if case["call"].startswith("score"):
        y = s["tokens"]
        # log1p of the others' share keeps the digits of a log probability next to zero
        best = z.argmax(1, keepdim=True)
        others = (z - z.gather(1, best)).exp().scatter(1, best, 0.0).sum(1, keepdim=True)
        lp = z - z.gather(1, best) - torch.log1p(others)
        plogp = torch.where(p > 0, p * lp, 0.0)
        h = -plogp.sum(1, keepdim=True)
        real = (y >= 0).double()[:, None]
        out = {"log_probs": torch.where(y < 0, 0.0, lp.gather(1, y.clamp(min=0)[:, None])[:, 0]), "entropy": h[:, 0]}
        if case["k"]:
            v, ids = torch.sort(s["logits"].double(), dim=1, descending=True, stable=True)
            v, ids = v[:, :case["k"]], ids[:, :case["k"]]
            out |= {"top_ids": torch.where(v == -math.inf, -1, ids).int(), "top_log_probs": lp.gather(1, ids)}
        if case["call"] == "score_grad":
            one = torch.zeros_like(z).scatter_(1, y.clamp(min=0)[:, None], real)
            a = s["a"].double()[:, None] * real
            out["grad"] = (a * (one - p) - s["b"].double()[:, None] * (plogp + h * p)) / T
        return out
    ids, v = s["teacher_ids"].long(), s["teacher_log_probs"].double()
    used = (ids >= 0) & (v > -math.inf)
    t = torch.where(used, v, -math.inf)
    if not case["rest"]:
        t = torch.where(used.any(1, keepdim=True), t - torch.logsumexp(t, 1, keepdim=True), t)
    teacher = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), torch.where(used, t.exp(), 0.0))
    logt = torch.where(used, t, 0.0)
    loss = torch.where(used, t.exp() * (logt - lp.gather(1, ids.clamp(min=0))), 0.0).sum(1)
    total = teacher.sum(1, keepdim=True)
    grad = total * p - teacher
    if case["rest"]:
        inside = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), used.double()) > 0
        left = torch.where(inside, 0.0, p).sum(1, keepdim=True)
        counts = used.any(1, keepdim=True) & (left > 0)
        rest = torch.where(counts, (1.0 - total).clamp(min=0.0), 0.0)
        loss = loss + torch.where(rest > 0, rest * (rest / left).log(), 0.0)[:, 0]
        grad = grad + torch.where(rest > 0, rest * (p - torch.where(inside, 0.0, p) / left), 0.0)
    w = s["weights"].double()
    out = {"loss": T * T * loss * (w if case["call"] == "distill_step" else 1.0)}
    if case["call"] != "distill":
        out["grad"] = T * w[:, None] * grad
    return out


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    n = case["rows"] * case["vocab"]
    grad = case["call"] in ("score_grad", "distill_grad", "distill_step")
    if case["call"].startswith("score"):
        small = case["rows"] * (8 + 8 + 8 * case["k"] + (8 if grad else 0))
    else:
        small = case["rows"] * (8 * case["k"] + 8)
    return {"bytes": n * e * (2 if grad else 1) + small, "flops": n * (11 if grad else 6)}
