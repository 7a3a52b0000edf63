"""Scores of a session's rows under penalties, biases and masks
(dtl_session_adjusted_scores), against the definitions in 64 bits."""
import numpy as np
import pytest

import adjust64
import rows64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tiny():
    from detllm_amd import synth
    from detllm_amd.model import F32Llama

    w = synth.WORKLOADS["tiny"]
    toks = [int(t) for t in synth.tokens(w)]
    model = F32Llama.from_gguf(synth.build_model(w))
    with model.forward_workspace(len(toks), len(toks)) as s:
        z = s.forward_chunk(toks, 0, want_logits=True)
        yield s, toks, z, w.vocab


def near(got, want, tol, what):
    assert abs(float(got) - want) <= tol or got == want, (what, got, want, tol)


def words(on):
    pad = np.concatenate([on, np.ones((*on.shape[:-1], -on.shape[-1] % 32), bool)], -1)
    return np.packbits(pad, axis=-1, bitorder="little").view(np.uint32)


@pytest.mark.parametrize("form", ["bits", "bytes", "shared", "numbers", "none"])
def test_adjusted_scores(tiny, form):
    s, toks, z, V = tiny
    rng = np.random.default_rng(len(form))
    n, T = len(toks) - 2, 1.5
    one = form in ("shared", "numbers")
    h = rng.integers(-1, V + 2, (1 if one else n, 40))
    h[:, ::3] = toks[2]
    prompt = 7 if one else rng.integers(0, 41, n)
    theta, pres, freq = (0.9, 0.3, -0.2) if one else (rng.uniform(0.6, 2, n).astype(np.float32), rng.normal(0, 1, n).astype(np.float32),
                                                     rng.normal(0, 1, n).astype(np.float32))
    ids, bias = rng.integers(-1, V, (1 if one else n, 9)), rng.normal(0, 3, (1 if one else n, 9)).astype(np.float32)
    on = rng.random((1 if one else n, V)) < 0.3
    on[:, toks] = True
    if not one:
        on[1] = False
    kw = dict(history=h[0] if one else h, prompt=prompt, repetition=theta, presence=pres, frequency=freq,
              bias_ids=ids[0] if one else ids, bias=bias[0] if one else bias)
    if form != "none":
        kw["allowed"] = (words(on) if form in ("bits", "shared") else on)[0 if one else slice(None)]
    got = s.token_scores(toks[1:1 + n], first=1, top=4, temperature=T, **kw)
    row = (lambda a, i: a[0] if one else a[i])
    for i in range(n):
        pick = lambda x: x if np.ndim(x) == 0 else x[i]  # noqa: E731
        a, off = adjust64.adjust(z[1 + i], "f32", row(h, i), pick(prompt), float(pick(theta)), float(pick(pres)), float(pick(freq)),
                                 row(ids, i), row(bias, i), None if form == "none" else row(on, i))
        # a logit that is off by e moves a log probability by up to 2 e / T, the entropy by as
        # much times the range of log p
        seen = np.isfinite(a)
        e = 2 * off[seen].max() / T if seen.any() else 0.0
        lp, tol, ent, tol_e = rows64.scores(a, toks[1 + i], T)
        near(got.log_probs[i], lp, tol + e, "log_prob")
        spread = (a[seen].max() - a[seen].min()) / T if seen.any() else 0.0
        near(got.entropy[i], ent, tol_e + e * (2 + spread), "entropy")
        want = rows64.top(a, 4, T)[0].tolist()
        for k, (x, y) in enumerate(zip(got.top_ids[i].tolist(), want)):  # ids that differ are as likely
            assert x == y or abs(a[x] - a[y]) <= off[x] + off[y], (i, k)
    assert np.array_equal(s.logits(), z)  # the session's own stay
    plain = s.token_scores(toks[1:1 + n], first=1, top=4, temperature=T)
    again = s.token_scores(toks[1:1 + n], first=1, top=4, temperature=T, **kw)
    assert all(np.array_equal(x, y) for x, y in zip(got, again)) and not np.array_equal(plain.log_probs, got.log_probs)


def test_one_row_of_a_decode_and_the_codec_beside_it(tiny):
    s, toks, z, V = tiny
    before = s.symbol_ranges(toks[1:], 0, 256)
    on = np.zeros(V, bool)
    on[[3, 5]] = True
    got = s.token_scores([5], first=2, top=8, allowed=on)
    assert sorted(got.top_ids[0][:2].tolist()) == [3, 5] and (got.top_ids[0][2:] == -1).all()
    assert abs(np.exp(got.top_log_probs[0][:2].astype(np.float64)).sum() - 1) < 1e-6
    assert all(np.array_equal(a, b) for a, b in zip(before, s.symbol_ranges(toks[1:], 0, 256)))


def test_refusals(tiny):
    from detllm_amd._lib import DetllmError

    s, toks, z, V = tiny
    n = 2
    for kw in (dict(prompt=3), dict(bias=[1.0]), dict(bias_ids=[1]), dict(history=[[1], [2], [3]]), dict(allowed=np.ones((n, V - 1), bool)),
               dict(allowed=np.ones(V, np.uint32)), dict(history=[1], repetition=[1.0, 2.0, 3.0]), dict(bias_ids=[1, 2], bias=[1.0])):
        with pytest.raises(ValueError):
            s.token_scores(toks[:n], **kw)
    with pytest.raises(TypeError):
        s.token_scores(toks[:n], allowed=np.ones(V))
    for kw, status in ((dict(history=[1], repetition=0.0), 42), (dict(history=[1], presence=float("nan")), 42),
                       (dict(bias_ids=np.zeros(4097, int), bias=np.zeros(4097)), 1), (dict(history=[1], top=V + 1), 1)):
        with pytest.raises(DetllmError) as e:
            s.token_scores(toks[:n], **kw)
        assert e.value.status == status
    empty = s.token_scores(toks[:n], history=[], bias_ids=[], bias=[])
    assert np.array_equal(empty.log_probs, s.token_scores(toks[:n]).log_probs)
