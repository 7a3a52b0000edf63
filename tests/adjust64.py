"""Adjusted logits of one row and their gradient in 64 bits, with how far results of
32-bit arithmetic, rounded once to the logits' type, may be from them."""
import numpy as np

# half a step relative to the value, and of the smallest numbers
ROUND = {"f32": (2.0**-24, 2.0**-150), "bf16": (2.0**-8, 2.0**-134), "f16": (2.0**-11, 2.0**-25)}


# what is at least this large rounds to infinity: half a step past the largest number
OVER = {"f32": 2.0**128 * (1 - 2.0**-25), "bf16": 2.0**128 * (1 - 2.0**-9), "f16": 65520.0}


def within(v, dtype):
    """v, infinite where it passes the type's range, as IEEE rounding has it."""
    return np.where(np.abs(v) >= OVER[dtype], np.copysign(np.inf, v), v)


def counts(history, prompt, vocab):
    """Whether each token stands in the history, and how often behind the prompt."""
    h = np.asarray(history, np.int64)
    real, answer = (h >= 0) & (h < vocab), np.arange(h.size) >= prompt
    return np.bincount(h[real], minlength=vocab) > 0, np.bincount(h[real & answer], minlength=vocab).astype(np.float64)


def rounded(v, dtype):
    half, least = ROUND[dtype]
    return np.abs(v) * half + least


def adjust(z, dtype, history=(), prompt=0, theta=1.0, presence=0.0, frequency=0.0, bias_ids=(), bias=(), allowed=None):
    """(adjusted, tolerance).  Each 32-bit step is off by at most 2^-24 of its result;
    what comes in off by e goes out off by e (a quotient's or product's is its own).
    The sums of such terms are taken 1.01 times for their products.  A step whose result
    passes the range is infinite and stays so."""
    z = np.asarray(z, np.float64)
    seen, n = counts(history, prompt, z.size)
    with np.errstate(all="ignore"):
        a = within(np.where(seen, np.where(z > 0, z / theta, z * theta), z), "f32")
        off = np.where(seen, np.abs(a), 0.0)
        less = np.where(n > 0, presence + frequency * n, 0.0)
        off = off + np.where(n > 0, np.abs(frequency * n) + np.abs(less), 0.0)
        a = within(a - less, "f32")
        off = off + np.where(n > 0, np.abs(a), 0.0)
        last = {}
        for t, b in zip(bias_ids, bias):
            if 0 <= t < z.size:
                last[int(t)] = float(b)
        for t, b in last.items():
            a[t] += b
            off[t] += np.abs(a[t])
        tol = 1.01 * 2.0**-24 * off + rounded(a, dtype)
        a = within(a, dtype)
    if allowed is not None:
        a = np.where(allowed, a, -np.inf)
    return a, tol


def gradient(z, g, dtype, history=(), theta=1.0, allowed=None):
    """(gradient of the logits, tolerance): one 32-bit step and the rounding."""
    z, g = np.asarray(z, np.float64), np.asarray(g, np.float64)
    seen, _ = counts(history, 0, z.size)
    with np.errstate(all="ignore"):
        d = np.where(seen, np.where(z > 0, g / theta, g * theta), g)
        if allowed is not None:
            d = np.where(allowed, d, 0.0)
        d = within(d, dtype)
        return d, 1.01 * 2.0**-24 * np.abs(d) + rounded(d, dtype)


def same(got, want, tol):
    """Whether every value is the same number, infinity or no number, within tol."""
    got = np.asarray(got, np.float64)
    finite = np.isfinite(want)
    ok = np.where(finite, False, np.where(np.isnan(want), np.isnan(got), got == want))
    with np.errstate(invalid="ignore"):
        return ok | (finite & (np.abs(got - want) <= tol))
