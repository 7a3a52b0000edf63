"""Scores and distillation of rows of logits in 64 bits, from their definitions,
and how far 32-bit results may be from them.

Bounds, with h = 2^-24 (half a step of float32, relative).  A term e = 2^t of a
sum, t = (z - m) c, carries the roundings of z - m, of c and of the product
(3 h |t| ln 2 relative) and of the hardware's 2^x (1 ulp: 2 h); a factor 2^d that
brings a segment's sum to the row's maximum carries the same again, with
|d| <= |t|.  A sum of 2048 such terms adds at most 8 + 2 + 6 roundings.  So the sum
over all but the maximum is off by at most (32 + 6 U) h relative, U the mean
|t| ln 2 under it.
"""
import numpy as np

H = 2.0 ** -24
DTYPES = {"f32": (0, 4, 2.0 ** -24), "bf16": (1, 2, 2.0 ** -8), "f16": (2, 2, 2.0 ** -11)}


def to_bits(x, dtype):
    """The values' bits in a type (round to nearest even), as an unsigned array."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x.view(np.uint32)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, dtype):
    if dtype == "f32":
        return b.view(np.float32).astype(np.float64)
    if dtype == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def _least(dtype):
    """Half the smallest step of a type."""
    return {"f32": 2.0 ** -149, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}[dtype]


class Row:
    """One row's softmax at temperature T."""

    def __init__(self, z, T):
        self.z, self.T = z, float(np.float32(T))
        self.bad = bool(np.isnan(z).any() or (z == np.inf).any())
        self.empty = not self.bad and bool((z == -np.inf).all())
        if self.bad or self.empty:
            return
        m = z.max()
        with np.errstate(over="ignore", invalid="ignore"):
            self.t = (z - m) / self.T
        rest = np.exp(self.t)
        rest[int(z.argmax())] = 0.0
        self.r = rest.sum()
        self.L = np.log1p(self.r)
        self.logp = self.t - self.L
        self.p = np.exp(self.logp)
        self.at = np.where(self.p > 0, np.abs(self.t), 0.0)
        self.plogp = np.where(self.p > 0, self.p * np.where(self.p > 0, self.logp, 0.0), 0.0)
        self.H = -self.plogp.sum()
        share = self.r / (1 + self.r)
        mean = float((self.p * self.at).sum()) / share if share > 0 else 0.0
        # the hardware's 2^x is 0 where the result would be subnormal: each of the
        # n terms may miss up to 2^-126 (with n = 5003 terms up to 5.9e-35)
        self.tol_L = share * (32 + 6 * mean) * H + H * self.L + z.size * 2.0 ** -126
        a1, a2 = float((self.p * self.at).sum()), float((self.p * self.at ** 2).sum())
        self.tol_H = self.tol_L + H * (40 * a1 + 8 * a2 + abs(self.H))


def scores(z, token, T):
    """(log_prob, its tolerance, entropy, its tolerance) of one row."""
    row = Row(z, T)
    if row.bad:
        return (0.0 if token < 0 else np.nan), 0.0, np.nan, 0.0
    if row.empty:
        lp = 0.0 if token < 0 else np.nan if token >= z.size else -np.inf
        return lp, 0.0, 0.0, 0.0
    if token < 0:
        lp, tol = 0.0, 0.0
    elif token >= z.size:
        lp, tol = np.nan, 0.0
    else:
        lp = row.logp[token]
        tol = row.tol_L + (2 * H * abs(lp) if np.isfinite(lp) else 0.0) + 2.0 ** -149
    return lp, tol, row.H, row.tol_H + 2.0 ** -149


def top(z, k, T):
    """ids and log probabilities of the k largest logits; -1 and -inf behind the unmasked ones."""
    row = Row(z, T)
    if row.bad:
        return np.full(k, -1), np.full(k, np.nan)
    order = np.argsort(-z, kind="stable")[:k]
    on = z[order] > -np.inf
    lps = np.where(on, row.logp[order], -np.inf) if not row.empty else np.full(k, -np.inf)
    return np.where(on, order, -1), lps


def scores_grad(z, token, T, g, h, entropy, dtype):
    """The gradient of one row and its tolerance; entropy: the float32 that the call is given."""
    n = z.size
    if token < 0:
        g = 0.0
    row = Row(z, T)
    if g == 0.0 and h == 0.0 or row.empty:
        return np.zeros(n), np.zeros(n)
    if row.bad or token >= n:
        return np.full(n, np.nan), np.zeros(n)
    one = np.zeros(n)
    if token >= 0:
        one[token] = 1.0
    grad = (g * (one - row.p) - h * (row.plogp + row.p * row.H)) / row.T
    if token >= 0:  # 1 - p without losing its digits
        grad[token] = (-g * np.expm1(row.logp[token]) - h * (row.plogp[token] + row.p[token] * row.H)) / row.T
    logp = np.where(row.p > 0, np.abs(row.logp), 0.0)
    size = row.p * (abs(g) + abs(h) * (logp + row.H))
    # p carries its own e (6 h |t| + 2 h), the sum's error and four roundings; H its tolerance
    tol = size * (H * (16 + 6 * row.at) + row.tol_L) + abs(h) * row.p * (row.tol_H + row.tol_L)
    if token >= 0:
        tol[token] += abs(g) * (row.tol_L * (1 - np.exp(-row.r) + row.p[token]) + 4 * H * abs(np.expm1(row.logp[token])))
        tol[token] += abs(g) * row.tol_L
    return grad, tol / row.T + np.abs(grad) * DTYPES[dtype][2] * 1.01 + _least(dtype)


def distill(z, ids, v, T, rest, weight, dtype):
    """(loss, tolerance, gradient, tolerance) of one row, the gradient that of weight * loss."""
    n = z.size
    used = (ids >= 0) & (v != -np.inf)
    zeros = np.zeros(n)
    if not used.any() or weight == 0.0:
        return 0.0, 0.0, zeros, zeros
    row = Row(z, T)
    if (ids[used] >= n).any() or not (v[used] < np.inf).all() or row.bad:
        return np.nan, 0.0, np.full(n, np.nan), zeros
    if row.empty:
        return np.inf, 0.0, zeros, zeros
    T = row.T
    ids, v = ids[used].astype(np.int64), v[used].astype(np.float64)
    if not rest:
        v = v - v.max()
        v = v - np.log(np.exp(v).sum())
    p = np.exp(v)
    terms = np.where(p > 0, p * (v - np.where(p > 0, row.logp[ids], 0.0)), 0.0)
    teacher = np.zeros(n)
    np.add.at(teacher, ids, p)
    loss = terms.sum()
    mass = p.sum()
    grad = mass * row.p - teacher
    size = mass * row.p
    tol = 0.0
    if rest:
        outside = np.ones(n, bool)
        outside[ids] = False
        outside &= z > -np.inf
        left = np.where(outside, row.p, 0.0).sum()
        over = max(0.0, 1.0 - mass) if outside.any() else 0.0
        if over > 0.0:
            q = np.where(outside, row.p / left, 0.0)
            with np.errstate(divide="ignore"):
                loss += over * (np.log(over) - np.log(left))
            grad += over * (row.p - q)
            size = size + over * (row.p + q)
            mean = float((q * row.at).sum())
            tol += over * (32 + 6 * mean) * H
            size_tol = over * q * (32 + 6 * mean) * H
        else:
            size_tol = 0.0
    else:
        size_tol = 0.0
    # L over all logits, by the sum outside the list where rest is set: the
    # terms are formed in 64 bits
    most = row.tol_L + H * row.L + (32 + 6 * float((row.p * row.at).sum())) * H
    tol = T * T * (tol + mass * most) + 1e-12
    loss = T * T * loss
    gtol = T * (size * (H * (16 + 6 * row.at) + most) + size_tol)
    gtol = np.abs(weight) * gtol + np.abs(weight * T * grad) * DTYPES[dtype][2] * 1.01 + _least(dtype)
    return weight * loss, abs(weight) * tol + 2 * H * abs(weight * loss), weight * T * grad, gtol
