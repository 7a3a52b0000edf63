"""Embeddings, their gradient, and the norm and clipping of gradients in 64 bits, with
how far results of 32-bit arithmetic, rounded once to their type, may be from them."""
import numpy as np

from adjust64 import rounded, within


def embedding(table, tokens, scale, dtype):
    """(rows, tolerance): one 32-bit product and the rounding."""
    table, tokens = np.asarray(table, np.float64), np.asarray(tokens)
    out = np.zeros((tokens.size, table.shape[1]))
    real = (tokens >= 0) & (tokens < table.shape[0])
    with np.errstate(all="ignore"):
        out[real] = within(within(table[tokens[real]] * scale, "f32"), dtype)
    out[tokens >= table.shape[0]] = np.nan
    return out, 1.01 * 2.0**-24 * np.abs(out) + rounded(out, dtype)


def gradient(tokens, grad, vocab, scale, dtype, old=None):
    """(gradient of the table, tolerance).  k rows are added in some order with k - 1
    roundings, each at most 2^-24 of the magnitudes' sum; then a rounding of the joined
    sums, the product's, and the sum's with what was there."""
    tokens, grad = np.asarray(tokens), np.asarray(grad, np.float64)
    out, size, n = np.zeros((vocab, grad.shape[1])), np.zeros((vocab, grad.shape[1])), np.zeros(vocab)
    for t, g in zip(tokens, grad):
        if 0 <= t < vocab:
            out[t] += g
            size[t] += np.abs(g)
            n[t] += 1
    out, size = out * scale, size * abs(scale)
    with np.errstate(all="ignore"):
        tol = 1.01 * 2.0**-24 * (n[:, None] + 1) * size
        if old is not None:
            touched = n > 0
            out = np.where(touched[:, None], out + old, old)
            tol += np.where(touched[:, None], 1.01 * 2.0**-24 * np.abs(out), 0.0)
        return within(out, dtype), tol + np.where(n[:, None] > 0, rounded(out, dtype), 0.0)


def norm(tensors, scale=1.0, largest=False):
    """(norm, tolerance): 64-bit squares and sums are off by less than a 32-bit rounding,
    which is the one that counts; 2^-150 where that is of the smallest numbers."""
    with np.errstate(all="ignore"):
        every = np.concatenate([np.zeros(1)] + [np.asarray(t, np.float64).ravel() for t in tensors])
        v = within(abs(scale) * (np.abs(every).max() if largest else np.sqrt(np.longdouble(1) * (every * every).sum())), "f32")
        return float(v), 1.01 * 2.0**-24 * float(np.abs(v)) + 2.0**-150


def clipped(t, norm, max_norm, scale, dtype):
    """(clipped, tolerance): the factor's rounding, the product's, and the type's."""
    with np.errstate(all="ignore"):
        c = max_norm / (norm + 1e-6)
        out = within(within(np.asarray(t, np.float64) * (scale * (1.0 if c > 1.0 else c)), "f32"), dtype)
        return out, 1.01 * 2.0**-23 * np.abs(out) + rounded(out, dtype) + 2.0**-149
