"""Distillation with the mass outside the list (rest), in 64 bits and in
logarithms, so that no share underflows however far the list's logits lie above
the others; and how far 32-bit results may be from it.

Bounds, with H = 2^-24 and rows64's for a sum of e (relative (32 + 6 U) H, U the
mean |t| under it, and up to 2^-126 a term that the hardware's 2^x gives as 0):
  log q of a listed id, through the sum over the row          tol_L
  log of the sum outside the list, relative to its maximum    tol_O, the same
  what is joined in 64 bits: 2^-50 of every term's size, and 2^-45 for rest = 1 -
  sum p (256 terms of up to 1), times what rest is multiplied with
  a gradient: its e (6 H |t| + 2 H), the sums' errors and the roundings to 32
  bits (16 H in all), of p relative to the row's sum and of q to the outside's;
  2^-126 for an e that is given as 0; the rounding of weight * T to 32 bits; one
  rounding to the gradient's type.
"""
import numpy as np

import rows64
from rows64 import DTYPES, H


def distill_rest(z, ids, v, T, weight, dtype):
    """(loss, tolerance, gradient, tolerance) of one row without NaN or +inf whose
    list has a slot in use; the gradient that of weight * loss."""
    row = rows64.Row(z, T)
    T = row.T
    used = (ids >= 0) & (v != -np.inf)
    ids, v = ids[used].astype(np.int64), v[used].astype(np.float64)
    p = np.exp(v)
    mass = p.sum()
    outside = z > -np.inf
    outside[ids] = False
    rest, q, at_q, log_q_rest, tol_O = 0.0, np.zeros(z.size), np.zeros(z.size), 0.0, 0.0
    if outside.any():
        rest = max(0.0, 1.0 - mass)
        others = rows64.Row(np.where(outside, z, -np.inf), T)
        q, at_q, tol_O = others.p, others.at, others.tol_L
        log_q_rest = (z[outside].max() - z.max()) / T + others.L - row.L
    logq = row.logp[ids]
    term = np.where(p > 0, p * (v - np.where(p > 0, logq, 0.0)), 0.0).sum()
    log_rest = np.log(rest) if rest > 0 else 0.0
    if rest > 0:
        term += rest * (log_rest - log_q_rest)
    large = abs(log_rest) + abs(log_q_rest) if rest > 0 else 0.0
    finite = np.where(np.isfinite(logq), np.abs(logq), 0.0)
    tol = (mass + rest) * row.tol_L + rest * tol_O + 2.0 ** -45 * (1 + large)
    tol += 2.0 ** -50 * ((p * (np.abs(v) + finite)).sum() + (mass + rest) * (1 + row.L) + rest * large)
    loss = T * T * term
    tol = T * T * tol + 2 * H * abs(loss) + 2.0 ** -149

    grad = (mass + rest) * row.p - rest * q
    np.add.at(grad, ids, -p)
    gtol = (mass + rest) * row.p * (H * (16 + 6 * row.at) + row.tol_L) + rest * q * (H * (16 + 6 * at_q) + tol_O)
    gtol = T * abs(weight) * (gtol + (mass + 2 * rest) * 2.0 ** -126 + 2.0 ** -45)
    grad = weight * T * grad
    gtol += np.abs(grad) * (H + DTYPES[dtype][2] * 1.01) + rows64._least(dtype)
    return weight * loss, abs(weight) * tol + 2 * H * abs(weight * loss), grad, gtol
