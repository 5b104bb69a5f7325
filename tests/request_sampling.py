"""Sampling with every row's own settings, from its definition in 64 bits
(include/noel_requests.h), for the tests.  Weights are rounded to multiples of
2^-43, as the definition has it, and added as whole numbers: with top-p a
millionth below 1 the ids at the cut have weights near 2^-36, and thousands of
them, so without that rounding counts differ there by ids (each weight's 2^-44,
the same for equal logits, times how many there are)."""
import math
from fractions import Fraction

import numpy as np


def sample_plain(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(ids, probabilities in 64 bits, counts) of rows x [B, V] (any floating type)."""
    B = len(x)
    t = np.ones(B, np.float32) if temperature is None else temperature
    k = np.zeros(B, np.int32) if top_k is None else top_k
    p = np.ones(B, np.float32) if top_p is None else top_p
    q = np.zeros(B, np.float32) if min_p is None else min_p
    rows = [_row(np.asarray(x[b], np.float64), float(u[b]), float(t[b]), int(k[b]), float(p[b]), float(q[b])) for b in range(B)]
    ids, probs, counts = zip(*rows)
    return np.array(ids, np.int32), np.array(probs), np.array(counts, np.int32)


def _row(x, u, t, k, p, q):
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    if m == -np.inf:
        return -1, 0.0, 0
    if not t > 0:
        return int(np.argmax(x)), 1.0, 1
    with np.errstate(invalid="ignore"):
        left = x == m
        if m < np.inf:
            floor = m - 30.0 * t
            if q > 0:
                log = math.log(min(q, 1.0))
                floor = max(floor, m + (t * log if log else 0.0))
            left = (x >= floor) & (x > -np.inf)
    ids = np.nonzero(left)[0]
    order = np.argsort(-x[ids], kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    ids = ids[order]
    w = np.exp((np.where(x[ids] == m, 0.0, x[ids] - (m if m < np.inf else 0.0))) / t)
    whole = np.rint(w * 2.0**43).astype(np.int64)
    if p < 1:
        want = math.ceil(Fraction(max(p, 0.0)) * int(whole.sum()))
        n = int(np.searchsorted(np.cumsum(whole), max(want, 1))) + 1
        ids, w, whole = ids[:n], w[:n], whole[:n]
    order = np.argsort(ids)
    ids, w, whole = ids[order], w[order], whole[order]
    run = np.cumsum(whole)
    total = int(run[-1])
    target = math.floor(Fraction(min(u, 1.0)) * total) if u > 0 else 0
    at = int(np.searchsorted(run, min(target, total - 1), side="right"))
    return int(ids[at]), float(w[at] / (total * 2.0**-43)), len(ids)
