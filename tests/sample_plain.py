"""Sampling from its definition, a row at a time (numpy; weights in whole multiples of 2^-40 of the first's, sums in whole numbers)."""
import numpy as np


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """-> (token, share)"""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, 0.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not temperature > 0:
        return int(order[0]), 1.0
    if top_k > 0:
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x[order] == top, 0.0, (x[order] - top) / np.float64(np.float32(temperature)))
    exact = np.exp(z)
    w = np.rint(exact * 2.0 ** 40).astype(np.int64)
    keep = exact >= np.float64(np.float32(min_p))
    if top_p < 1:
        before = np.concatenate([[0], np.cumsum(w)[:-1]])
        keep &= (before < np.float64(np.float32(top_p)) * np.float64(w.sum())) | (np.arange(len(w)) == 0)
    order, w = order[keep], w[keep]
    by = np.argsort(order)
    order, w = order[by], w[by]
    c = np.cumsum(w)
    num, den = float(min(max(np.float32(u), np.float32(0)), np.float32(1 - 2.0 ** -24))).as_integer_ratio()
    j = int(np.searchsorted(c, num * int(c[-1]) // den, side="right"))
    return int(order[j]), float(w[j]) / float(c[-1])
