"""Sampling in plain numpy, in 64 bits: one row."""
import numpy as np


def draw(x, u, temperature, top_k, top_p, min_p):
    """(token, logprob, room): ``room``: how far the nearest border of the choice is, in what a sum of weights (or a weight) may be off:
    2^-39 of itself and 2^-45 a weight."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf, np.inf
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, 0.0 if temperature <= 0 else np.exp((x - top) / np.float64(temperature)))
    w = np.where(np.isfinite(x) | (x == top), w, 0.0)
    order = np.argsort(-x, kind="stable")
    k = 1 if temperature <= 0 else top_k if 0 < top_k < len(x) else len(x)
    order = order[:k]
    room = np.inf
    if top_p < 1:
        c = np.cumsum(w[order])
        before, target = c - w[order], np.float64(top_p) * c[-1]
        room = min(room, np.abs(before[1:] - target).min(initial=np.inf) / (c[-1] * 2.0 ** -39 + len(x) * 2.0 ** -45))
        order = order[:max(1, int((before < target).sum()))]
    room = min(room, np.abs(w[order] - min_p).min() / (min_p * 2.0 ** -39)) if 0 < min_p < 1 else room
    order = np.sort(order[w[order] >= min(min_p, 1.0)])
    c = np.cumsum(w[order])
    aim = np.float64(u) * c[-1]
    room = min(room, np.abs(c[:-1] - aim).min(initial=np.inf) / (c[-1] * 2.0 ** -39 + len(x) * 2.0 ** -45))
    i = min(int((c <= aim).sum()), len(order) - 1)
    return int(order[i]), float(np.log(w[order[i]] / c[-1])), room
