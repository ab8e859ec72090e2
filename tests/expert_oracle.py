"""Routed experts from their definitions, in 64 bits and sample by sample (the tests' oracle; CPU)."""
import math

import torch


def route(z, k, renorm, dw=None):
    """(weights, experts, gradient of z) for float64 logits ``[T, E]``."""
    T, E = z.shape
    w, ids, dz = torch.zeros(T, k).double(), torch.full((T, k), -1), torch.zeros(T, E).double()
    for t in range(T):
        row = z[t].tolist()
        order = sorted((e for e in range(E) if row[e] > -math.inf), key=lambda e: (-row[e], e))[:k]
        among = order if renorm else [e for e in range(E) if row[e] > -math.inf]
        total = sum(math.exp(row[e] - row[order[0]]) for e in among)
        for j, e in enumerate(order):
            ids[t, j], w[t, j] = e, math.exp(row[e] - row[order[0]]) / total
        if dw is not None:
            s = sum(float(w[t, j] * dw[t, j]) for j in range(len(order)))
            for e in among:
                p = math.exp(row[e] - row[order[0]]) / total
                dz[t, e] = p * ((float(dw[t, order.index(e)]) if e in order else 0.0) - s)
    return w, ids, dz


def plan(ids, E, capacity):
    """(position, source, load, offsets) as lists, from ``ids`` ``[T, k]``."""
    T, k = ids.shape
    lists = [[] for _ in range(E)]
    for i, e in enumerate(ids.reshape(-1).tolist()):
        if 0 <= e < E:
            lists[e].append(i)
    rows = E * capacity if capacity else T * k
    position, source, offsets, at = [-1] * (T * k), [-1] * rows, [], 0
    for e in range(E):
        at = e * capacity if capacity else at
        offsets.append(at)
        for r, i in enumerate(lists[e]):
            if not capacity or r < capacity:
                position[i], source[at + r] = at + r, i
        at += capacity if capacity else len(lists[e])
    return position, source, [len(v) for v in lists], offsets + [at]


def dispatch(x, position, rows, k):
    out = torch.zeros(rows, x.shape[1]).double()
    for i, r in enumerate(position):
        if r >= 0:
            out[r] = x[i // k]
    return out


def combine(h, position, T, k, w=None):
    y = torch.zeros(T, h.shape[1]).double()
    for i, r in enumerate(position):
        if r >= 0:
            y[i // k] += h[r] * (1.0 if w is None else w[i // k, i % k])
    return y
