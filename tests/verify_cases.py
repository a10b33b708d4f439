"""Drafted tokens against the target's probabilities in 64 bits, one request after the other."""
import numpy as np


def distribution(logits, temperature, top_k):
    """(tokens in the order in which their weights are summed, probabilities)"""
    l = np.asarray(logits, np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    if temperature <= 0:
        return np.array([int(l.argmax())]), np.ones(1)
    names = np.argsort(-l, kind="stable")[:top_k] if top_k else np.arange(len(l))
    names = names[l[names] > -np.inf]
    if not len(names):
        return np.array([0]), np.zeros(1)
    d = l[names]
    with np.errstate(invalid="ignore"):
        e = np.exp(np.where(d == d.max(), 0.0, d - d.max()) / temperature)
    return names, e / e.sum()


def pick(names, weight, u):
    total = np.cumsum(weight)
    if not total[-1] > 0:
        return int(names[0])
    over = np.nonzero(total > u * total[-1])[0]
    return int(names[over[0]]) if len(over) else int(names[np.nonzero(weight)[0][-1]])


def verify(logits, starts, drafts, probs, u_accept, u_pick, temperature, top_k, rows):
    tokens, accepted, p_out = np.full(rows, -9, np.int32), np.full(len(starts) - 1, -1, np.int32), np.full(rows, -9.0)
    for r in range(len(starts) - 1):
        first, end = starts[r], starts[r + 1]
        if end == first:
            continue
        stop = None
        for row in range(first, end):
            names, p = distribution(logits[row], temperature, top_k)
            x, inner = int(drafts[row]), row < end - 1
            there = np.nonzero(names == x)[0]
            px = p[there[0]] if len(there) and inner else 0.0
            p_out[row] = px
            q = np.zeros(len(names))
            if temperature <= 0:
                stands = px > 0 and logits[row][x] > -np.inf
                if not stands:
                    p_out[row] = 0.0
            else:
                qx = 0.0
                if 0 <= x < len(logits[row]):
                    qx = 1.0 if probs is None else float(probs[row][x])
                stands = float(u_accept[row]) * qx < px
                q = (names == x).astype(float) if probs is None else probs[row][names].astype(np.float64)
            if stop is None and not (inner and stands):
                stop = row
                w = np.maximum(p - np.where(q > 0, q, 0), 0) if inner and temperature > 0 else p
                token = pick(names, w if w.sum() > 0 else p, float(u_pick[r]))
        tokens[first:end] = -1
        tokens[first:stop] = drafts[first:stop]
        tokens[stop] = token
        accepted[r] = stop - first
    return tokens, accepted, p_out
