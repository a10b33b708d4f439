"""How far the batch attention may be from 64 bits: bounds for queries and weights of two fp16 terms each."""
import numpy as np


def close(q, key, value, limit):
    """One query q [dim] (normalised, rotated) over rows 0..limit: the result, and how far the kernel's may be from it before the output's rounding.
    Scores: q in two terms of 11 bits, 2^-22 of an element; sums of 32 bits, cut off at 2^-22 of what is added at each of the four steps of a group and the join of the groups; scale and
    log2(e) / sqrt(dim) 2^-22: less than 2^-19 of sum |q| |k_t| / sqrt(dim).
    Weights: the exponential's argument, up to 2^5 here, rounded to 24 bits (2^-20), its own 2^-22, two terms 2^-22 twice; the sums of weight times code and of weight times lowest as
    above: less than 2^-18 of what is added, a code taken as 15.
    Products of a code are cut off at 2^-19 of a code times the largest of the 16 operands that are added at a time (and so is what was added up before).  A first term has 11 bits, so only
    operands below 2^-8 of the largest lose by that: features of a group, here all of its 64 against its largest; rows of a block.
    Below 2^-23 of the largest, weights (and weights times scales) keep their place and lose bits: 2^-45 of the largest each; 2^-44 for the reference's place."""
    dim = q.shape[0]
    (kl, ks, kc), (vl, vs, vc) = ([x[:limit + 1] for x in p] for p in (key, value))
    k, v = kl + ks * kc, vl + vs * vc
    s = k @ q / np.sqrt(dim)
    p = np.exp(s - s.max())
    p /= p.sum()
    out = p @ v
    d = 2.0 ** -19 * ((np.abs(kl) + ks * kc) @ np.abs(q)) / np.sqrt(dim)
    for g in range(0, dim, 64):
        large = np.abs(q[g:g + 64]).max()
        d += 2.0 ** -19 * ks[:, g] * large * ((np.abs(q[g:g + 64]) < 2.0 ** -8 * large).sum() + 4) / np.sqrt(dim)
    tol = (p * np.expm1(d + d.max())) @ np.abs(v - out) + 2.0 ** -18 * (p @ (np.abs(vl) + 15 * vs))
    tol += 2.0 ** -44 * (p.max() * np.abs(vl).sum(0) + (p[:, None] * vs).max(0) * vc.sum(0))
    w = np.zeros((-(-(limit + 1) // 16) * 16, dim))
    w[:limit + 1] = p[:, None] * vs
    w = w.reshape(-1, 16, dim)
    large = w.max(1)
    tol += 2.0 ** -19 * (large * ((w < 2.0 ** -8 * large[:, None]).sum(1) + 1)).sum(0)
    return out, tol


def rounded(out, tol):
    """and behind the output's rounding to fp16"""
    return tol + 2.0 ** -11 * (np.abs(out) + tol) + 2.0 ** -25


def terms(x, n):
    """x in n fp16 terms, scaled by a power of two as the kernel does: the largest to [2^13, 2^14)"""
    up = 2.0 ** (13 - np.floor(np.log2(np.abs(x).max())))
    out = np.zeros_like(x)
    for _ in range(n):
        out += (x * up - out).astype(np.float16).astype(np.float64)
    return out / up


def attend_in_terms(q, key, value, limit, q_terms, w_terms):
    """attention in 64 bits but for queries, probabilities and probabilities times scales, which have so many terms of 11 bits"""
    (kl, ks, kc), (vl, vs, vc) = ([x[:limit + 1] for x in p] for p in (key, value))
    s = (kl + ks * kc) @ terms(q, q_terms) / np.sqrt(len(q))
    p = np.exp(s - s.max())
    rounded_p = terms(p, w_terms)
    out = rounded_p @ vl
    for g in range(len(q) // 64):
        out[64 * g:64 * g + 64] += terms(p * vs[:, 64 * g], w_terms) @ vc[:, 64 * g:64 * g + 64]
    return out / rounded_p.sum()
