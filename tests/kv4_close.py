"""How far the batch attention may be from 64 bits: bounds for queries and weights of two fp16 terms each."""
import numpy as np


def close(q, key, value, limit):
    """One query q [dim] (normalised, rotated) over rows 0..limit: the result, and how far the kernel's may be from it before the output's rounding.
    Scores: q in two terms of 11 bits, 2^-22 of an element; sums of 32 bits whose products' additions are cut off, 2^-22 of what is added at each of the four steps of a group and the join of
    the groups; scale and log2(e) / sqrt(dim) 2^-22: less than 2^-19 of sum |q| |k_t| / sqrt(dim).
    Weights: the exponential's argument, up to 2^5 here, rounded to 24 bits (2^-20), its own 2^-22, two terms 2^-22 twice; the same for the sums of weight times code, in which a code is the
    difference of two sums with one neighbour: less than 2^-18 of what is added, a code taken as 15.
    Below 2^-23 of the largest, weights (and weights times scales) keep their place and lose bits: 2^-45 of the largest each; 2^-44 for the reference's place."""
    dim = q.shape[0]
    (kl, ks, kc), (vl, vs, vc) = ([x[:limit + 1] for x in p] for p in (key, value))
    k, v = kl + ks * kc, vl + vs * vc
    s = k @ q / np.sqrt(dim)
    p = np.exp(s - s.max())
    p /= p.sum()
    out = p @ v
    d = 2.0 ** -19 * ((np.abs(kl) + ks * kc) @ np.abs(q)) / np.sqrt(dim)
    tol = (p * np.expm1(d + d.max())) @ np.abs(v - out) + 2.0 ** -18 * (p @ (np.abs(vl) + 15 * vs))
    tol += 2.0 ** -44 * (p.max() * np.abs(vl).sum(0) + (p[:, None] * vs).max(0) * vc.sum(0))
    return out, tol


def rounded(out, tol):
    """and behind the output's rounding to fp16"""
    return tol + 2.0 ** -11 * (np.abs(out) + tol) + 2.0 ** -25
