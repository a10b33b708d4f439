"""The plain form of draft verification: what it promises, shown on distributions that can be counted."""
import numpy as np

import verify_cases as vc


def test_result_has_the_targets_distribution():
    """over a grid of uniform numbers and all drafts, the first token comes out with the target's probability"""
    rng = np.random.default_rng(0)
    V, n = 6, 60
    logits = rng.standard_normal((2, V)).astype(np.float32)
    q = rng.random(V).astype(np.float32)
    q /= q.sum()
    u = (np.arange(n) + 0.5) / n
    got = np.zeros(V)
    for x in range(V):
        for a in u:
            stands = vc.verify(logits, [0, 2], np.array([x, 0]), np.stack([q, q]), np.array([a, 0]), np.array([0.5]), 0.9, 0, 2)
            if stands[1][0]:
                got[x] += q[x] / n
            else:
                for b in u:
                    t, _, _ = vc.verify(logits, [0, 2], np.array([x, 0]), np.stack([q, q]), np.array([a, 0]), np.array([b]), 0.9, 0, 2)
                    got[t[0]] += q[x] / n / n
    # a grid of n numbers is off by less than 1 / n in each of the two choices
    assert np.abs(got - vc.distribution(logits[0], 0.9, 0)[1]).max() < 2 / n


def test_refused_without_a_context(lb):
    assert lb.lib().lb_verify_drafts(None, 16, 8, 16, 1, 1, 16, 0, 16, 16, 16, 16, 1.0, 0, 0) == lb.LB_ERR_INVALID
