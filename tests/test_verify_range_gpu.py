"""Draft verification on the GPU against 64-bit numpy: logits far from 0, the longest vocabulary."""
import numpy as np
import pytest

from test_verify_gpu import case, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("temperature", [1e-6, 0.3, 1.0, 1e6])
@pytest.mark.parametrize("size", [1e9, 1e13, 1e16, 1e20, 3.4028235e38])
def test_verify_logits_far_from_zero(lb, ctx, size, temperature, probs):
    """rows that are all at one value as far from 0 as the type goes (nothing but masked tokens, say), or one step of the type apart: what is left are the differences"""
    c = case(9000, [1, 1, 1, 0], seed=31)
    size = np.float32(size)
    for row, sign in ((0, -1), (1, 1), (2, -1), (3, 1), (4, -1), (5, 1), (6, -1)):
        c["logits"][row] = sign * size
    c["logits"][[0, 3], ::2] = np.nextafter(c["logits"][[0, 3], ::2], np.float32(0))
    c["u_accept"][:], c["probs"][:, 77] = 0.999, 0.5
    c["drafts"][:], c["best"][:] = 77, 77
    run(lb, ctx, c, temperature, 0, probs)


def test_verify_longest_vocabulary(lb, ctx):
    """2^24 logits nearly alike: a probability is 2^-24, and that of a logit 692.9 below them 2^-1023"""
    V = 1 << 24
    c = case(8, [1], seed=32)
    l, q = np.zeros((2, V), np.float32), np.full((2, V), 2.0 ** -24, np.float32)
    l[:, [3, 9000000]] = -692.9
    l[:, 8] = -692.5
    q[0, [3, 8, 9000000]], q[0, 77] = np.nan, 0.5
    c.update(logits=l, probs=q, drafts=np.array([77, 0], np.int32), best=np.array([8, 0], np.int32), u_accept=np.full(2, 0.999, np.float32))
    for u in (0.0, 0.3, 1.0):
        c["u_pick"][:] = u
        for probs in (True, False):
            run(lb, ctx, c, 1.0, 0, probs, tol=2.0 ** -14)
    q[0] = 0.5  # nothing is left of p: from p itself
    run(lb, ctx, c, 1.0, 0, tol=2.0 ** -14)
