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


@pytest.mark.parametrize("V,rows", [(248320, 192), (50257, 300), (32768, 8), (1 << 24, 5)])
def test_verify_long_sums(lb, ctx, V, rows):
    """p to 2^-19 of itself where it hangs on a long sum: most of a row's weight in logits alike, some way below a few"""
    rng = np.random.default_rng(33)
    gap = np.linspace(1, 17, rows)
    l = np.zeros((rows, V), np.float32)
    for i in range(rows):
        l[i, rng.integers(0, V, 3)] = gap[i]
    drafts = rng.integers(0, V, rows).astype(np.int32)
    u = np.full(rows, 0.5, np.float32)
    s, d = ctx.to_device(np.array([0, rows], np.int32)), {k: ctx.to_device(a) for k, a in (("l", l), ("d", drafts), ("u", u))}
    tokens, accepted, p = ctx.alloc(4 * rows), ctx.alloc(4), ctx.alloc(4 * rows)
    for temperature in (1.0, 0.7, 1.3):
        ctx.verify_drafts(d["l"], V, s, 1, rows, d["d"], None, d["u"], d["u"], tokens, accepted, temperature, 0, p)
        got, worst = p.download(np.float32), 0.0
        for i in range(rows - 1):
            x = l[i].astype(np.float64) / temperature
            want = np.exp(x[drafts[i]] - x.max()) / np.exp(x - x.max()).sum()
            worst = max(worst, abs(got[i] / want - 1))
        assert worst <= 2.0 ** -19, np.log2(worst)
    for b in (s, *d.values(), tokens, accepted, p):
        b.free()
