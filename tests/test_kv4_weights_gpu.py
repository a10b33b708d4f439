"""Weights of the batch attention far below the largest, and scales far apart: against 64 bits, with bounds for the 22 bits that the header gives."""
import numpy as np
import pytest

import kv4_cases as kc
from kv4_close import close, rounded
from test_kv4_gpu import attention

pytestmark = pytest.mark.gpu


def rows_case(ctx, dim, length, new, below, scale, seed, heads=2):
    """One sequence whose row t has a score below[t] under 0 in log2 units (and 0.1 to both sides) and values of scale scale[t]"""
    case = kc.Case(ctx, dim, heads, 2, -(-length // 16) * 16, seqs=[1], pos=[length - new], new=[new], seed=seed)
    S, rows = dim // 64, case.max_ctx
    rng = np.random.default_rng(seed)
    fill = lambda a: np.concatenate([a, np.zeros(rows - len(a))]).reshape(1, rows // 16, 1, 16)  # noqa: E731
    pairs = case.cache[1, :, :, 16 * dim:].copy().view(np.float16).reshape(heads, rows // 16, 2, S, 16, 2)
    shape = pairs.shape[:2] + pairs.shape[3:5]
    pairs[:, :, 0, :, :, 0] = 0.02 / 15 * rng.random(shape)
    pairs[:, :, 0, :, :, 1] = np.broadcast_to(fill(-np.asarray(below) * np.log(2) / np.sqrt(dim)), shape)
    s = fill(np.asarray(scale, np.float64)) * (0.5 + rng.random(shape))
    pairs[:, :, 1, :, :, 0] = s.clip(max=8700)
    pairs[:, :, 1, :, :, 1] = (s * (rng.random(shape) - 7.5)).clip(-65504, 65504)
    case.cache[1, :, :, 16 * dim:] = pairs.view(np.uint8).reshape(heads, rows // 16, -1)
    case.d_cache.upload(case.cache)
    return case


def check(lb, ctx, case, G, seed=3, tokens=None):
    rng, D, HQ, new = np.random.default_rng(seed), case.dim, case.heads * G, case.new[0]
    q = 0.5 + rng.random((new, HQ, D))
    q = (q * D / q.sum(-1, keepdims=True)).astype(np.float32)
    d_q, out = ctx.to_device(q), ctx.alloc(new * HQ * D * 2)
    ctx.kv4_attention(case.desc, case.batch, d_q, None, 0, 0, lb.IN_F32, None, out, HQ, new, 0, 1e7, 1e-6)
    got = out.download(np.float16).astype(np.float64).reshape(new, HQ, D)
    assert ctx.device_status() == 0
    for h in range(HQ):
        rows = kc.cache_rows(case.cache, D, 1, h // G, case.pos[0] + new)
        for i in range(new) if tokens is None else tokens:
            want, tol = close(q[i, h].astype(np.float64), *rows, case.pos[0] + i)
            err, tol = np.abs(got[i, h] - want), rounded(want, tol)
            assert (err <= tol).all(), (i, h, float((err / tol).max()), float(np.linalg.norm(got[i, h] - want) / np.linalg.norm(want)))
    for b in (d_q, out):
        b.free()
    case.free()


@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("large,small", [(300, 0.05), (3000, 0.02), (8700, 0.01)])
@pytest.mark.parametrize("dim,length,new", [(64, 500, 1), (64, 1800, 5), (128, 900, 5), (256, 100, 1), (256, 700, 1)])
def test_row_of_large_values_without_weight(lb, ctx, dim, length, new, large, small, where):
    """a row 60 below the largest score has values of another order of magnitude: the others keep their bits"""
    below, scale = np.random.default_rng(1).uniform(0, 6, length), np.full(length, float(small))
    row = {"first": 0, "middle": length // 2, "last": length - new}[where]
    below[row], scale[row] = 60, large
    check(lb, ctx, rows_case(ctx, dim, length, new, below, scale, seed=dim + length), 3)


@pytest.mark.parametrize("dim,length,new", [(64, 1500, 1), (128, 700, 3), (256, 600, 1)])
def test_large_values_behind_a_row_that_has_none(lb, ctx, dim, length, new):
    """the top score's values are 0, those of a row without weight are large: what is left are rows 20 below the one, of a millionth of the other's size"""
    below, scale = np.random.default_rng(2).uniform(20, 22, length), np.full(length, 0.01)
    below[0], scale[0] = 0, 0
    below[5], scale[5] = 70, 8700
    check(lb, ctx, rows_case(ctx, dim, length, new, below, scale, seed=dim), 4)


@pytest.mark.parametrize("where", ["first", "later"])
@pytest.mark.parametrize("gap,spread", [(12, 0), (16.3, 0), (18.3, 0), (18.3, 4), (24, 0), (28, 8)])
@pytest.mark.parametrize("dim,length,new", [(64, 4096, 1), (128, 4096, 2), (256, 4096, 1), (256, 700, 5)])
def test_rows_far_below_the_largest(lb, ctx, dim, length, new, gap, spread, where):
    """one row has the top score and values of 0; the result is the others', all `gap` below it or up to `spread` more"""
    below, scale = gap + spread * np.random.default_rng(3).random(length), np.full(length, 100.0)
    row = 0 if where == "first" else length - 100
    below[row], scale[row] = 0, 0
    check(lb, ctx, rows_case(ctx, dim, length, new, below, scale, seed=dim + new), 3)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows_far_below_the_largest(lb, ctx, dim):
    for gap in (16.3, 20.0):
        below, scale = np.full(100001, gap), np.full(100001, 100.0)
        below[0], scale[0] = 0, 0
        check(lb, ctx, rows_case(ctx, dim, 100001, 1, below, scale, seed=dim, heads=1), 1)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("size", [1e30, 1e35, 2e38])
@pytest.mark.parametrize("dim", [64, 256])
def test_queries_as_large_as_their_type(lb, ctx, dim, size, kind):
    """scores of up to 2^127: one row has all of the weight"""
    case = kc.Case(ctx, dim, 1, 1, 512, seqs=[0], pos=[400], new=[1])
    raw, q = kc.typed(size * np.where(np.arange(2 * dim).reshape(2, dim) % dim < 3, [[1.0], [-0.5]], 0.0), kind)
    d_q, out = ctx.to_device(raw), ctx.alloc(2 * dim * 2)
    # keys of about a thousandth, so that 3 of them times a query and 1 / sqrt(dim) are a number that 32 bits hold
    pairs = case.cache[0, 0, :, 16 * dim:].copy().view(np.float16).reshape(-1, 2, dim // 64, 16, 2)
    pairs[:, 0] *= np.float16(1e-3)
    case.cache[0, 0, :, 16 * dim:] = pairs.view(np.uint8).reshape(len(pairs), -1)
    case.d_cache.upload(case.cache)
    ctx.kv4_attention(case.desc, case.batch, d_q, None, 0, 0, kind, None, out, 2, 1, 0, 1e7, 1e-6)
    got = out.download(np.float16).astype(np.float64).reshape(2, dim)
    (kl, ks, kcode), (vl, vs, vc) = kc.cache_rows(case.cache, dim, 0, 0, 401)
    for h in range(2):
        s = (kl + ks * kcode) @ (q[h] / size)
        best = int(s.argmax())
        assert s[best] - np.delete(s, best).max() > 2.0 ** -20 * np.abs(s).max()  # beyond the scores' own rounding
        want = (vl + vs * vc)[best]
        assert (np.abs(got[h] - want) <= rounded(want, 2.0 ** -18 * (np.abs(vl) + 15 * vs)[best])).all()
    for b in (d_q, out):
        b.free()
    case.free()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("size", [1e15, 1e20, 1e36])
@pytest.mark.parametrize("dim", [64, 256])
def test_normalised_queries_of_any_size(lb, ctx, dim, size, kind):
    """the sum of their squares may be beyond fp32"""
    case = kc.Case(ctx, dim, 2, 1, 512, seqs=[0], pos=[300], new=[2])
    attention(lb, ctx, case, 3, kind, norm=True, rot=32, size=size)
    case.free()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length,size", [(2, 1.0), (30, 3.0), (1000, 3.0), (1000, 8.0), (5000, 1.0)])
def test_two_terms(lb, ctx, dim, length, size):
    """ordinary rows and queries, to the bits of two terms"""
    case = kc.Case(ctx, dim, 2, 2, -(-length // 16) * 16, seqs=[1, 0], pos=[length - 1, length // 2], new=[1, 1])
    rng, G = np.random.default_rng(7), 3
    q = (size * rng.standard_normal((2, 2 * G, dim))).astype(np.float32)
    d_q, out = ctx.to_device(q), ctx.alloc(q.size * 2)
    ctx.kv4_attention(case.desc, case.batch, d_q, None, 0, 0, lb.IN_F32, None, out, 2 * G, 1, 0, 1e7, 1e-6)
    got = out.download(np.float16).astype(np.float64).reshape(q.shape)
    for row, seq, pos in case.places():
        for h in range(2 * G):
            want, tol = close(q[row, h].astype(np.float64), *kc.cache_rows(case.cache, dim, seq, h // G, pos + 1), pos)
            assert (np.abs(got[row, h] - want) <= rounded(want, tol)).all(), (row, h)
    for b in (d_q, out):
        b.free()
    case.free()


@pytest.mark.parametrize("dim,heads,G", [(64, 2, 5), (128, 4, 4), (256, 2, 6)])
def test_a_sequence_alone_and_in_any_batch(lb, ctx, dim, heads, G):
    """where a batch cuts a sequence's rows depends on what else is in it, and so does the order of sums, but not the result beyond the bounds"""
    pos, n = [4000, 10, 700, 2000, 3000, 55], 6
    case = kc.Case(ctx, dim, heads, n, 4096, seqs=range(n), pos=pos, new=[1] * n)
    HQ = heads * G
    q = np.random.default_rng(8).standard_normal((n, HQ, dim)).astype(np.float32)
    rows = [[kc.cache_rows(case.cache, dim, s, h, p + 1) for h in range(heads)] for s, p in enumerate(pos)]
    bounds = [[close(q[s, h].astype(np.float64), *rows[s][h // G], pos[s]) for h in range(HQ)] for s in range(n)]
    starts = ctx.to_device(np.arange(n + 1, dtype=np.int32))
    for batch in ([0], [1], [2], [3], [4], [5], [0, 1, 2, 3, 4, 5], [5, 4, 3, 2, 1, 0], [3, 0, 5, 1], [0, 0, 4, 0]):
        d = [ctx.to_device(np.array(a, np.int32)) for a in (batch, [pos[s] for s in batch])]
        d_q, out = ctx.to_device(q[batch]), ctx.alloc(len(batch) * HQ * dim * 2)
        call = lb.Kv4Batch(d[0].ptr, d[1].ptr, starts.ptr, len(batch), len(batch))
        ctx.kv4_attention(case.desc, call, d_q, None, 0, 0, lb.IN_F32, None, out, HQ, 1, 0, 1e7, 1e-6)
        got = out.download(np.float16).astype(np.float64).reshape(len(batch), HQ, dim)
        for i, s in enumerate(batch):
            for h in range(HQ):
                assert (np.abs(got[i, h] - bounds[s][h][0]) <= rounded(*bounds[s][h])).all(), (batch, i, h)
        for b in (*d, d_q, out):
            b.free()
    starts.free()
    case.free()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("gap", [12.0, 16.3, 18.3, 21.0])
@pytest.mark.parametrize("length", [4096, 100001])
def test_rows_exactly_alike_far_below_the_largest(lb, ctx, dim, length, gap):
    """equal scores and scales, so that every row's weight is rounded to the same side: nothing averages out"""
    case = rows_case(ctx, dim, length, 1, np.where(np.arange(length) == 0, 0.0, gap), np.where(np.arange(length) == 0, 0.0, 0.3), seed=dim, heads=1)
    pairs = case.cache[1, :, :, 16 * dim:].copy().view(np.float16).reshape(1, -1, 2, dim // 64, 16, 2)
    pairs[:, :, 0, :, :, 0] = 0
    pairs[:, :, 1, :, :, 0], pairs[:, :, 1, :, :, 1] = 0.3, -2.25
    pairs[:, 0, 1, :, 0] = 0
    case.cache[1, :, :, 16 * dim:] = pairs.view(np.uint8).reshape(1, pairs.shape[1], -1)
    case.d_cache.upload(case.cache)
    check(lb, ctx, case, 1)
