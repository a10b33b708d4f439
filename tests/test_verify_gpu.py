"""Draft verification on the GPU against 64-bit numpy: the same tokens, the same counts; probabilities to the last bits of fp32."""
import numpy as np
import pytest

import verify_cases as vc

pytestmark = pytest.mark.gpu


def case(V, drafts, seed=1, spread=2.0, noise=0.7, temperature=1.0, spare=0):
    rng = np.random.default_rng(seed)
    starts = np.concatenate([[0], np.cumsum([d + 1 if d >= 0 else 0 for d in drafts])]).astype(np.int32)
    rows = int(starts[-1]) + spare
    logits = (spread * rng.standard_normal((rows, V))).astype(np.float32)
    guess = logits + noise * rng.standard_normal((rows, V)).astype(np.float32)
    q = np.exp((guess - guess.max(1, keepdims=True)) / (temperature or 1.0))
    q = (q / q.sum(1, keepdims=True)).astype(np.float32)
    cum = np.cumsum(q.astype(np.float64), 1)
    drawn = (cum < rng.random((rows, 1)) * cum[:, -1:]).sum(1).clip(max=V - 1).astype(np.int32)
    return {"logits": logits, "starts": starts, "probs": q, "drafts": drawn, "best": guess.argmax(1).astype(np.int32), "rows": rows, "n": len(drafts),
            "u_accept": rng.random(rows).astype(np.float32), "u_pick": rng.random(len(drafts)).astype(np.float32)}


def run(lb, ctx, c, temperature, top_k, probs=True, shift=0, want_p=True, tol=2.0 ** -18):
    """the call's results, checked against the plain form"""
    V, n, rows = c["logits"].shape[1], c["n"], c["rows"]
    drafts = c["drafts"] if probs else c["best"]
    flat = np.concatenate([np.zeros(shift, np.float32), c["logits"].ravel()])
    d = {k: ctx.to_device(v) for k, v in (("l", flat), ("s", c["starts"]), ("d", drafts), ("q", c["probs"]), ("a", c["u_accept"]), ("u", c["u_pick"]))}
    tokens, accepted, p_out = ctx.to_device(np.full(rows, -9, np.int32)), ctx.to_device(np.full(n, -9, np.int32)), ctx.to_device(np.full(rows, -9, np.float32))
    logits = type("At", (), {"ptr": d["l"].ptr + 4 * shift})
    ctx.verify_drafts(logits, V, d["s"], n, rows, d["d"], d["q"] if probs else None, d["a"], d["u"], tokens, accepted, temperature, top_k, p_out if want_p else None)
    got = tokens.download(np.int32, rows), accepted.download(np.int32, n), p_out.download(np.float32, rows)
    assert ctx.device_status() == 0
    want = vc.verify(c["logits"], c["starts"], drafts, c["probs"] if probs else None, c["u_accept"], c["u_pick"], temperature, top_k, rows)
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0])
    # a row's sum is one of 32-bit exponentials: arguments to 2^-23 of themselves, weighted by what they add at most 2^-18 here; the output's rounding 2^-24
    if want_p:
        assert np.allclose(got[2], want[2], rtol=tol, atol=1e-30)
    else:
        assert (got[2] == -9).all()
    for b in (*d.values(), tokens, accepted, p_out):
        b.free()
    return got


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("top_k", [0, 1, 7, 50, 64])
@pytest.mark.parametrize("V,shift", [(1, 0), (5, 1), (63, 0), (1000, 0), (4096, 2), (32768, 0), (50001, 3)])
def test_verify(lb, ctx, V, shift, top_k, probs):
    run(lb, ctx, case(V, [3, 0, 5, 1, -1, 2], seed=V + top_k), 0.8, top_k, probs, shift)


@pytest.mark.parametrize("top_k", [0, 20])
def test_verify_large_vocabulary(lb, ctx, top_k):
    got = run(lb, ctx, case(248320, [4, 2, 3], seed=3, spread=1.0, noise=1.0), 1.0, top_k)
    run(lb, ctx, case(300007, [2, 1], seed=4), 0.5, top_k, probs=False)  # more than a cluster's threads hold at once
    assert (got[1] <= [4, 2, 3]).all()


@pytest.mark.parametrize("V", [2, 1000, 40000])
def test_verify_greedy(lb, ctx, V):
    c = case(V, [4, 0, 2, 6], seed=V, noise=0.1)
    run(lb, ctx, c, 0.0, 0, probs=False)
    run(lb, ctx, c, -1.0, 30, probs=True)
    c["logits"][:, :] = np.float32(0.5)  # all equal: the first index
    c["best"][:3] = 0
    got = run(lb, ctx, c, 0.0, 0, probs=False)
    assert got[1][0] == 3


@pytest.mark.parametrize("top_k", [0, 50])
@pytest.mark.parametrize("u", [0.0, np.float32(1 - 2.0 ** -24), 1.0])
def test_verify_ends_of_the_uniform_range(lb, ctx, u, top_k):
    """u = 0 takes the first token with weight, u just below 1 the last; 0 accepts whatever has probability"""
    c = case(3000, [2, 3, 0], seed=11)
    c["u_accept"][:], c["u_pick"][:] = u, u
    run(lb, ctx, c, 1.0, top_k)
    run(lb, ctx, c, 1.0, top_k, probs=False)


@pytest.mark.parametrize("top_k", [0, 5, 64])
def test_verify_masked_logits(lb, ctx, top_k):
    """-infinity almost everywhere, everywhere, the type's lowest value, NaN, +infinity"""
    c = case(9000, [2, 2, 2, 2, 2], seed=12)
    l, low = c["logits"], np.finfo(np.float32).min
    l[0:3] = np.where(np.arange(9000) % 3000 == 17, l[0:3], -np.inf)  # three tokens each
    l[3:6] = -np.inf
    l[6:9] = np.where(np.arange(9000) % 1000 == 5, l[6:9], low)
    l[9:12, ::7] = np.nan
    l[12:15, [100, 8000]] = np.inf
    c["drafts"][[0, 1]], c["drafts"][12] = (17, 3017), 8000
    run(lb, ctx, c, 1.0, top_k)
    run(lb, ctx, c, 0.0, 0, probs=False)
    c["best"][[0, 6, 12]] = (17, 5, 100)
    run(lb, ctx, c, 0.7, top_k, probs=False)


@pytest.mark.parametrize("V", [3000, 70000])
def test_verify_many_equal_logits(lb, ctx, V):
    """more equal logits than are sorted at once: the smaller indices are taken"""
    c = case(V, [2, 3], seed=13)
    c["logits"][:, ::2] = 9.0
    c["logits"][1] = np.float32(-3.0)
    c["logits"][2, : V // 2] = np.sort(c["logits"][2, : V // 2])  # and a thread's own logits all large or all small
    run(lb, ctx, c, 1.0, 33)
    run(lb, ctx, c, 1.0, 64, probs=False)


@pytest.mark.parametrize("temperature", [1e-6, 0.01, 1e6])
def test_verify_temperatures(lb, ctx, temperature):
    """from nearly greedy to uniform; logits far from 0 and far apart"""
    c = case(5000, [3, 2], seed=19, temperature=1.0)
    c["logits"][0:4] += np.float32(1e4)
    c["logits"][5, 10] = np.float32(3e38)
    c["logits"][6] *= np.float32(1e30)
    for top_k in (0, 30):
        run(lb, ctx, c, temperature, top_k, tol=2.0 ** -16)
        run(lb, ctx, c, temperature, top_k, probs=False, tol=2.0 ** -16)


def test_verify_draft_equals_target(lb, ctx):
    """q = p to rounding: drafts stand for every u below 1, and a residue of rounding falls back to p"""
    c = case(500, [3, 3], seed=14, noise=0.0)
    run(lb, ctx, c, 1.0, 0)
    c["probs"][:] = 2.0  # no probabilities at all: nothing is left of p, so p itself gives the token
    c["u_accept"][:] = 0.9
    run(lb, ctx, c, 1.0, 0)
    run(lb, ctx, c, 1.0, 10)
    c["probs"][:] = np.nan
    c["u_accept"][:] = 0.5
    got = run(lb, ctx, c, 1.0, 0)
    assert (got[1] == 0).all()


def test_verify_drafts_out_of_the_vocabulary(lb, ctx):
    c = case(700, [3, 2], seed=15)
    c["drafts"][[0, 5]] = (-1, 700)
    c["best"][[1, 4]] = (2 ** 31 - 1, -2 ** 31)
    for top_k in (0, 9):
        run(lb, ctx, c, 1.0, top_k)
        run(lb, ctx, c, 1.0, top_k, probs=False)
    run(lb, ctx, c, 0.0, 0, probs=False)


def test_verify_many_requests_and_rows_left_alone(lb, ctx):
    rng = np.random.default_rng(16)
    c = case(300, rng.integers(-1, 9, 256).tolist(), seed=16, spare=4)
    for top_k in (0, 12):
        got = run(lb, ctx, c, 0.9, top_k, want_p=top_k == 0)
        assert (got[0][-4:] == -9).all()


def test_verify_bottom_row_agrees_with_sampling(lb, ctx):
    """without drafts the token is lb_sample_topk's, for its uniform number"""
    V, k, seed = 5000, 40, 77
    u = lb.fill_uniform(64, seed, 7777, 0.0, 1.0)
    rng = np.random.default_rng(17)
    for counter in (0, 5, 63):
        x = (2 * rng.standard_normal(V)).astype(np.float32)
        d, out, idx = ctx.to_device(x), ctx.alloc(16), ctx.alloc(16)
        ctx.sample_topk(d, V, 0.8, k, seed, counter, idx)
        one = [ctx.to_device(np.array(a)) for a in (np.array([0, 1], np.int32), np.array([0], np.int32), np.array([0.5], np.float32), u[counter:counter + 1])]
        acc = ctx.alloc(16)
        ctx.verify_drafts(d, V, one[0], 1, 1, one[1], None, one[2], one[3], out, acc, float(np.float32(0.8)), k)
        assert out.download(np.int32, 1)[0] == idx.download(np.int32, 1)[0]


def test_verify_bad_requests(lb, ctx):
    c = case(100, [2, 2], seed=18)
    d = [ctx.to_device(a) for a in (c["logits"], c["drafts"], c["u_accept"], c["u_pick"])]
    tokens, accepted = ctx.to_device(np.full(6, -9, np.int32)), ctx.to_device(np.full(2, -9, np.int32))
    for starts, want in (([0, 3, 7], [True, False]), ([-1, 3, 6], [False, True]), ([3, 0, 3], [False, True])):
        s = ctx.to_device(np.array(starts, np.int32))
        ctx.verify_drafts(d[0], 100, s, 2, 6, d[1], None, d[2], d[3], tokens, accepted, 1.0, 0)
        with pytest.raises(lb.LithosError, match="0x1006"):
            ctx.device_status()
        assert [a >= 0 for a in accepted.download(np.int32)[:2]] == want
        s.free()


def test_verify_refusals(lb, ctx):
    b = ctx.alloc(4096)
    null, odd = type("At", (), {"ptr": 0}), type("At", (), {"ptr": b.ptr + 2})
    good = [b, 10, b, 1, 2, b, None, b, b, b, b, 1.0, 0, None]
    for i, v in ((0, null), (0, odd), (1, 0), (1, (1 << 24) + 1), (2, null), (3, 0), (3, 257), (4, 0), (4, 8193), (5, null), (6, odd), (7, null), (8, null), (9, null), (10, null),
                 (11, float("nan")), (11, float("inf")), (11, 1e-7), (11, 1e7), (12, -1), (12, 65), (13, odd)):
        a = list(good)
        a[i] = v
        with pytest.raises(lb.LithosError) as e:
            ctx.verify_drafts(*a)
        assert e.value.status == lb.LB_ERR_INVALID
    b.free()


def test_verify_captured(lb, ctx):
    """captured once, replayed on new logits: the same as the call"""
    a, b = case(20000, [3, 1, 2], seed=20), case(20000, [3, 1, 2], seed=21)
    names = ("logits", "starts", "drafts", "probs", "u_accept", "u_pick")
    for top_k in (0, 25):
        want = [run(lb, ctx, c, 1.0, top_k) for c in (a, b)]
        d = [ctx.to_device(a[k]) for k in names]
        tokens, accepted, p = ctx.alloc(4 * a["rows"]), ctx.alloc(4 * 3), ctx.alloc(4 * a["rows"])
        ctx.begin_capture()
        ctx.verify_drafts(d[0], 20000, d[1], 3, a["rows"], d[2], d[3], d[4], d[5], tokens, accepted, 1.0, top_k, p)
        g = ctx.end_capture()
        for c, w in zip((a, b), want):
            for buf, k in zip(d, names):
                buf.upload(c[k])
            g.launch()
            assert np.array_equal(tokens.download(np.int32), w[0]) and np.array_equal(accepted.download(np.int32), w[1]) and np.array_equal(p.download(np.float32), w[2])
        g.destroy()
