"""The 4-bit KV cache on the GPU against 64-bit numpy: rows in and out, attention of ragged batches, refusals."""
import numpy as np
import pytest

import kv4_cases as kc

pytestmark = pytest.mark.gpu
THETA, EPS = 1e7, 1e-6


# ---- rows in, rows out --------------------------------------------------------------------------------------------
def append(lb, ctx, case, kind, norm, rot, gap=0, seed=5, shift=0):
    """new rows for the case's batch; returns the cache's bytes as they should be"""
    rng, H, D = np.random.default_rng(seed), case.heads, case.dim
    width = 2 * H * D + gap
    raw, x = kc.typed(rng.standard_normal((case.rows, width)) * np.exp(rng.standard_normal(width)), kind)
    w = lb.f32_to_bf16((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)) if norm else None
    flat = np.concatenate([np.zeros(shift, raw.dtype), raw.ravel()])
    d_x, d_w = ctx.to_device(flat), ctx.to_device(w) if norm else None

    class At:
        def __init__(self, off):
            self.ptr = d_x.ptr + (shift + off) * raw.itemsize
    ctx.kv4_append(case.desc, case.batch, At(0), At(H * D), width, kind, d_w, rot, THETA, EPS)
    want, written = case.cache.copy(), {}
    for row, seq, pos in case.places():
        written[seq, pos] = row
    for (seq, pos), row in written.items():
        k = kc.norm_rotate(x[row, :H * D].reshape(H, D), pos, kc.bf16_values(w) if norm else None, rot, THETA, EPS)
        put(want, D, seq, pos, k, x[row, H * D:2 * H * D].reshape(H, D))
    got = case.download()
    d_x.free()
    return got, want


def put(cache, D, seq, pos, k, v):
    f = np.arange(D)
    for part, (x, place) in enumerate(((k, kc.key_byte), (v, kc.value_byte))):
        code, scale, lowest = kc.quantise(x)
        for h in range(x.shape[0]):
            blk = cache[seq, h, pos // 16]
            c = code[h].reshape(-1)
            blk[place(D, pos % 16, f[::2])] = c[::2] | c[1::2] << 4
            for g in range(D // 64):
                at = kc.pair_byte(D, part, pos % 16, g)
                pair = np.array([scale[h, g], lowest[h, g]], np.float16)
                blk[at:at + 4] = pair.view(np.uint8)


@pytest.mark.parametrize("dim,heads,kind,norm,rot", [(256, 4, 1, True, 64), (128, 8, 0, False, 128), (64, 1, 2, True, 32), (64, 3, 1, False, 0), (256, 9, 2, True, 256), (128, 2, 1, True, 8)])
def test_append_bytes(lb, ctx, dim, heads, kind, norm, rot):
    """every byte of the cache: the new rows' as the 64-bit form has them, the others' as they were"""
    case = kc.Case(ctx, dim, heads, 4, 64, seqs=[2, 0, 3], pos=[0, 13, 63], new=[1, 6, 1])
    got, want = append(lb, ctx, case, kind, norm, rot)
    assert np.array_equal(got, want)
    case.free()


@pytest.mark.parametrize("shift,gap", [(0, 0), (1, 3), (4, 8)])
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_append_alignments(lb, ctx, kind, shift, gap):
    case = kc.Case(ctx, 64, 2, 2, 32, seqs=[1, 0], pos=[3, 30], new=[17, 2])
    got, want = append(lb, ctx, case, kind, True, 16, gap=gap, shift=shift)
    assert np.array_equal(got, want)
    case.free()


def test_append_far_position(lb, ctx):
    """angles of a position near the longest cache, and a row whose place lies beyond 32 bits of bytes"""
    n, H, D, L = 2, 16, 256, 1 << 20
    big = ctx.alloc(lb.kv4_bytes(n, L, H, D))  # 9.7 GB
    assert big.nbytes > 1 << 33
    rng = np.random.default_rng(9)
    raw, x = kc.typed(rng.standard_normal((1, 2 * H * D)), lb.IN_F32)
    d = [ctx.to_device(np.array([v], np.int32)) for v in (1, L - 1)]
    d_x, k_out, v_out = ctx.to_device(raw), ctx.alloc(H * D * 4), ctx.alloc(H * D * 4)
    cache, batch = lb.Kv4Cache(big.ptr, n, L, H, D), lb.Kv4Batch(d[0].ptr, d[1].ptr, 0, 1, 1)
    v = type("At", (), {"ptr": d_x.ptr + 4 * H * D})
    ctx.kv4_append(cache, batch, d_x, v, 0, lb.IN_F32, None, 256, THETA, EPS)
    ctx.kv4_read(cache, batch, k_out, v_out, lb.IN_F32)
    for out, rows in ((k_out, kc.norm_rotate(x[0, :H * D].reshape(H, D), L - 1, None, 256, THETA, EPS)), (v_out, x[0, H * D:].reshape(H, D))):
        assert np.array_equal(out.download(np.float32).reshape(H, D), kc.values(*kc.quantise(rows)).astype(np.float32))
    for b in (big, d_x, k_out, v_out, *d):
        b.free()


def test_append_same_row_twice(lb, ctx):
    """two requests with the same rows of one sequence: the later one's stay, whole"""
    case = kc.Case(ctx, 128, 4, 2, 64, seqs=[1, 0, 1, 1], pos=[10, 10, 12, 13], new=[6, 6, 6, 1])
    got, want = append(lb, ctx, case, 1, True, 64)
    assert np.array_equal(got, want)
    case.free()


def test_append_special_values(lb, ctx):
    """a constant group, a zero row, values beyond fp16, tiny ones; NaN and infinity make their group NaN and no other"""
    D, H = 128, 1
    case = kc.Case(ctx, D, H, 1, 16, seqs=[0], pos=[0], new=[7])
    x = np.random.default_rng(1).standard_normal((7, 2 * D)).astype(np.float32)
    x[0], x[1], x[2, 3], x[2, 200], x[3] = 1.5, 0.0, 1e6, -3e38, x[3] * 1e-7
    x[4, 5], x[5, 70], x[6, 130] = np.nan, np.inf, -np.inf
    d_x = ctx.to_device(x)
    ctx.kv4_append(case.desc, case.batch, d_x, type("At", (), {"ptr": d_x.ptr + 4 * D}), 2 * D, lb.IN_F32, None, 0, THETA, EPS)
    k_out, v_out = ctx.alloc(7 * D * 4), ctx.alloc(7 * D * 4)
    ctx.kv4_read(case.desc, case.batch, k_out, v_out, lb.IN_F32)
    for out, rows in ((k_out, x[:, :D]), (v_out, x[:, D:])):
        want = kc.values(*kc.quantise(rows)).astype(np.float32)
        assert np.array_equal(out.download(np.float32).reshape(7, D), want, equal_nan=True)
        assert np.isnan(want).sum() == (128 if rows is not None and np.isnan(rows).any() else 64)
    for b in (d_x, k_out, v_out):
        b.free()
    case.free()


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("dim,heads", [(64, 5), (128, 1), (256, 4)])
def test_read_types(lb, ctx, kind, dim, heads):
    case = kc.Case(ctx, dim, heads, 3, 48, seqs=[2, 1], pos=[40, 0], new=[8, 3], spare=2)
    n = case.rows * heads * dim
    fill = np.full(n, 7, kc.TYPES[kind])
    outs = [ctx.to_device(fill) for _ in range(2)]
    ctx.kv4_read(case.desc, case.batch, *outs, kind)
    for part, out in enumerate(outs):
        got = out.download(kc.TYPES[kind]).reshape(case.rows, heads, dim)
        for row, seq, pos in case.places():
            for h in range(heads):
                low, scale, code = (x[pos] for x in kc.cache_rows(case.cache, dim, seq, h, pos + 1)[part])
                v = (low + scale * code).astype(np.float32)
                assert np.array_equal(got[row, h], kc.typed(v, kind)[0])
        assert (got[-2:] == 7).all()  # rows behind the last request's stay as they were
        out.free()
    case.free()


# ---- attention ----------------------------------------------------------------------------------------------------
def attention(lb, ctx, case, G, kind, norm=False, rot=0, gate=False, max_new=None, seed=6, gap=0, size=1.0, change=None, shift=0, gate_at=None, row_gap=0):
    """the call's result and its check against 64 bits; `change` may edit the queries (by reference)"""
    rng, D, H = np.random.default_rng(seed), case.dim, case.heads
    HQ, at = H * G, D if gate_at is None else gate_at
    width = (at + D if gate else D) + gap
    x = size * rng.standard_normal((case.rows, HQ * width + row_gap))
    if change:
        change(x)
    raw, x = kc.typed(x, kind)
    row_stride = x.shape[1]
    raw, x = np.concatenate([np.zeros(shift, raw.dtype), raw.ravel()]), x[:, :HQ * width].reshape(case.rows, HQ, width)
    w = lb.f32_to_bf16((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)) if norm else None
    d_x, d_w = ctx.to_device(raw), ctx.to_device(w) if norm else None
    where = lambda n: type("At", (), {"ptr": d_x.ptr + n * raw.itemsize})  # noqa: E731
    out = ctx.to_device(np.full(shift + case.rows * HQ * D, 9.0, np.float16))
    d_out = type("At", (), {"ptr": out.ptr + 2 * shift})
    ctx.kv4_attention(case.desc, case.batch, where(shift), where(shift + at) if gate else None, row_stride if row_gap else 0, width, kind, d_w, d_out, HQ, max_new or max(case.new), rot,
                      THETA, EPS)
    got = out.download(np.float16)[shift:].astype(np.float64).reshape(case.rows, HQ, D)
    assert ctx.device_status() == 0
    worst, rows = 0.0, {}
    for row, seq, pos in case.places():
        q = kc.norm_rotate(x[row, :, :D], pos, kc.bf16_values(w) if norm else None, rot, THETA, EPS)
        for h in range(HQ):
            if (seq, h // G) not in rows or rows[seq, h // G][0] <= pos:
                n = min(case.max_ctx, pos + max(case.new) + 1)
                rows[seq, h // G] = n, kc.cache_rows(case.cache, D, seq, h // G, n)
            want, tol = kc.attend(q[h], *rows[seq, h // G][1], pos)
            if gate:
                g = 1 / (1 + np.exp(-x[row, h, at:at + D]))
                want, tol = want * g, tol * g + np.abs(want * g) * 2.0 ** -20
            tol = tol + 2.0 ** -11 * (np.abs(want) + tol) + 2.0 ** -25  # the output's rounding
            err = np.abs(got[row, h] - want)
            assert (err <= tol).all(), (row, h, float((err / tol).max()))
            worst = max(worst, float((err / tol).max()))
    left = case.rows - int(case.starts[-1])
    if left:
        assert (got[-left:] == 9.0).all()
    d_x.free()
    out.free()
    return worst, got


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 127, 128, 129, 1000])
def test_attention_lengths(lb, ctx, dim, length):
    case = kc.Case(ctx, dim, 2, 1, 1024, seqs=[0], pos=[length - 1], new=[1])
    attention(lb, ctx, case, 3, lb.IN_F32)
    case.free()


@pytest.mark.parametrize("dim,heads,G,kind,norm,rot,gate", [(256, 4, 6, 1, True, 64, True), (128, 8, 4, 0, False, 128, False), (64, 1, 8, 2, True, 32, True), (256, 2, 1, 0, True, 256, True),
                                                           (128, 3, 16, 1, False, 0, False), (64, 4, 5, 1, False, 64, True)])
def test_attention_ragged(lb, ctx, dim, heads, G, kind, norm, rot, gate):
    """sequences of all lengths, one without tokens, in another order than their places"""
    case = kc.Case(ctx, dim, heads, 8, 2048, seqs=[5, 0, 7, 1, 2, 6], pos=[0, 2047, 300, 127, 128, 1111], new=[1, 1, 0, 1, 1, 1], spare=3)
    attention(lb, ctx, case, G, kind, norm, rot, gate)
    case.free()


@pytest.mark.parametrize("dim,heads,G,new", [(256, 4, 6, [5, 1, 3]), (256, 1, 6, [16, 2, 7]), (128, 2, 4, [4, 0, 8]), (64, 3, 16, [16, 1, 3]), (128, 1, 1, [16, 16, 1]), (64, 2, 5, [3, 4, 2])])
def test_attention_drafts(lb, ctx, dim, heads, G, new):
    """several new tokens see as many rows as their places allow; columns beyond one set of products"""
    case = kc.Case(ctx, dim, heads, 4, 528, seqs=[3, 1, 0], pos=[0, 500, 250], new=new)
    attention(lb, ctx, case, G, lb.IN_F32, norm=True, rot=64, gate=True)
    case.free()


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("shift,gap,row_gap,gate_at", [(0, 0, 0, 67), (1, 0, 0, 64), (0, 5, 3, 64), (0, 8, 16, 72), (3, 1, 1, 65), (8, 0, 0, 128)])
def test_attention_alignments(lb, ctx, kind, shift, gap, row_gap, gate_at):
    """queries, gates, rows and results at any place that their type allows, each for itself"""
    case = kc.Case(ctx, 64, 2, 2, 256, seqs=[1, 0], pos=[200, 30], new=[2, 1])
    attention(lb, ctx, case, 3, kind, True, 32, True, shift=shift, gap=gap, row_gap=row_gap, gate_at=gate_at)
    case.free()


def test_attention_most_columns(lb, ctx):
    """16 heads on one, 16 new tokens: 32 passes over the rows"""
    case = kc.Case(ctx, 128, 2, 2, 512, seqs=[1, 0], pos=[300, 0], new=[16, 3])
    attention(lb, ctx, case, 16, lb.IN_F16, rot=128)
    case.free()


def test_attention_more_tiles_than_ctas(lb, ctx):
    """items that begin, go on and end in every way in a CTA's share"""
    rng = np.random.default_rng(12)
    pos = rng.integers(0, 700, 40)
    case = kc.Case(ctx, 64, 8, 40, 704, seqs=rng.permutation(40), pos=pos, new=[1] * 40)
    attention(lb, ctx, case, 1, lb.IN_F32)
    case.free()


def test_attention_token_alone_or_together(lb, ctx):
    """a sequence's result does not depend on the batch that it travels with, beyond the order of its parts' sums"""
    case = kc.Case(ctx, 128, 4, 6, 4096, seqs=[0, 1, 2, 3, 4, 5], pos=[4000, 10, 700, 2000, 3000, 55], new=[1] * 6)
    _, got = attention(lb, ctx, case, 4, lb.IN_F32)
    one = lb.Kv4Batch(case.d[0].ptr, case.d[1].ptr, 0, 6, 6)
    case.batch = one
    _, again = attention(lb, ctx, case, 4, lb.IN_F32)
    assert np.array_equal(got, again)  # starts left out: one token each; and run to run the same
    case.free()


def test_attention_many_requests(lb, ctx):
    rng = np.random.default_rng(2)
    pos = rng.integers(0, 200, 256)
    case = kc.Case(ctx, 64, 2, 256, 208, seqs=rng.permutation(256), pos=pos, new=[1] * 256)
    attention(lb, ctx, case, 2, lb.IN_F16)
    case.free()


def test_attention_long(lb, ctx):
    """one sequence over every SM, scores with a wide spread"""
    case = kc.Case(ctx, 256, 2, 1, 60000, seqs=[0], pos=[59990], new=[4])
    attention(lb, ctx, case, 2, lb.IN_F32, norm=True, rot=64, size=2.0)
    case.free()


@pytest.mark.parametrize("size", [1e-30, 1e-4, 30.0, 1e4])
def test_attention_query_sizes(lb, ctx, size):
    """queries of any size keep their 11 bits: uniform weights at one end, one row at the other"""
    case = kc.Case(ctx, 64, 1, 1, 256, seqs=[0], pos=[200], new=[1])
    attention(lb, ctx, case, 4, lb.IN_F32, size=size)
    case.free()


def test_attention_value_scales(lb, ctx):
    """values whose scales grow and shrink by orders of magnitude along the cache, and groups of very different sizes"""
    case = kc.Case(ctx, 128, 2, 1, 2048, seqs=[0], pos=[2000], new=[2])
    raw = case.cache[0, :, :, 16 * 128:].copy().view(np.float16).reshape(2, 128, 2, 2, 16, 2)
    size = 10.0 ** np.interp(np.arange(2048), [0, 500, 1000, 1500, 2047], [-4, 3, -2, 2, -5]).reshape(128, 16)
    raw[:, :, 1] = (raw[:, :, 1] * size[None, :, None, :, None] * np.array([1.0, 1e-2])[None, None, :, None, None]).astype(np.float16)
    case.cache[0, :, :, 16 * 128:] = raw.reshape(2, 128, -1).view(np.uint8)
    case.d_cache.upload(case.cache)
    attention(lb, ctx, case, 3, lb.IN_F32)
    case.free()


def test_attention_rows_that_are_not_there(lb, ctx):
    """rows behind a sequence's last one may hold NaN; a NaN among the new rows reaches the tokens that see it and no other"""
    case = kc.Case(ctx, 64, 1, 2, 64, seqs=[0, 1], pos=[20, 33], new=[4, 3])
    pairs = case.cache[:, :, :, 16 * 64:].copy().view(np.uint16).reshape(2, 1, 4, 2, 1, 16, 2)
    for seq, end in ((0, 24), (1, 36)):
        for row in range(end, 64):
            pairs[seq, :, row // 16, :, :, row % 16] = 0x7fff
    case.cache[:, :, :, 16 * 64:] = pairs.reshape(2, 1, 4, -1).view(np.uint8)
    case.d_cache.upload(case.cache)
    _, clean = attention(lb, ctx, case, 2, lb.IN_F32)
    for part in range(2):  # a key, then a value of row 22 of sequence 0: its third new token's
        bad = case.cache.copy()
        p = bad[0, 0, 1, 16 * 64:].copy().view(np.uint16).reshape(2, 1, 16, 2)
        p[part, 0, 6] = 0x7fff
        bad[0, 0, 1, 16 * 64:] = p.reshape(-1).view(np.uint8)
        case.d_cache.upload(bad)
        rng = np.random.default_rng(6)
        d_x, out = ctx.to_device(rng.standard_normal((7, 2, 64)).astype(np.float32)), ctx.alloc(7 * 2 * 64 * 2)
        ctx.kv4_attention(case.desc, case.batch, d_x, None, 0, 0, lb.IN_F32, None, out, 2, 4, 0, THETA, EPS)
        got = out.download(np.float16).astype(np.float64).reshape(7, 2, 64)
        assert np.array_equal(got[[0, 1, 4, 5, 6]], clean[[0, 1, 4, 5, 6]])
        assert np.isnan(got[2:4]).all()
        d_x.free()
        out.free()
    case.free()


def test_attention_bad_queries_stay_alone(lb, ctx):
    case = kc.Case(ctx, 128, 1, 1, 256, seqs=[0], pos=[150], new=[3])
    _, clean = attention(lb, ctx, case, 4, lb.IN_F32)
    rng = np.random.default_rng(6)
    x = rng.standard_normal((3, 4, 128)).astype(np.float32)
    x[1, 2, 7], x[2, 0, 0] = np.nan, np.inf
    d_x, out = ctx.to_device(x), ctx.alloc(3 * 4 * 128 * 2)
    ctx.kv4_attention(case.desc, case.batch, d_x, None, 0, 0, lb.IN_F32, None, out, 4, 3, 0, THETA, EPS)
    got = out.download(np.float16).astype(np.float64).reshape(3, 4, 128)
    same = np.ones((3, 4), bool)
    same[1, 2] = same[2, 0] = False
    assert np.array_equal(got[same], clean[same])
    assert np.isnan(got[1, 2]).all() and not np.isfinite(got[2, 0]).any()
    case.free()


# ---- requests that are not there, refusals, graphs ---------------------------------------------------------------
@pytest.mark.parametrize("what,code", [("pos", 0x1005), ("negative", 0x1005), ("seq", 0x1006), ("rows", 0x1006), ("new", 0x1006)])
def test_bad_requests_are_left_out(lb, ctx, what, code):
    """the request is skipped whole and named by the status word; the others' results are there"""
    case = kc.Case(ctx, 64, 1, 3, 64, seqs=[0, 1, 2], pos=[20, 30, 40], new=[2, 3, 2])
    seqs, pos, starts, rows, max_new = [0, 1, 2], [20, 30, 40], [0, 2, 5, 7], 7, 3
    if what == "pos":
        pos[1] = 62
    elif what == "negative":
        pos[1] = -1
    elif what == "seq":
        seqs[1] = 3
    elif what == "rows":
        starts, rows = [0, 2, 4, 7], 6  # the last request ends behind the tensors
    else:
        max_new = 2
    for b, a in zip(case.d, (seqs, pos, starts)):
        b.upload(np.array(a, np.int32))
    case.batch.rows = rows
    x = np.random.default_rng(4).standard_normal((7, 1, 64)).astype(np.float32)
    d_x, out = ctx.to_device(x), ctx.to_device(np.full(7 * 64, 9.0, np.float16))
    ctx.kv4_attention(case.desc, case.batch, d_x, None, 0, 0, lb.IN_F32, None, out, 1, max_new, 0, THETA, EPS)
    with pytest.raises(lb.LithosError, match=f"0x{code:x}"):
        ctx.device_status()
    got = out.download(np.float16).reshape(7, 64)
    gone = slice(4, 7) if what == "rows" else slice(2, 5)
    assert (got[gone] == 9.0).all()
    there = [i for i in range(7) if not gone.start <= i < gone.stop]
    assert (got[there] != 9.0).any(1).all()
    if what != "new":
        ctx.kv4_append(case.desc, case.batch, d_x, d_x, 0, lb.IN_F32, None, 0, THETA, EPS)
        with pytest.raises(lb.LithosError, match=f"0x{code:x}"):
            ctx.device_status()
        changed = (case.download() != case.cache).any((1, 2, 3))
        assert list(changed) == [True, what == "rows", what != "rows"]
    assert ctx.device_status() == 0
    case.free()


def test_refusals(lb, ctx):
    b = ctx.alloc(1 << 16)
    cache, batch = (16 + b.ptr // 16 * 16, 1, 16, 1, 64), (0, b.ptr, 0, 1, 1)

    def bad(call, *a):
        with pytest.raises(lb.LithosError) as e:
            call(*a)
        assert e.value.status == lb.LB_ERR_INVALID

    def desc(i=None, v=None, of=cache, kind=lb.Kv4Cache):
        of = list(of)
        if i is not None:
            of[i] = v
        return kind(*of)
    good = desc(), desc(of=batch, kind=lb.Kv4Batch)
    at = lambda n: type("At", (), {"ptr": b.ptr + n})  # noqa: E731
    for i, v in ((0, 0), (0, b.ptr + 8), (1, 0), (2, 24), (2, 0), (3, 0), (3, 40), (4, 32), (4, 192)):
        for call, rest in ((ctx.kv4_append, (b, b)), (ctx.kv4_read, (b, b)), (ctx.kv4_attention, (b, None, 0, 0, 1, None, b, 1))):
            bad(call, desc(i, v), good[1], *rest)
    for i, v in ((1, 0), (1, b.ptr + 2), (3, 0), (3, 257), (4, 0), (4, 2), (4, (1 << 24) + 1)):
        for call, rest in ((ctx.kv4_append, (b, b)), (ctx.kv4_read, (b, b)), (ctx.kv4_attention, (b, None, 0, 0, 1, None, b, 1))):
            bad(call, good[0], desc(i, v, batch, lb.Kv4Batch), *rest)
    null = type("At", (), {"ptr": 0})
    for rest in ((null, b), (b, null), (at(2), b, 0, 1), (b, b, 63), (b, b, 0, 3), (b, b, 0, -1), (b, b, 0, 0, None, 4), (b, b, 0, 0, None, 72), (b, b, 0, 0, None, 8, -1.0),
                 (b, b, 0, 0, None, 8, 1e7, float("nan"))):
        bad(ctx.kv4_append, *good, *rest)
    for rest in ((null, b, 1), (b, at(2), 1), (b, b, 3)):
        bad(ctx.kv4_read, *good, *rest)
    for rest in ((null, None, 0, 0, 1, None, b, 1), (b, None, 0, 0, 1, None, null, 1), (b, None, 0, 0, 1, None, b, 0), (b, None, 0, 0, 1, None, b, 17), (b, None, 0, 0, 1, None, b, 1, 0),
                 (b, None, 0, 0, 1, None, b, 1, 17), (b, None, 0, 60, 1, None, b, 1), (b, None, -8, 0, 1, None, b, 1), (b, at(2), 0, 0, 1, None, b, 1), (b, None, 0, 0, 1, None, at(1), 1)):
        bad(ctx.kv4_attention, *good, *rest)
    # 256 requests that all read the longest cache with every column there is: 256 * 32 * 32 items of 2 * 8192 + 3 places pass 2^32
    most = lb.Kv4Cache(cache[0], 1, 1 << 20, 32, 256), lb.Kv4Batch(b.ptr, b.ptr, b.ptr, 256, 256)
    bad(ctx.kv4_attention, *most, b, None, 0, 0, 1, None, b, 512, 16)
    b.free()


def test_captured_graph_takes_new_positions(lb, ctx):
    """append and attention captured once, replayed as the sequences grow: the same as the calls one by one"""
    D, H, G, n = 128, 2, 4, 3
    case = kc.Case(ctx, D, H, n, 256, seqs=[2, 0, 1], pos=[0, 100, 127], new=[1, 1, 1])
    rng = np.random.default_rng(8)
    kv, q = (rng.standard_normal((4, n, w)).astype(np.float32) for w in (2 * H * D, H * G * D))
    d_kv, d_q, out = ctx.to_device(kv[0]), ctx.to_device(q[0]), ctx.alloc(n * H * G * D * 2)
    v = type("At", (), {"ptr": d_kv.ptr + 4 * H * D})

    def step():
        ctx.kv4_append(case.desc, case.batch, d_kv, v, 2 * H * D, lb.IN_F32, None, 64, THETA, EPS)
        ctx.kv4_attention(case.desc, case.batch, d_q, None, 0, 0, lb.IN_F32, None, out, H * G, 1, 64, THETA, EPS)

    def play(run):
        case.d_cache.upload(case.cache)
        outs = []
        for i in range(4):
            d_kv.upload(kv[i]), d_q.upload(q[i])
            case.d[1].upload(np.array([p + i for p in case.pos], np.int32))
            run()
            outs.append(out.download(np.float16).copy())
        return np.stack(outs), case.download()
    eager = play(step)
    ctx.begin_capture()
    step()
    graph = ctx.end_capture()
    assert graph.kernels == 3
    replayed = play(graph.launch)
    assert np.array_equal(eager[0], replayed[0]) and np.array_equal(eager[1], replayed[1])
    graph.destroy()
    case.free()


@pytest.mark.parametrize("dim,new", [(64, 1), (128, 5), (256, 1), (256, 5)])
@pytest.mark.parametrize("way", ["up", "down", "mixed"])
def test_attention_scales_by_block(lb, ctx, dim, new, way):
    """every block of 16 rows and every group has its own order of magnitude: the scales that warps take theirs against differ, and move at different tiles"""
    S, blocks = dim // 64, 128
    case = kc.Case(ctx, dim, 2, 1, 16 * blocks, seqs=[0], pos=[16 * blocks - 20], new=[new])
    raw = case.cache[0, :, :, 16 * dim:].copy().view(np.float16).reshape(2, blocks, 2, S, 16, 2)
    rng = np.random.default_rng(21)
    power = {"up": np.linspace(-4, 3, blocks)[:, None] + np.zeros(S), "down": np.linspace(3, -4, blocks)[:, None] + np.zeros(S), "mixed": rng.uniform(-4, 3, (blocks, S))}[way]
    raw[:, :, 1] = (raw[:, :, 1] * (10.0 ** power)[None, :, :, None, None]).astype(np.float16)
    case.cache[0, :, :, 16 * dim:] = raw.reshape(2, blocks, -1).view(np.uint8)
    case.d_cache.upload(case.cache)
    attention(lb, ctx, case, 3, lb.IN_F32)
    case.free()


def test_attention_requests_of_one_sequence(lb, ctx):
    """several requests may read the same sequence, each up to its own place"""
    case = kc.Case(ctx, 128, 2, 2, 1024, seqs=[1, 1, 0, 1], pos=[900, 3, 500, 900], new=[2, 1, 1, 2])
    attention(lb, ctx, case, 4, lb.IN_F32)
    case.free()


def test_two_graphs_in_turn(lb, ctx):
    """graphs of different shapes share the context's workspace: replayed in turn and twice in a row, the same as the calls"""
    rng = np.random.default_rng(4)
    cases = [kc.Case(ctx, 256, 2, 3, 2048, seqs=[2, 0, 1], pos=[2000, 5, 700], new=[2, 1, 3]), kc.Case(ctx, 64, 4, 2, 4096, seqs=[1, 0], pos=[4000, 100], new=[1, 1])]
    steps, graphs, outs, want = [], [], [], []
    for case, G in zip(cases, (3, 2)):
        d_q = ctx.to_device(rng.standard_normal((case.rows, case.heads * G * case.dim)).astype(np.float32))
        out = ctx.alloc(case.rows * case.heads * G * case.dim * 2)
        steps.append((case, d_q, out, case.heads * G))
        outs.append(out)

    def run(case, d_q, out, heads):
        ctx.kv4_attention(case.desc, case.batch, d_q, None, 0, 0, lb.IN_F32, None, out, heads, max(case.new), 64, THETA, EPS)
    for step in steps:
        run(*step)
        want.append(step[2].download(np.float16).copy())
        ctx.begin_capture()
        run(*step)
        graphs.append(ctx.end_capture())
    for order in ((0, 1, 0, 1), (1, 1, 0, 0)):
        for out in outs:
            out.upload(np.zeros(out.nbytes // 2, np.float16))
        for g in order:
            graphs[g].launch()
        for out, w in zip(outs, want):
            assert np.array_equal(out.download(np.float16), w)
    for g in graphs:
        g.destroy()
    for case, d_q, out, _ in steps:
        d_q.free(), out.free(), case.free()
