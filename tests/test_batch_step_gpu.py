"""A decode step of several sequences as a host's own loop makes it: int4 projections, rows into the 4-bit cache, attention, the target's logits, drafts verified.  Every stage is checked
against 64 bits on what the stage before left on the device, and the captured step against the calls."""
import numpy as np
import pytest

import kv4_cases as kc
import verify_cases as vc
from helpers import gptq_case, rel_err_max

pytestmark = pytest.mark.gpu
THETA, EPS = 1e7, 1e-6


def dense(w):
    q, s, z, _ = w
    K, N = 8 * q.shape[0], q.shape[1]
    codes = ((q[:, None, :] >> (4 * np.arange(8, dtype=np.uint32))[None, :, None]) & 15).reshape(K, N).astype(np.float64)
    zero = ((z[:, :, None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(K // 128, N).astype(np.float64)
    return ((codes.reshape(K // 128, 128, N) - zero[:, None]) * s.astype(np.float64)[:, None]).reshape(K, N)


class Step:
    D, HQ, HKV, W, V, R = 64, 4, 2, 512, 1024, 3

    def __init__(self, lb, ctx, drafts):
        self.lb, self.ctx = lb, ctx
        D, HQ, HKV, W, V = self.D, self.HQ, self.HKV, self.W, self.V
        self.N = 2 * HQ * D + 2 * HKV * D  # every head's query and gate, keys, values
        self.w = {n: gptq_case(K, N, seed) for n, K, N, seed in (("in", W, self.N, 1), ("out", HQ * D, W, 2), ("head", W, V, 3))}
        self.dw = {n: [ctx.to_device(a) for a in w[:3]] for n, w in self.w.items()}
        self.new = [d + 1 for d in drafts]
        self.rows, self.starts = sum(self.new), np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.ctx_rows = 64
        self.cache = ctx.to_device(np.zeros(lb.kv4_bytes(self.R, self.ctx_rows, HKV, D), np.uint8))
        self.norm = {n: lb.f32_to_bf16((1 + 0.05 * np.random.default_rng(i).standard_normal(D)).astype(np.float32)) for i, n in enumerate("qk")}
        self.dn = {n: ctx.to_device(a) for n, a in self.norm.items()}
        rng = self.rng = np.random.default_rng(7)
        self.x, self.y, self.o, self.h, self.logits = (ctx.alloc(n) for n in (self.rows * W * 2, self.rows * self.N * 4, self.rows * HQ * D * 2, self.rows * W * 2, self.rows * V * 4))
        self.drafts, self.ua, self.up = (rng.integers(0, V, self.rows).astype(np.int32), rng.random(self.rows).astype(np.float32), rng.random(self.R).astype(np.float32))
        self.small = {n: ctx.to_device(a) for n, a in (("starts", self.starts), ("pos", np.zeros(self.R, np.int32)), ("drafts", self.drafts), ("ua", self.ua), ("up", self.up))}
        self.tokens, self.accepted, self.p = ctx.alloc(4 * self.rows), ctx.alloc(4 * self.R), ctx.alloc(4 * self.rows)
        self.desc = lb.Kv4Cache(self.cache.ptr, self.R, self.ctx_rows, HKV, D)
        self.batch = lb.Kv4Batch(0, self.small["pos"].ptr, self.small["starts"].ptr, self.R, self.rows)

    def at(self, column):
        return type("At", (), {"ptr": self.y.ptr + 4 * column})

    def launch(self):
        lb, c, D, HQ, HKV, rows = self.lb, self.ctx, self.D, self.HQ, self.HKV, self.rows
        c.gemm_int4(*self.dw["in"], self.x, self.y, self.W, self.N, rows, lb.GEMV_Y_F32)
        keys = 2 * HQ * D
        c.kv4_append(self.desc, self.batch, self.at(keys), self.at(keys + HKV * D), self.N, lb.IN_F32, self.dn["k"], 32, THETA, EPS)
        c.kv4_attention(self.desc, self.batch, self.at(0), self.at(D), self.N, 2 * D, lb.IN_F32, self.dn["q"], self.o, HQ, max(self.new), 32, THETA, EPS)
        c.gemm_int4(*self.dw["out"], self.o, self.h, HQ * D, self.W, rows)
        c.gemm_int4(*self.dw["head"], self.h, self.logits, self.W, self.V, rows, lb.GEMV_Y_F32)
        s = self.small
        c.verify_drafts(self.logits, self.V, s["starts"], self.R, rows, s["drafts"], None, s["ua"], s["up"], self.tokens, self.accepted, 1.0, 20, self.p)

    def feed(self, step):
        self.x.upload(np.random.default_rng(100 + step).standard_normal((self.rows, self.W)).astype(np.float16))
        self.small["pos"].upload(np.array([3 * step, 10 + step, 2 * step], np.int32))

    def results(self):
        return [b.download(t) for b, t in ((self.y, np.float32), (self.o, np.float16), (self.logits, np.float32), (self.tokens, np.int32), (self.accepted, np.int32), (self.cache, np.uint8))]


@pytest.mark.parametrize("drafts", [[2, 0, 3], [0, 0, 0]])
def test_step(lb, ctx, drafts):
    s = Step(lb, ctx, drafts)
    D, HQ, HKV, rows = s.D, s.HQ, s.HKV, s.rows
    w = {n: dense(a) for n, a in s.w.items()}
    steps = []
    for step in range(3):
        s.feed(step)
        s.launch()
        steps.append(s.results())
        y, o, logits, tokens, accepted, cache = steps[-1]
        x = s.x.download(np.float16).reshape(rows, s.W).astype(np.float64)
        assert rel_err_max(y.reshape(rows, s.N), x @ w["in"]) < 1e-5
        y, cache = y.reshape(rows, s.N).astype(np.float64), cache.reshape(s.R, HKV, s.ctx_rows // 16, -1)
        qg = y[:, :2 * HQ * D].reshape(rows, HQ, 2, D)
        for r, (p, n) in enumerate(zip(s.small["pos"].download(np.int32), s.new)):
            stored = [kc.cache_rows(cache, D, r, h, int(p) + n) for h in range(HKV)]
            for i in range(n):
                row, pos = int(s.starts[r]) + i, int(p) + i
                k, v = y[row, 2 * HQ * D:].reshape(2, HKV, D)
                k = kc.norm_rotate(k, pos, kc.bf16_values(s.norm["k"]), 32, THETA, EPS)
                for h in range(HKV):
                    for part, want in ((0, k[h]), (1, v[h])):
                        low, scale, code = (a[pos] for a in stored[h][part])
                        assert np.array_equal(low + scale * code, kc.values(*kc.quantise(want[None]))[0])
                q = kc.norm_rotate(qg[row, :, 0], pos, kc.bf16_values(s.norm["q"]), 32, THETA, EPS)
                for h in range(HQ):
                    want, tol = kc.attend(q[h], *stored[h * HKV // HQ], pos)
                    g = 1 / (1 + np.exp(-qg[row, h, 1]))
                    want, tol = want * g, tol * g + np.abs(want) * 2.0 ** -20
                    assert (np.abs(o.reshape(rows, HQ, D)[row, h] - want) <= tol + 2.0 ** -11 * (np.abs(want) + tol) + 2.0 ** -25).all()
        h = s.h.download(np.float16).reshape(rows, s.W).astype(np.float64)
        assert rel_err_max(h, o.reshape(rows, -1).astype(np.float64) @ w["out"]) < 2.0 ** -10
        assert rel_err_max(logits.reshape(rows, s.V), h @ w["head"]) < 1e-5
        want = vc.verify(logits.reshape(rows, s.V), s.starts, s.drafts, None, s.ua, s.up, 1.0, 20, rows)
        assert np.array_equal(tokens, want[0]) and np.array_equal(accepted, want[1])
    s.cache.zero()
    ctx.begin_capture()
    s.launch()
    graph = ctx.end_capture()
    for step in range(3):
        s.feed(step)
        graph.launch()
        for a, b in zip(s.results(), steps[step]):
            assert np.array_equal(a, b)
    graph.destroy()
