"""The 4-bit KV cache and what is computed from it, in 64 bits with numpy: the layout as include/lithos_b200.h gives it, rows in, attention, and bounds on what the
kernels' roundings may do to a result."""
import numpy as np

import lithos_b200 as lb

TYPES = {lb.IN_BF16: np.uint16, lb.IN_F32: np.float32, lb.IN_F16: np.float16}


def typed(x, kind):
    """x as the kernels take it, and the 64-bit values it then has"""
    if kind == lb.IN_BF16:
        b = lb.f32_to_bf16(np.asarray(x, np.float32))
        return b, lb.bf16_to_f32(b).astype(np.float64)
    t = np.asarray(x).astype(TYPES[kind])
    return t, t.astype(np.float64)


def bf16_values(x):
    return lb.bf16_to_f32(x).astype(np.float64)


def block_bytes(dim):
    return 18 * dim


def key_byte(dim, row, feature):
    """place of a key's code inside its block of 16 rows"""
    half, place, S = row // 2 % 2, 2 * (row // 4) + row % 2, dim // 64
    return ((half * S + feature // 64) * 8 + place) * 32 + feature % 64 // 2


def value_byte(dim, row, feature):
    return 8 * dim + ((feature // 64 * 8 + feature % 64 // 8) * 16 + row) * 4 + feature % 8 // 2


def pair_byte(dim, part, row, group):
    return (16 + part) * dim + (group * 16 + row) * 4


def quantise(x):
    """rows [.., dim] -> codes, scale, lowest: groups of 64 features"""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 64)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    lowest = np.clip(g.min(-1), -65504, 65504).astype(np.float32).astype(np.float16).astype(np.float64)
    scale = np.maximum((np.clip(g.max(-1), -65504, 65504) - lowest) / 15, 0).astype(np.float32).astype(np.float16).astype(np.float64)
    code = np.where(scale[..., None] > 0, (g - lowest[..., None]) / np.where(scale > 0, scale, 1)[..., None], 0)
    code = np.clip(np.rint(code), 0, 15)
    nan = np.where(bad, np.nan, 0.0)
    return code.astype(np.int64), scale + nan, lowest + nan


def values(code, scale, lowest):
    return (lowest[..., None] + scale[..., None] * code).reshape(*code.shape[:-2], -1)


def cache_rows(cache, dim, seq, head, count):
    """keys and values of rows 0..count-1 from the cache's bytes [seqs, heads, blocks, 18 dim]"""
    row, f = np.arange(count)[:, None], np.arange(dim)[None]
    raw, out = cache[seq, head], []
    for part, place in ((0, key_byte), (1, value_byte)):
        byte = raw[row // 16, place(dim, row % 16, f)].astype(np.int64)
        at = pair_byte(dim, part, row % 16, f // 64)
        half = lambda o: (raw[row // 16, at + o].astype(np.uint16) | raw[row // 16, at + o + 1].astype(np.uint16) << 8).view(np.float16).astype(np.float64)  # noqa: B023,E731
        out.append((half(2), half(0), (byte >> (4 * (f % 2))) & 15))
    return out  # (lowest, scale, code) of keys, of values


def norm_rotate(x, pos, weight, rot, theta, eps):
    """x [heads, dim] of position pos"""
    x = np.array(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * weight
    half = rot // 2
    if half:
        a = pos * np.exp2(-np.log2(np.float64(np.float32(theta))) * np.arange(half) / half)
        u, v = x[:, 0:rot:2].copy(), x[:, 1:rot:2].copy()
        x[:, 0:rot:2], x[:, 1:rot:2] = u * np.cos(a) - v * np.sin(a), u * np.sin(a) + v * np.cos(a)
    return x


def attend(q, key, value, limit):
    """One query q [dim] (normalised, rotated) over rows 0..limit: the result, and how far the kernel's may be from it before the output's rounding.
    q goes in with 11 bits, so a score is off by at most d_t = 2^-11 sum |q| |k_t| / sqrt(dim), and a probability's weight by a factor of exp(d_t + max d): the weights add up
    to one, so that moves the result by sum p_t (exp(..) - 1) |v_t - out|.  p_t scale_t is rounded to 11 bits, 2^-11 of its code's part.  2^-18 of everything is for the
    32-bit arithmetic: sums of 128 rows at a time, exponentials to 2^-22 of arguments up to 2^4, a sine's 2^-22."""
    dim = q.shape[0]
    (kl, ks, kc), (vl, vs, vc) = ([x[:limit + 1] for x in p] for p in (key, value))
    k, v = kl + ks * kc, vl + vs * vc
    s = k @ q / np.sqrt(dim)
    p = np.exp(s - s.max())
    p /= p.sum()
    out = p @ v
    d = (2.0 ** -11 + 2.0 ** -18) * ((np.abs(kl) + ks * kc) @ np.abs(q)) / np.sqrt(dim)
    tol = (p * np.expm1(d + d.max())) @ np.abs(v - out) + 2.0 ** -11 * (p @ (vs * vc)) + 2.0 ** -18 * (p @ (np.abs(vl) + vs * vc))
    return out, tol


class Case:
    """a cache and a batch on the device, and the same on the host"""

    def __init__(self, ctx, dim, heads, n_seqs, max_ctx, seqs, pos, new, seed=1, starts=True, spare=0):
        self.ctx, self.dim, self.heads, self.max_ctx = ctx, dim, heads, max_ctx
        self.seqs, self.pos, self.new = list(seqs), list(pos), list(new)
        rng = self.rng = np.random.default_rng(seed)
        shape = (n_seqs, heads, max_ctx // 16)
        self.cache = rng.integers(0, 256, (*shape, block_bytes(dim)), dtype=np.uint8)
        S = dim // 64
        pairs = np.stack([0.2 + 0.2 * rng.random((*shape, 2, S, 16)), -2.0 + 0.5 * rng.standard_normal((*shape, 2, S, 16))], -1).astype(np.float16)
        self.cache[..., 16 * dim:] = np.ascontiguousarray(pairs).view(np.uint8).reshape(*shape, -1)
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + spare
        self.d_cache = ctx.to_device(self.cache)
        self.d = [ctx.to_device(np.asarray(a, np.int32)) for a in (seqs, pos, self.starts)]
        self.desc = lb.Kv4Cache(self.d_cache.ptr, n_seqs, max_ctx, heads, dim)
        self.batch = lb.Kv4Batch(self.d[0].ptr, self.d[1].ptr, self.d[2].ptr if starts else 0, len(seqs), self.rows)

    def places(self):
        for r, (s, p, n) in enumerate(zip(self.seqs, self.pos, self.new)):
            for i in range(n):
                yield int(self.starts[r]) + i, s, p + i

    def download(self):
        return self.d_cache.download(np.uint8).reshape(self.cache.shape)

    def free(self):
        for b in [self.d_cache, *self.d]:
            b.free()
