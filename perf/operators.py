"""Decoding several sequences at a time from a 4-bit cache, with drafted tokens, as cases that can be timed and compared.

Kinds of work, each one call of a host that keeps its own decode loop (its projections are lb_gemm_int4's):

* "append"     new key and value rows of a batch of sequences: per-head norm and rotation of the keys, groups of 64 features rounded to
               4 bits, stored in the cache; the rows are read back as the values that the cache stands for;
* "attention"  grouped-query attention of a batch's new tokens (one per sequence, or a few drafted ones) over the 4-bit cache;
* "verify"     drafted tokens held against the target's probabilities with given uniform numbers: how many stand, the token that follows, and
               the target's probability of every draft.

The cache is blocks of 16 rows of one sequence and KV head, 18 D bytes each, groups of 64 features (S = D / 64 of them) apart:
  keys     [2][S][8 rows][32 bytes]    row 4 (g / 2) + 2 i + g % 2 of the block lies at half i, place g; a byte holds two neighbouring features, the lower one in its low half
  values   [S][8][16 rows][4 bytes]    eight neighbouring features of a row to four bytes
  (scale, lowest value) of the keys, then of the values, fp16: [S][16 rows][2]; a code c of 0..15 stands for lowest + scale * c
"""
import math
import random

import torch

own = False
THETA, EPS = 1e7, 1e-6
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
CODE = {"bf16": 0, "f32": 1, "f16": 2}


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    wide = {"HQ": 24, "HKV": 4, "D": 256, "rot": 64, "norm": True, "gate": True}  # the 27B model's attention
    return [
        # one sequence, one token: the smallest call, latency counts
        {"name": "attention_1x4096", "kind": "attention", "seqs": 1, "new": 1, "lo": 4096, "hi": 4096, "type": "f32", **wide},
        # a batch of conversations of all lengths, one token each
        {"name": "attention_32x_ragged", "kind": "attention", "seqs": 32, "new": 1, "lo": 40, "hi": 16000, "type": "f32", **wide},
        # drafted tokens of a batch: ragged numbers of them, up to five a sequence
        {"name": "attention_16x5_drafts", "kind": "attention", "seqs": 16, "new": 5, "lo": 500, "hi": 9001, "type": "f16", **wide},
        # one very long document
        {"name": "attention_1x100001", "kind": "attention", "seqs": 1, "new": 1, "lo": 100001, "hi": 100001, "type": "f32", **wide},
        # many short sequences with heads of 128, neither norm nor gate
        {"name": "attention_64x_d128", "kind": "attention", "seqs": 64, "new": 1, "lo": 17, "hi": 3001, "type": "bf16", "HQ": 32, "HKV": 8, "D": 128, "rot": 128,
         "norm": False, "gate": False},
        # a decode step's rows of a batch; a long prompt's rows
        {"name": "append_32x1", "kind": "append", "seqs": 32, "new": 1, "lo": 40, "hi": 16000, "type": "f32", **wide},
        {"name": "append_prompt_4001", "kind": "append", "seqs": 1, "new": 4001, "lo": 0, "hi": 0, "type": "f32", **wide},
        # one sequence whose drafts were the draft's first choices; whole vocabulary
        {"name": "verify_1x4", "kind": "verify", "seqs": 1, "new": 4, "vocab": 248320, "probs": False, "temperature": 1.0, "top_k": 0},
        # a batch with the draft's probabilities, whole vocabulary
        {"name": "verify_48x5", "kind": "verify", "seqs": 48, "new": 5, "vocab": 248320, "probs": True, "temperature": 0.8, "top_k": 0},
        # the same question to the model's top-k sampling, and to greedy decoding
        {"name": "verify_16x4_top50", "kind": "verify", "seqs": 16, "new": 4, "vocab": 248320, "probs": True, "temperature": 0.7, "top_k": 50},
        {"name": "verify_32x3_greedy", "kind": "verify", "seqs": 32, "new": 3, "vocab": 32768, "probs": False, "temperature": 0.0, "top_k": 0},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "verify", "verify"])
    if kind == "verify":
        seqs, greedy = _log(rng, 1, 48), rng.random() < 0.2
        return {"kind": kind, "seqs": seqs, "new": rng.randint(1, 5), "vocab": _log(rng, 1000, 248320), "probs": rng.random() < 0.6,
                "temperature": 0.0 if greedy else round(rng.uniform(0.3, 1.3), 2), "top_k": 0 if greedy or rng.random() < 0.5 else rng.randint(1, 64)}
    D = rng.choice([64, 128, 256, 256])
    HKV = rng.choice([1, 2, 4, 8])
    c = {"kind": kind, "D": D, "HKV": HKV, "HQ": HKV * rng.choice([1, 2, 3, 4, 6, 8]), "rot": rng.choice([0, 32, 64]), "norm": rng.random() < 0.6,
         "gate": rng.random() < 0.5, "type": rng.choice(["bf16", "f32", "f16"])}
    if kind == "append" and rng.random() < 0.5:  # prompts
        seqs = rng.randint(1, 4)
        return {**c, "seqs": seqs, "new": _log(rng, 20, 4000 // seqs), "lo": 0, "hi": rng.choice([0, 1000])}
    seqs = _log(rng, 1, 48)
    hi = _log(rng, 20, min(100000, 256_000_000 // (seqs * HKV * D)))
    return {**c, "seqs": seqs, "new": rng.choice([1, 1, rng.randint(2, 8)]), "lo": rng.randint(0, hi // 2), "hi": hi}


def lengths(case):
    """(rows of every sequence before the call, new tokens of every sequence): the longest one has case["hi"] rows; drafted tokens are ragged"""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    lo, hi, n = case.get("lo", 0), case.get("hi", 0), case["seqs"]
    pos = [hi] + [_log(rng, lo + 1, hi + 1) - 1 for _ in range(n - 1)]
    new = [case["new"]] + [rng.randint(1, case["new"]) for _ in range(n - 1)]
    return pos, new


# ---- inputs ------------------------------------------------------------------------------------------------------
def _starts(new):
    return torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def _cache(case, g, n, ctx):
    """rows like those of normal keys and values: codes around the middle, scales a few tenths"""
    D, S = case["D"], case["D"] // 64
    shape = (n, case["HKV"], ctx // 16)
    code = lambda: torch.randn((*shape, 16 * D), generator=g, device="cuda", dtype=torch.float16).mul_(2.7).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)  # noqa: E731
    out = torch.empty((*shape, 18 * D), dtype=torch.uint8, device="cuda")
    for part in range(2):
        c = code()
        out[..., part * 8 * D:(part + 1) * 8 * D] = c[..., 0::2] | (c[..., 1::2] << 4)
        del c
        scale = 0.28 + 0.1 * torch.rand((*shape, S * 16), generator=g, device="cuda")
        low = -7.5 * scale + 0.2 * torch.randn((*shape, S * 16), generator=g, device="cuda")
        out[..., (16 + part) * D:(17 + part) * D] = torch.stack([scale, low], -1).to(torch.float16).reshape(*shape, -1).view(torch.uint8)
    return out


class Buffer:
    """device memory of a tensor, as the library's calls take it"""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


_kept = {}


def context():
    if "ctx" not in _kept:
        import lithos_b200 as lb

        torch.cuda.init()
        _kept["ctx"] = lb.Context(0)
    return _kept["ctx"]


def inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    pos, new = lengths(case)
    n = case["seqs"]
    if case["kind"] == "verify":
        V, T = case["vocab"], case["temperature"] or 1.0
        rows = sum(new) + n  # every sequence's drafts, and the token behind them
        logits = 2.0 * rnd(rows, V) + 6.0 * (torch.rand((rows, V), generator=g, device="cuda") > 1 - 20 / V)
        guess = logits + 0.5 * rnd(rows, V)
        t = {"logits": logits, "starts": _starts([k + 1 for k in new]), "u_accept": torch.rand(rows, generator=g, device="cuda"), "u_pick": torch.rand(n, generator=g, device="cuda")}
        if case["probs"]:
            t["probs"] = torch.softmax(guess / T, 1)
            t["drafts"] = torch.multinomial(t["probs"], 1, generator=g)[:, 0].to(torch.int32)
        else:
            t["drafts"] = guess.argmax(1).to(torch.int32)
        t["tokens"], t["accepted"] = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (rows, n))
        t["p"] = torch.empty(rows, device="cuda")
        return t
    D, HQ, HKV, dt, rows = case["D"], case["HQ"], case["HKV"], TYPES[case["type"]], sum(new)
    ctx = -(-(max(pos) + case["new"]) // 16) * 16
    t = {"pos": torch.tensor(pos, dtype=torch.int32).cuda(), "starts": _starts(new), "seqs": torch.randperm(n, generator=g, device="cuda").to(torch.int32)}
    if case["kind"] == "append":  # key and value rows lie side by side in a projection's result
        t["cache"] = torch.zeros((n, HKV, ctx // 16, 18 * D), dtype=torch.uint8, device="cuda")
        t["kv"] = (rnd(rows, 2 * HKV * D) * torch.exp(0.5 * rnd(2 * HKV * D))).to(dt)
        t["k_out"], t["v_out"] = (torch.empty((rows, HKV, D), device="cuda") for _ in range(2))
    else:  # every head's query lies beside its gate
        t["cache"] = _cache(case, g, n, ctx)
        t["q"] = rnd(rows, HQ, (1 + case["gate"]) * D).to(dt)
        t["out"] = torch.empty((rows, HQ * D), dtype=torch.float16, device="cuda")
    if case["norm"]:
        t["norm"] = (1 + 0.02 * rnd(D)).to(torch.bfloat16)
    return t


def prepare(case, seed):
    t = inputs(case, seed)
    state = {"case": case, "t": t}
    state["b"] = {k: Buffer(x) for k, x in t.items()}
    if "kv" in t:
        half = t["kv"].shape[1] // 2
        state["b"]["k"], state["b"]["v"] = Buffer(t["kv"][:, :half]), Buffer(t["kv"][:, half:])
    if case.get("gate") and "q" in t:
        state["b"]["gate"] = Buffer(t["q"][:, :, case["D"]:])
    torch.cuda.synchronize()  # the library's calls go to a stream of its own, which waits for no other
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return run_own(state)
    return {"append": plain_append, "attention": plain_attention, "verify": plain_verify}[state["case"]["kind"]](state)


def run_own(state):
    import lithos_b200 as lb

    c, b, ctx = state["case"], state["b"], context()
    if c["kind"] == "verify":
        rows, n = len(state["t"]["drafts"]), c["seqs"]
        ctx.verify_drafts(b["logits"], c["vocab"], b["starts"], n, rows, b["drafts"], b.get("probs"), b["u_accept"], b["u_pick"], b["tokens"], b["accepted"],
                          c["temperature"], c["top_k"], b["p"])
        return {"tokens": b["tokens"].t, "accepted": b["accepted"].t, "p": b["p"].t}
    cache = lb.Kv4Cache(b["cache"].ptr, c["seqs"], state["t"]["cache"].shape[2] * 16, c["HKV"], c["D"])
    if c["kind"] == "append":
        rows = len(state["t"]["kv"])
        batch = lb.Kv4Batch(b["seqs"].ptr, b["pos"].ptr, b["starts"].ptr, c["seqs"], rows)
        ctx.kv4_append(cache, batch, b["k"], b["v"], 2 * c["HKV"] * c["D"], CODE[c["type"]], b.get("norm"), c["rot"], THETA, EPS)
        ctx.kv4_read(cache, batch, b["k_out"], b["v_out"], CODE["f32"])
        return {"keys": b["k_out"].t, "values": b["v_out"].t}
    rows, width = len(state["t"]["q"]), (1 + c["gate"]) * c["D"]
    batch = lb.Kv4Batch(b["seqs"].ptr, b["pos"].ptr, b["starts"].ptr, c["seqs"], rows)
    ctx.kv4_attention(cache, batch, b["q"], b.get("gate"), c["HQ"] * width, width, CODE[c["type"]], b.get("norm"), b["out"], c["HQ"], c["new"], c["rot"], THETA, EPS)
    return b["out"].t


def places(t, rows):
    """the request and the position of every row of a batch"""
    row = torch.arange(rows, device="cuda")
    req = torch.searchsorted(t["starts"][1:].long(), row, right=True)
    return req, t["pos"].long()[req] + row - t["starts"].long()[req]


def norm_rotate(x, at, case, weight):
    """x [rows, heads, D] at positions `at`: rms norm per head, then neighbouring pairs of the first features turn; angles in 64 bits"""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)
    if case["rot"]:
        half = case["rot"] // 2
        angle = at.double()[:, None] * THETA ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
        c, s = angle.cos().to(x.dtype)[:, None], angle.sin().to(x.dtype)[:, None]
        u, v = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        x = torch.cat([torch.stack([u * c - v * s, u * s + v * c], -1).flatten(-2), x[..., 2 * half:]], -1)
    return x


def plain_append(state):
    """in 64 bits: a value next to a border between two codes has to fall on the same side"""
    c, t = state["case"], state["t"]
    D, HKV, rows = c["D"], c["HKV"], len(t["kv"])
    k, v = t["kv"].double().view(rows, 2, HKV, D).unbind(1)
    k = norm_rotate(k, places(t, rows)[1], c, t.get("norm"))
    x = torch.stack([k, v]).view(2, rows, HKV, D // 64, 64)
    low = x.amin(-1, keepdim=True).clamp(-65504, 65504).float().half().double()
    scale = ((x.amax(-1, keepdim=True).clamp(-65504, 65504) - low) / 15).clamp(min=0).float().half().double()
    code = torch.where(scale > 0, (x - low) / scale, 0).round().clamp(0, 15)
    k, v = (low + scale * code).float().view(2, rows, HKV, D)
    return {"keys": k, "values": v}


def unpack(blocks, D):
    """blocks [..., 18 D] -> keys and values [..., 16, D] in 32 bits"""
    S, lead = D // 64, blocks.shape[:-1]
    bits = lambda x: torch.stack([x & 15, x >> 4], -1)  # noqa: E731
    k = bits(blocks[..., :8 * D]).view(-1, 2, S, 4, 2, 64).permute(0, 3, 1, 4, 2, 5).reshape(*lead, 16, S, 64)
    v = bits(blocks[..., 8 * D:16 * D]).view(-1, S, 8, 16, 8).permute(0, 3, 1, 2, 4).reshape(*lead, 16, S, 64)
    scales = blocks[..., 16 * D:].contiguous().view(torch.float16).view(*lead, 2, S, 16, 2).transpose(-3, -2).float()
    both = [sc[..., 1:] + sc[..., :1] * x.float() for sc, x in zip(scales.unbind(-4), (k, v))]
    return [x.reshape(*lead, 16, D) for x in both]


def plain_attention(state):
    c, t = state["case"], state["t"]
    D, HQ, HKV, n, m, rows = c["D"], c["HQ"], c["HKV"], c["seqs"], c["new"], len(t["q"])
    req, at = places(t, rows)
    i = at - t["pos"].long()[req]
    q = norm_rotate(t["q"][..., :D].float(), at, c, t.get("norm"))
    full = q.new_zeros((n, m, HKV, HQ // HKV, D))
    full[req, i] = q.reshape(rows, HKV, HQ // HKV, D)
    full = full.permute(0, 2, 3, 1, 4).reshape(n, HKV, -1, D)  # the queries that share a head of the cache
    keys, values = (x.reshape(n, HKV, -1, D) for x in unpack(t["cache"][t["seqs"].long()], D))
    s = (full @ keys.transpose(-1, -2) * D ** -0.5).view(n, HKV, HQ // HKV, m, -1)
    seen = torch.arange(s.shape[-1], device="cuda") <= t["pos"][:, None, None] + torch.arange(m, device="cuda")[:, None]
    s = torch.where(seen[:, None, None], s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = torch.where(seen[:, None, None], p, 0)
    values = torch.where(seen[:, None, -1, :, None], values, 0)  # rows behind a sequence's last one may hold anything
    o = (p.view(n, HKV, -1, s.shape[-1]) @ values).view(n, HKV, HQ // HKV, m, D) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, m, HQ, D)[req, i]
    if c["gate"]:
        o = o * torch.sigmoid(t["q"][..., D:].float())
    return o.half().view(rows, HQ * D)


def plain_verify(state):
    """in 64 bits: a uniform number next to a border between two tokens has to fall on the same side"""
    c, t = state["case"], state["t"]
    V, n, m, rows, k = c["vocab"], c["seqs"], c["new"] + 1, len(t["drafts"]), c["top_k"]
    first, last = t["starts"][:-1].long(), t["starts"][1:].long() - 1
    row = torch.arange(rows, device="cuda")
    req = torch.searchsorted(t["starts"][1:].long(), row, right=True)
    drafts = t["drafts"].long()
    if c["temperature"] <= 0:
        best = t["logits"].argmax(1)
        stands = drafts == best
        mine = stands.double()
    else:
        x = t["logits"]
        if k:  # the k largest, the smaller index first among equals
            x, order = (y[:, :k] for y in torch.sort(x, dim=1, descending=True, stable=True))
        e = torch.exp((x.double() - x.amax(1, keepdim=True).double()) / c["temperature"])
        p = e / e.sum(1, keepdim=True)
        mine = torch.where(order == drafts[:, None], p, 0).sum(1) if k else p.gather(1, drafts[:, None])[:, 0]
        theirs = t["probs"].gather(1, drafts[:, None])[:, 0].double() if c["probs"] else 1.0
        stands = t["u_accept"].double() * theirs < mine
    stop = torch.where(stands & (row < last[req]), rows, row)  # a sequence goes on at its first row that does not stand, or at its last
    at = torch.full((n,), rows, device="cuda").scatter_reduce(0, req, stop, "amin")
    if c["temperature"] <= 0:
        token = best[at]
    else:
        p, inner = p[at], (at < last)[:, None]
        names = order[at] if k else torch.arange(V, device="cuda").expand(n, V)
        theirs = t["probs"][at].double().gather(1, names) if c["probs"] else (names == drafts[at][:, None]).double()
        left = torch.where(inner, (p - theirs).clamp(min=0), p)
        left = torch.where(left.sum(1, keepdim=True) > 0, left, p)
        total = left.cumsum(1)
        goal = t["u_pick"].double()[:, None] * total[:, -1:]
        token = names.gather(1, (total <= goal).sum(1).clamp(max=names.shape[1] - 1)[:, None])[:, 0]
    tokens = torch.where(row < at[req], drafts, torch.where(row == at[req], token[req], -1)).int()
    return {"tokens": tokens, "accepted": (at - first).int(), "p": torch.where(row < last[req], mine, 0).float()}


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    pos, new = lengths(case)
    if case["kind"] == "verify":  # the target's logits once; of the draft's probabilities one value a row, and a row where a draft falls
        V, rows = case["vocab"], sum(new) + case["seqs"]
        return {"bytes": 4 * V * (rows + (case["seqs"] if case["probs"] and not case["top_k"] else 0)), "flops": 4 * V * rows}
    D, HQ, HKV, size, rows = case["D"], case["HQ"], case["HKV"], 4 if case["type"] == "f32" else 2, sum(new)
    packed = 9 * D // 8  # bytes of a row and head: keys and values with their scales
    if case["kind"] == "append":  # rows in, codes out and in again, values out
        return {"bytes": rows * HKV * (2 * D * size + 2 * packed + 8 * D), "flops": 20 * rows * HKV * D}
    seen = sum(p + k for p, k in zip(pos, new))
    pairs = sum(k * p + k * (k + 1) // 2 for p, k in zip(pos, new))
    return {"bytes": seen * HKV * packed + rows * HQ * D * (size * (1 + case["gate"]) + 2), "flops": 4 * pairs * HQ * D}


# ---- the same in 64 bits, sequence by sequence -------------------------------------------------------------------
def turned(x, at, case, weight):
    """one row x [heads, D] of position `at`"""
    x = x.clone()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.double()
    half = case["rot"] // 2
    if half:
        z = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:-1], half, 2).contiguous())
        angle = at * torch.exp(-math.log(THETA) * torch.arange(half, dtype=torch.float64, device=x.device) / half)
        x[..., :2 * half] = torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)).flatten(-2)
    return x


def cached_rows(cache, seq, head, count, D):
    """keys and values of rows 0..count-1 of a sequence and head, taken from the bytes by their places"""
    raw = cache[seq, head].long()
    row, f = torch.arange(count, device="cuda")[:, None], torch.arange(D, device="cuda")[None]
    block, r, g = row // 16, row % 16, f // 64
    S = D // 64
    place = 2 * (r // 4) + r % 2
    kb = raw[block, (((r // 2) % 2 * S + g) * 8 + place) * 32 + f % 64 // 2]
    vb = raw[block, 8 * D + ((g * 8 + f % 64 // 8) * 16 + r) * 4 + f % 8 // 2]
    half = cache[seq, head][:, 16 * D:].contiguous().view(torch.float16).double()
    scale = lambda part: half[block, ((part * S + g) * 16 + r) * 2]  # noqa: E731
    low = lambda part: half[block, ((part * S + g) * 16 + r) * 2 + 1]  # noqa: E731
    return [low(part) + scale(part) * ((byte >> (4 * (f % 2))) & 15).double() for part, byte in enumerate((kb, vb))]


def exact(case, seed):
    t, (pos, new) = inputs(case, seed), lengths(case)
    n, at = case["seqs"], 0
    if case["kind"] == "verify":
        p = torch.zeros(len(t["drafts"]), dtype=torch.float64, device="cuda")
        for r in range(n):
            for row in range(at, at + new[r]):
                x, draft = t["logits"][row].double(), int(t["drafts"][row])
                if case["temperature"] <= 0:
                    p[row] = float(x[draft] == x.max())
                    continue
                if case["top_k"]:
                    x = x.masked_fill(x < torch.topk(x, case["top_k"]).values[-1], -math.inf)
                p[row] = torch.softmax(x / case["temperature"], 0)[draft]
            at += new[r] + 1
        return {"tokens": None, "accepted": None, "p": p}
    D, HQ, HKV = case["D"], case["HQ"], case["HKV"]
    if case["kind"] == "append":
        kv, keys, at = t["kv"].double().view(-1, 2, HKV, D), [], 0
        for r in range(n):
            for i in range(new[r]):
                keys.append(turned(kv[at, 0], pos[r] + i, case, t.get("norm")))
                at += 1
        out = []
        for x in (torch.stack(keys), kv[:, 1]):
            g = x.reshape(-1, 64)
            lo, hi = (m(g, 1).values.clamp(-65504, 65504) for m in (torch.min, torch.max))
            lo = lo.to(torch.float32).to(torch.float16).double()
            step = torch.clamp((hi - lo) / 15, min=0).to(torch.float32).to(torch.float16).double()
            code = torch.clamp(torch.round((g - lo[:, None]) / torch.where(step > 0, step, math.inf)[:, None]), 0, 15)  # halves to the even code
            out.append((lo[:, None] + step[:, None] * code).view(x.shape))
        return {"keys": out[0], "values": out[1]}
    if sum(p + k for p, k in zip(pos, new)) * HKV > 4_000_000:
        return None
    out = torch.empty((sum(new), HQ, D), dtype=torch.float64, device="cuda")
    where = t["seqs"].tolist()
    for r in range(n):
        last = pos[r] + new[r]
        q = torch.stack([turned(t["q"][at + i, :, :D].double(), pos[r] + i, case, t.get("norm")) for i in range(new[r])])
        mask = torch.arange(last, device="cuda")[None] <= pos[r] + torch.arange(new[r], device="cuda")[:, None]
        for h in range(HKV):
            k, v = cached_rows(t["cache"], where[r], h, last, D)
            for j in range(h * HQ // HKV, (h + 1) * HQ // HKV):
                s = (q[:, j] @ k.T / math.sqrt(D)).masked_fill(~mask, -math.inf)
                out[at:at + new[r], j] = torch.softmax(s, 1) @ v
        at += new[r]
    if case["gate"]:
        out = out / (1 + torch.exp(-t["q"][..., D:].double()))
    return out.view(-1, HQ * D)
