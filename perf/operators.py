"""Cases of the operators that draw several continuations of one prompt: rows written to a KV
cache and read back, attention of a batch over a prefix that all its sequences share, and sampling.

Geometries are the framework's own (32 query heads over 4 key/value heads of 128, a vocabulary of
151,936) and smaller generic ones.  Lengths go from one token to a 32K prompt.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ONE = 2.0 ** 40   # a sampling weight of 1
TINY = 2.0 ** -50  # rows of the 8-bit cache below this are stored as zero


def listed():
    kv = dict(op="kv", heads=4, dim=128)
    at = dict(op="attend", heads=32, kv_heads=4, dim=128)
    sm = dict(op="sample", n=151936)
    return [
        # one decode step's new keys and values of 16 sequences, cut out of the fused projection
        dict(kv, name="kv-step-16", seqs=16, new=1, capacity=1024, src="f32", cache="q8", fused=True),
        # a prompt's rows of odd length, f16 cache, smaller heads
        dict(kv, name="kv-prompt-4097-f16", seqs=1, new=4097, capacity=8192, src="f32", cache="f16", fused=False, heads=8, dim=64),
        # the rows of a 32K prompt
        dict(kv, name="kv-prompt-32768", seqs=1, new=32768, capacity=32768, src="f32", cache="q8", fused=False),
        # one sequence, a short prompt: the smallest call
        dict(at, name="attend-1-short", seqs=1, queries=1, prefix=40, capacity=64, low=1, high=1, q="f32", cache="f16"),
        # a few sequences some way into their continuations, f32 rows as the decoder holds them
        dict(at, name="attend-8-4k-q8", seqs=8, queries=1, prefix=4096, capacity=512, low=3, high=400, q="f32", cache="q8"),
        # several new tokens a sequence (a drafted run being verified), odd sizes, smaller heads
        dict(at, name="attend-5x7-odd", seqs=5, queries=7, prefix=1003, capacity=333, low=7, high=333, q="f32", cache="f16", heads=12, dim=64),
        # a batch whose own tokens outweigh the prompt
        dict(at, name="attend-48-own", seqs=48, queries=1, prefix=777, capacity=2048, low=1, high=2048, q="f16", cache="f16"),
        # best of 64 over an 8-bit prompt of 16K
        dict(at, name="attend-64-16k-q8", seqs=64, queries=1, prefix=16384, capacity=512, low=1, high=512, q="f16", cache="q8"),
        # 128 sequences over a 32K prompt: the largest
        dict(at, name="attend-128-32k", seqs=128, queries=1, prefix=32768, capacity=256, low=1, high=256, q="f16", cache="f16"),
        # one sequence's next token, every filter on
        dict(sm, name="sample-1", rows=1, temperature=0.7, top_k=20, top_p=0.8, min_p=0.01, spread=2.5),
        # 64 continuations, nucleus only
        dict(sm, name="sample-64-top-p", rows=64, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, spread=2.5),
        # many rows of a smaller odd vocabulary, flat scores, a wide top-k
        dict(sm, name="sample-300-flat", rows=300, n=49999, temperature=1.3, top_k=5000, top_p=0.99, min_p=0.0, spread=1.0),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["kv", "attend", "attend", "sample"])
    if op == "kv":
        seqs = log(1, 64)
        new = log(1, 32768 // seqs)
        return dict(op="kv", heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]), seqs=seqs, new=new,
                    capacity=new + rng.randint(0, 500), src=rng.choice(["f32", "f16", "bf16"]), cache=rng.choice(["q8", "q8", "f16"]),
                    fused=rng.random() < 0.5)
    if op == "sample":
        n = log(1000, 151936)
        return dict(op="sample", n=n, rows=log(1, 300), temperature=round(rng.uniform(0.3, 1.5), 3),
                    top_k=rng.choice([0, log(1, n)]), top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                    min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]), spread=round(rng.uniform(1.0, 4.0), 2))
    while True:
        kv_heads = rng.choice([1, 2, 4, 8])
        c = dict(op="attend", heads=kv_heads * rng.choice([1, 3, 4, 8]), kv_heads=kv_heads, dim=rng.choice([64, 128]), seqs=log(1, 128),
                 queries=rng.choice([1, 1, 1, log(1, 16)]), prefix=log(1, 32768), capacity=log(16, 2048), q=rng.choice(["f32", "f16"]),
                 cache=rng.choice(["f16", "q8"]))
        c["low"] = min(c["queries"], c["capacity"])
        c["high"] = rng.randint(c["low"], c["capacity"])
        w, most = work(c), work(next(x for x in listed() if x["name"] == "attend-128-32k"))
        if w["flops"] <= most["flops"] and w["bytes"] <= most["bytes"]:
            return c


# ------------------------------------------------------------------ inputs
def lengths(c):
    """The sequences' lengths: spread evenly from low to high."""
    n = c["seqs"]
    return [c["low"] + (c["high"] - c["low"]) * i // max(1, n - 1) for i in range(n)]


def rows_q8(x):
    """Levels and scales of rows (the last dimension) in the 8-bit cache."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    zero = amax < TINY
    levels = torch.round(x * (127.0 / torch.where(zero, torch.ones_like(amax), amax)))
    levels = torch.where(zero, torch.zeros_like(levels), levels).to(torch.int8)
    scale = torch.where(zero, torch.zeros_like(amax), amax / 127.0)
    return levels, scale[..., 0].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = dict(case)
    if c["op"] == "sample":
        B, n = c["rows"], c["n"]

        def full(v, dtype=torch.float32):
            return torch.full((B,), v, dtype=dtype, device="cuda")

        # a wide body and a few tokens that stand out, as a model's scores have
        logits = torch.randn(B, n, device="cuda", generator=g) * c["spread"]
        logits += 6.0 * torch.randn(B, n, device="cuda", generator=g).clamp_(min=3.5).sub_(3.5)
        return dict(c, logits=logits, u=torch.rand(B, device="cuda", generator=g), temperature=full(c["temperature"]),
                    top_k=full(c["top_k"], torch.int32), top_p=full(c["top_p"]), min_p=full(c["min_p"]))

    H, D, B = c["heads"], c["dim"], c["seqs"]
    # channels of unequal size, as keys have
    size = 0.5 + 1.5 * torch.rand(D, device="cuda", generator=g)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if c["op"] == "kv":
        n, cap = c["new"], c["capacity"]
        lead = H * D if c["fused"] else 0  # what stands before the keys in a fused row
        rows = normal(B * n, lead + 2 * H * D).to(DTYPES[c["src"]])
        k = rows[:, lead:lead + H * D].unflatten(0, (B, n)).unflatten(2, (H, D))
        v = rows[:, lead + H * D:].unflatten(0, (B, n)).unflatten(2, (H, D))
        lens = n + torch.randint(0, cap - n + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        return state_of(dict(c, k=k, v=v, lens=lens), "cache", cache_of(c["cache"], torch.zeros(B, cap, H, D, device="cuda"),
                                                                        torch.zeros(B, cap, H, D, device="cuda")))
    Hkv = c["kv_heads"]
    q = (1.5 * normal(B, c["queries"], H, D)).to(DTYPES[c["q"]])
    lens = torch.tensor(lengths(c), dtype=torch.int32, device="cuda")[torch.randperm(B, device="cuda", generator=g)]
    s = dict(c, q=q, lens=lens, scale=D ** -0.5)
    state_of(s, "prefix_rows", cache_of(c["cache"], normal(1, c["prefix"], Hkv, D) * size, normal(1, c["prefix"], Hkv, D)))
    state_of(s, "suffix_rows", cache_of(c["cache"], normal(B, c["capacity"], Hkv, D) * size, normal(B, c["capacity"], Hkv, D)))
    return s


def cache_of(kind, k, v):
    """A cache's tensors for rows k and v: f16 rows, or int8 levels with one f32 scale a row."""
    if kind == "f16":
        return dict(k=k.half(), v=v.half(), k_scale=None, v_scale=None)
    (kl, ks), (vl, vs) = rows_q8(k), rows_q8(v)
    return dict(k=kl, v=vl, k_scale=ks, v_scale=vs)


def state_of(state, name, tensors):
    """Puts a cache's tensors into the state, and the framework's view of them, which a program keeps
    for the cache's life (it holds the four tensors; nothing is computed or laid out)."""
    state[name] = tensors
    if own:
        import ramvamp_b200 as rv

        state[name + "_view"] = rv.KvCache.of(tensors["k"], tensors["v"], tensors["k_scale"], tensors["v_scale"])
    return state


# --------------------------------------------------------------- one pass
def run(state):
    s = state
    if own:
        import ramvamp_b200 as rv

        if s["op"] == "kv":
            rv.kv_append(s["cache_view"], s["k"], s["v"], lens=s["lens"])
            return rv.kv_read(s["cache_view"], s["new"], lens=s["lens"], dtype=torch.float16 if s["cache"]["k_scale"] is None else torch.float32)
        if s["op"] == "attend":
            return rv.prefix_attention(s["q"], s["prefix_rows_view"], s["prefix"], s["suffix_rows_view"], s["lens"], scale=s["scale"])
        return rv.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return {"kv": plain_kv, "attend": plain_attend, "sample": plain_sample}[s["op"]](s)


def plain_kv(s):
    c, B, n = s["cache"], s["seqs"], s["new"]
    seq = torch.arange(B, device="cuda")[:, None]
    pos = s["lens"].long()[:, None] - n + torch.arange(n, device="cuda")
    if c["k_scale"] is None:
        c["k"][seq, pos] = s["k"].half()
        c["v"][seq, pos] = s["v"].half()
        return c["k"][seq, pos], c["v"][seq, pos]
    c["k"][seq, pos], c["k_scale"][seq, pos] = rows_q8(s["k"])
    c["v"][seq, pos], c["v_scale"][seq, pos] = rows_q8(s["v"])
    return c["k"][seq, pos].float() * c["k_scale"][seq, pos][..., None], c["v"][seq, pos].float() * c["v_scale"][seq, pos][..., None]


def values(c, name):
    x = c[name].float()
    return x if c[name + "_scale"] is None else x * c[name + "_scale"][..., None]


def plain_attend(s):
    B, Q, H, D = s["q"].shape
    Hkv = s["kv_heads"]
    G, cap = H // Hkv, s["capacity"]
    q = s["q"].float().reshape(B, Q, Hkv, G, D)
    pk, pv = (values(s["prefix_rows"], x)[0].transpose(0, 1) for x in ("k", "v"))   # [Hkv, P, D]
    sk, sv = (values(s["suffix_rows"], x).transpose(1, 2) for x in ("k", "v"))      # [B, Hkv, cap, D]
    qp = q.permute(2, 0, 1, 3, 4).reshape(Hkv, B * Q * G, D)
    qs = q.permute(0, 2, 1, 3, 4).reshape(B, Hkv, Q * G, D)
    a = (qp @ pk.transpose(1, 2)) * s["scale"]                                       # [Hkv, B*Q*G, P]
    b = (qs @ sk.transpose(2, 3)) * s["scale"]                                       # [B, Hkv, Q*G, cap]
    seen = s["lens"].long()[:, None] - Q + 1 + torch.arange(Q, device="cuda")        # [B, Q]
    hidden = torch.arange(cap, device="cuda") >= seen[:, :, None]                    # [B, Q, cap]
    b = b.view(B, Hkv, Q, G, cap).masked_fill(hidden[:, None, :, None, :], -math.inf)
    a = a.view(Hkv, B, Q, G, -1).transpose(0, 1)                                     # [B, Hkv, Q, G, P]
    m = torch.maximum(a.amax(-1), b.amax(-1))[..., None]
    a, b = torch.exp(a - m), torch.exp(b - m)
    total = a.sum(-1) + b.sum(-1)
    o = (a.transpose(0, 1).reshape(Hkv, B * Q * G, -1) @ pv).view(Hkv, B, Q, G, D).transpose(0, 1)
    o = o + (b.reshape(B, Hkv, Q * G, cap) @ sv).view(B, Hkv, Q, G, D)
    o = o / total[..., None]
    return o.permute(0, 2, 1, 3, 4).reshape(B, Q, H, D).to(s["q"].dtype)


def plain_sample(s):
    logits, n = s["logits"], s["n"]
    top = logits.amax(1, keepdim=True)
    z = (logits - top) * (1.0 / s["temperature"])[:, None]
    e = torch.exp(z)
    w = (e * ONE).to(torch.int64)
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    rank = torch.arange(n, device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"].long(), n)[:, None]
    ranked = torch.where(rank < k, ranked, 0)
    before = ranked.cumsum(1) - ranked
    limit = (s["top_p"].double() * ranked.sum(1).double()).to(torch.int64)[:, None]
    keep = (rank < k) & ((before < limit) | (rank == 0) | (s["top_p"] >= 1.0)[:, None]) & (e.gather(1, order) >= s["min_p"][:, None])
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ranked, 0))
    total = kept.sum(1)
    target = torch.minimum((s["u"].double() * total.double()).to(torch.int64), total - 1)
    token = (kept.cumsum(1) > target[:, None]).to(torch.uint8).argmax(1)
    logprob = z.gather(1, token[:, None])[:, 0] - torch.log(total.double() / ONE).float()
    return token.to(torch.int32), logprob


# -------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "sample":
        return {"bytes": 4.0 * c["rows"] * c["n"] + 28.0 * c["rows"], "flops": 0.0}
    if c["op"] == "kv":
        rows = 2.0 * c["seqs"] * c["new"] * c["heads"]
        src = {"f32": 4, "f16": 2, "bf16": 2}[c["src"]]
        kept, back = (c["dim"] + 4, 4) if c["cache"] == "q8" else (2 * c["dim"], 2)
        return {"bytes": rows * (c["dim"] * (src + back) + 2 * kept), "flops": 0.0}
    Q, D, H = c["queries"], c["dim"], c["heads"]
    own_tokens = sum(lengths(c))
    row = 2 * (D + 4 if c["cache"] == "q8" else 2 * D)
    seen = sum(max(0, n - Q + 1 + i) for n in lengths(c) for i in range(Q))
    return {"bytes": float(c["kv_heads"] * (c["prefix"] + own_tokens) * row + 2 * c["seqs"] * Q * H * D * (4 if c["q"] == "f32" else 2)),
            "flops": 4.0 * H * D * (c["seqs"] * Q * c["prefix"] + seen)}


# ------------------------------------------------------ the values in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "kv":
        # the level that stands nearest to each value in units of its row's largest magnitude / 127
        def stored(x):
            if s["cache"]["k_scale"] is None:
                return x.double().half().double()
            x = x.double()
            unit = x.abs().amax(-1, keepdim=True) / 127
            return torch.where(unit > 0, torch.round(x / unit.clamp(min=1e-300)) * unit, torch.zeros_like(x))

        return stored(s["k"]), stored(s["v"])
    if s["op"] == "sample":
        x = s["logits"].double() / s["temperature"].double()[:, None]
        out = torch.empty(s["rows"], dtype=torch.float64, device="cuda")
        for r in range(s["rows"]):
            p = torch.softmax(x[r], 0)
            ranks = torch.argsort(s["logits"][r], descending=True, stable=True)
            if int(s["top_k"][r]) > 0:
                ranks = ranks[:int(s["top_k"][r])]
            pr = p[ranks] / p[ranks].sum()
            if float(s["top_p"][r]) < 1:
                pr = pr[:max(1, int((pr.cumsum(0) - pr < s["top_p"][r].double()).sum()))]
            pr = pr[pr >= s["min_p"][r].double() * pr[0]]
            ids, at = torch.sort(ranks[:len(pr)])
            pr = pr[at] / pr.sum()
            cdf = pr.cumsum(0)
            hit = min(int((cdf <= s["u"][r].double()).sum()), len(pr) - 1)
            out[r] = torch.log(pr[hit])
        return None, out

    B, Q, H, D = s["q"].shape
    G = H // s["kv_heads"]

    def wide(c, name):
        x = c[name].double()
        return x if c[name + "_scale"] is None else x * c[name + "_scale"].double().unsqueeze(-1)

    pk, pv, sk, sv = (wide(s[c], n) for c in ("prefix_rows", "suffix_rows") for n in ("k", "v"))
    lens, out = s["lens"].tolist(), torch.zeros(B, Q, H, D, dtype=torch.float64, device="cuda")
    if B * H * Q > 20000:
        return None
    for b in range(B):
        keys = torch.cat([pk[0], sk[b, :lens[b]]]).repeat_interleave(G, 1)
        vals = torch.cat([pv[0], sv[b, :lens[b]]]).repeat_interleave(G, 1)
        scores = torch.einsum("qhd,khd->hqk", s["q"][b].double(), keys) * D ** -0.5
        last = s["prefix"] + lens[b] - Q + torch.arange(Q, device="cuda")
        scores = scores.masked_fill(torch.arange(len(keys), device="cuda") > last[:, None], -math.inf)
        out[b] = torch.einsum("hqk,khd->qhd", torch.softmax(scores, -1), vals)
    return out
