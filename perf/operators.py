"""Timed cases of the serving and scoring operators: attention with a sliding
window and visible first tokens, attention of a batch over one shared prefix,
and token log probabilities with entropy and alternatives, with their gradient.

Each case runs either in its plain form (elementary torch operations in 32
bits) or through the package's entry points (``own``); ``exact`` computes the
same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NO_TOKEN = -1  # u32 0xffffffff: this row's token is not scored


def listed():
    return [
        # a long prompt through a windowed layer
        dict(name="window prompt 8192", kind="window", dtype="bf16", batch=1, heads=32, kv_heads=8, depth=128, queries=8192,
             keys=8192, window=1024, sinks=4, ragged=False),
        # one chunk of a prompt behind what the cache already holds, odd sizes
        dict(name="window chunk 777", kind="window", dtype="f16", batch=2, heads=12, kv_heads=12, depth=64, queries=777,
             keys=2311, window=500, sinks=1, ragged=True),
        # a serving batch, one token per sequence, caches filled unevenly
        dict(name="window decode x16", kind="window", dtype="bf16", batch=16, heads=32, kv_heads=8, depth=128, queries=1,
             keys=16384, window=4096, sinks=4, ragged=True),
        # one user's next token: latency
        dict(name="window decode x1", kind="window", dtype="bf16", batch=1, heads=32, kv_heads=8, depth=128, queries=1,
             keys=1000, window=256, sinks=4, ragged=True),
        # many continuations sampled from one long prompt
        dict(name="prefix decode x64", kind="prefix", dtype="bf16", batch=64, heads=32, kv_heads=8, depth=128, queries=1,
             prefix=8192, keys=512, ragged=True),
        # given answers scored against one prompt, all their tokens at once
        dict(name="prefix answers 16x33", kind="prefix", dtype="bf16", batch=16, heads=32, kv_heads=8, depth=128, queries=33,
             prefix=4096, keys=33, ragged=False),
        # a few candidates behind a short prompt: latency
        dict(name="prefix decode x4", kind="prefix", dtype="f16", batch=4, heads=12, kv_heads=4, depth=64, queries=1,
             prefix=1001, keys=40, ragged=True),
        # scoring of a batch of texts, a few alternatives per token
        dict(name="logprobs 2048x131072", kind="logprobs", dtype="bf16", rows=2048, classes=131072, top=5),
        # a serving step: one row per sequence, f16 logits
        dict(name="logprobs 64x32000", kind="logprobs", dtype="f16", rows=64, classes=32000, top=8),
        # one user's next token with its alternatives, odd vocabulary: latency
        dict(name="logprobs 1x50021", kind="logprobs", dtype="f32", rows=1, classes=50021, top=20),
        # the policy and entropy gradient of a batch of sampled tokens
        dict(name="gradient 2048x131072", kind="gradient", dtype="bf16", rows=2048, classes=131072, entropy=True),
        # a small step in f32, odd vocabulary
        dict(name="gradient 37x50021", kind="gradient", dtype="f32", rows=37, classes=50021, entropy=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _size(rng, lo, hi):
    n = _log(rng, lo, hi)
    return n + 1 if n == 3 * 1024 else n


HEADS = ((32, 8), (12, 4), (12, 12), (16, 2), (8, 8), (32, 4))


def draw(rng):
    while True:
        kind = rng.choice(("window", "window", "prefix", "prefix", "logprobs", "gradient"))
        if kind in ("window", "prefix"):
            heads, kv_heads = rng.choice(HEADS)
            c = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "f16")), batch=1, heads=heads, kv_heads=kv_heads,
                     depth=rng.choice((64, 128)), ragged=rng.random() < 0.6)
            if kind == "window":
                decode = rng.random() < 0.5
                c["queries"] = rng.choice((1, 1, 1, 2, 4)) if decode else _size(rng, 17, 8192)
                c["keys"] = max(c["queries"], _size(rng, 64, 16384 if decode else 8192))
                c["batch"] = _size(rng, 1, 64 if decode else 4)
                c["window"] = _size(rng, 32, 4096)
                c["sinks"] = rng.choice((0, 1, 4, 4, 64))
            else:
                c["queries"] = rng.choice((1, 1, 1, 2, _size(rng, 3, 64)))
                c["batch"] = _size(rng, 2, 64)
                c["prefix"] = _size(rng, 64, 16384)
                c["keys"] = max(c["queries"], _size(rng, 1, 1024))
            keys = c["keys"] + c.get("prefix", 0)
            if c["batch"] * heads * c["queries"] * keys > 32 * 8192 * 8192:
                continue
            if c["batch"] * kv_heads * c["keys"] * c["depth"] * 4 > 1.1e9:
                continue
        else:
            c = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "f16", "f32")), rows=_size(rng, 1, 4096),
                     classes=_size(rng, 1000, 140000))
            if kind == "logprobs":
                c["top"] = rng.choice((0, 1, 5, 8, 20, 32))
            else:
                c["entropy"] = rng.random() < 0.5
            if c["rows"] * c["classes"] * (2 if c["dtype"] == "f32" else 1) > 2048 * 131072:
                continue
        return c


# --------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(shape, dtype, g):
    return torch.randn(shape, device=DEV, generator=g, dtype=torch.float32).to(dtype)


def _lengths(c, g):
    """How many keys of each sequence's cache are filled: between a quarter and all, at least the queries."""
    lo = max(c["queries"], c["keys"] // 4)
    return torch.randint(lo, c["keys"] + 1, (c["batch"],), device=DEV, generator=g, dtype=torch.int32)


def prepare(case, seed):
    c, g = case, _gen(seed)
    dtype = TYPES[c["dtype"]]
    if c["kind"] in ("window", "prefix"):
        b, h, hk, d = c["batch"], c["heads"], c["kv_heads"], c["depth"]
        # queries and keys as a projection leaves them: [batch, tokens, heads, depth], seen as [batch, heads, tokens, depth]
        st = dict(case=c, q=_normal((b, c["queries"], h, d), dtype, g).transpose(1, 2),
                  k=_normal((b, hk, c["keys"], d), dtype, g), v=_normal((b, hk, c["keys"], d), dtype, g),
                  lengths=_lengths(c, g) if c["ragged"] else None)
        if c["kind"] == "prefix":
            st["pk"], st["pv"] = _normal((hk, c["prefix"], d), dtype, g), _normal((hk, c["prefix"], d), dtype, g)
        return st
    n, v = c["rows"], c["classes"]
    logits = torch.randn((n, v), device=DEV, generator=g, dtype=torch.float32).mul_(2.5)
    logits[:, v - v % 64:] = -math.inf  # padding classes of a vocabulary rounded up
    # tokens: half of them the likeliest of a random few, half any; one in twenty not scored
    few = torch.randint(0, v - v % 64, (n, 64), device=DEV, generator=g)
    best = few.gather(1, logits.gather(1, few).argmax(1, keepdim=True))[:, 0]
    u = torch.rand((n,), device=DEV, generator=g)
    targets = torch.where(u < 0.5, best, few[:, 0])
    targets = torch.where(u > 0.95, torch.full_like(targets, NO_TOKEN), targets).to(torch.int32)
    st = dict(case=c, logits=logits.to(dtype), targets=targets)
    if c["kind"] == "gradient":
        x = st["logits"].float()
        z = x - x.amax(1, keepdim=True)
        e = z.exp()
        s = e.sum(1)
        st["lse"] = s.log() + x.amax(1)
        st["entropy"] = s.log() - torch.where(e > 0, z * e, torch.zeros_like(z)).sum(1) / s
        # advantages, under the loss scale that f16 gradients need
        st["scale"] = 4096.0 if c["dtype"] == "f16" else 1.0
        st["g_logprob"] = torch.randn((n,), device=DEV, generator=g) * st["scale"]
        st["g_entropy"] = torch.rand((n,), device=DEV, generator=g) * (0.02 * st["scale"]) if c["entropy"] else None
    return st


# ---------------------------------------------------------- plain forms

def _attend(scores, values):
    """softmax(scores) @ values over the last axes; rows with no key (all -inf) are zeros."""
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, values)
    return torch.where(total > 0, o / total, torch.zeros_like(o))


def _grouped(st):
    """Queries as [batch, kv heads, group x queries, depth] in 32 bits, scaled."""
    c = st["case"]
    g = c["heads"] // c["kv_heads"]
    q = st["q"].float() * (1.0 / math.sqrt(c["depth"]))
    return q.reshape(c["batch"], c["kv_heads"], g * c["queries"], c["depth"])


def _positions(st):
    """(position of each query [batch, queries], filled keys [batch, 1])"""
    c = st["case"]
    filled = st["lengths"].long()[:, None] if st["lengths"] is not None else torch.full((c["batch"], 1), c["keys"], device=DEV)
    return filled - c["queries"] + torch.arange(c["queries"], device=DEV)[None], filled


def _plain_window(st):
    c = st["case"]
    b, hk, lq, g = c["batch"], c["kv_heads"], c["queries"], c["heads"] // c["kv_heads"]
    pos, filled = _positions(st)
    j = torch.arange(c["keys"], device=DEV)[None, None]
    p = pos[:, :, None]
    seen = (j <= p) & (j < filled[:, :, None]) & ((j > p - c["window"]) | (j < c["sinks"]))
    s = torch.matmul(_grouped(st), st["k"].float().transpose(-1, -2)).view(b, hk, g, lq, c["keys"])
    s = s.masked_fill_(~seen[:, None, None], -math.inf).view(b, hk, g * lq, c["keys"])
    return _attend(s, st["v"].float()).view(b, c["heads"], lq, c["depth"]).to(st["q"].dtype)


def _plain_prefix(st):
    c = st["case"]
    b, hk, lq, g = c["batch"], c["kv_heads"], c["queries"], c["heads"] // c["kv_heads"]
    pos, _ = _positions(st)
    q = _grouped(st)
    shared = torch.matmul(q, st["pk"].float().transpose(-1, -2))
    j = torch.arange(c["keys"], device=DEV)[None, None]
    seen = j <= pos[:, :, None]
    s = torch.matmul(q, st["k"].float().transpose(-1, -2)).view(b, hk, g, lq, c["keys"])
    s = s.masked_fill_(~seen[:, None, None], -math.inf).view(b, hk, g * lq, c["keys"])
    top = torch.maximum(shared.amax(-1, keepdim=True), s.amax(-1, keepdim=True))
    shared, s = torch.exp(shared - top), torch.exp(s - top)
    o = torch.matmul(shared, st["pv"].float()) + torch.matmul(s, st["v"].float())
    o = o / (shared.sum(-1, keepdim=True) + s.sum(-1, keepdim=True))
    return o.view(b, c["heads"], lq, c["depth"]).to(st["q"].dtype)


def _plain_logprobs(st):
    c = st["case"]
    x = st["logits"].float()
    top = x.amax(1, keepdim=True)
    z = x - top
    e = z.exp()
    s = e.sum(1)
    lse = s.log() + top[:, 0]
    entropy = s.log() - torch.where(e > 0, z * e, torch.zeros_like(z)).sum(1) / s
    t = st["targets"].long()
    at = x.gather(1, t.clamp(min=0)[:, None])[:, 0]
    out = dict(logprob=torch.where(t >= 0, at - lse, torch.zeros_like(lse)), entropy=entropy, logsumexp=lse)
    if c["top"]:
        # the IEEE total order, lowest index first among equals
        bits = x.view(torch.int32)
        order = torch.sort(bits ^ ((bits >> 31) & 0x7FFFFFFF), dim=1, descending=True, stable=True)[1][:, : c["top"]]
        out["top_index"] = order.to(torch.int32)
        out["top_logprob"] = x.gather(1, order) - lse[:, None]
    return out


def _plain_gradient(st):
    x = st["logits"].float()
    z = x - st["lse"][:, None]
    p = z.exp()
    t = st["targets"].long()
    gl = torch.where(t >= 0, st["g_logprob"], torch.zeros_like(st["g_logprob"]))
    d = p * -gl[:, None]
    d.scatter_add_(1, t.clamp(min=0)[:, None], gl[:, None])
    if st["g_entropy"] is not None:
        d -= st["g_entropy"][:, None] * torch.where(p > 0, p * (z + st["entropy"][:, None]), torch.zeros_like(p))
    return d.to(st["logits"].dtype)


def run(state):
    c = state["case"]
    if not own:
        return {"window": _plain_window, "prefix": _plain_prefix, "logprobs": _plain_logprobs,
                "gradient": _plain_gradient}[c["kind"]](state)
    from forma_b200 import api

    if c["kind"] == "window":
        return api.attention_window(state["q"], state["k"], state["v"], c["window"], c["sinks"], state["lengths"])
    if c["kind"] == "prefix":
        return api.attention_prefix(state["q"], state["pk"], state["pv"], state["k"], state["v"], state["lengths"])
    if c["kind"] == "logprobs":
        r = api.token_logprobs(state["logits"], state["targets"], c["top"])
        out = dict(logprob=r.logprob, entropy=r.entropy, logsumexp=r.logsumexp)
        if c["top"]:
            out["top_index"], out["top_logprob"] = r.top_index, r.top_logprob
        return out
    return api.token_logprobs_grad(state["logits"], state["targets"], state["lse"], state["g_logprob"], state["entropy"],
                                   state["g_entropy"])


# ------------------------------------------------------------- the floor

def _visible(c):
    """Pairs (query, key) that a sequence's mask leaves, its cache 5/8 filled on the average where it is ragged."""
    lq = c["queries"]
    filled = max(lq, int(c["keys"] * 0.625)) if c["ragged"] else c["keys"]
    p = torch.arange(filled - lq, filled, dtype=torch.float64)
    if c["kind"] == "prefix":
        return float((p + 1).sum()), filled
    near = torch.clamp(p + 1, max=c["window"])
    first = torch.clamp(p + 1 - near, min=0).clamp(max=c["sinks"])
    touched = min(filled, lq + c["window"] - 1 + c["sinks"])
    return float((near + first).sum()), touched


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] in ("window", "prefix"):
        pairs, touched = _visible(c)
        kv = 2 * c["batch"] * c["kv_heads"] * touched * c["depth"] * size
        io = 2 * c["batch"] * c["heads"] * c["queries"] * c["depth"] * size
        if c["kind"] == "prefix":
            pairs += c["queries"] * c["prefix"]
            kv += 2 * c["kv_heads"] * c["prefix"] * c["depth"] * size
        return {"bytes": kv + io, "flops": 4.0 * c["batch"] * c["heads"] * pairs * c["depth"]}
    n = c["rows"] * c["classes"]
    if c["kind"] == "logprobs":
        return {"bytes": n * size + c["rows"] * (16 + 8 * c["top"]), "flops": 4.0 * n}
    return {"bytes": 2 * n * size + c["rows"] * 20, "flops": 5.0 * n}


# ---------------------------------------------------- 64-bit definitions

def _exact_attention(c, st):
    """Sequence by sequence and key/value head by head, over the keys that a block of queries may see."""
    b, hk, lq, d = c["batch"], c["kv_heads"], c["queries"], c["depth"]
    g = c["heads"] // hk
    out = torch.zeros((b, c["heads"], lq, d), dtype=torch.float64, device=DEV)
    filled = st["lengths"].tolist() if st["lengths"] is not None else [c["keys"]] * b
    for i in range(b):
        for n in range(hk):
            q = st["q"][i, n * g:(n + 1) * g].double()
            k, v = st["k"][i, n].double(), st["v"][i, n].double()
            for a in range(0, lq, 512):
                z = min(a + 512, lq)
                p = torch.arange(a, z, device=DEV) + (filled[i] - lq)
                hi = max(0, min(filled[i], filled[i] - lq + z))
                lo = 0 if c["kind"] == "prefix" else max(0, filled[i] - lq + a - c["window"] + 1)
                first = min(0 if c["kind"] == "prefix" else c["sinks"], lo, hi)
                j = torch.cat([torch.arange(first, device=DEV), torch.arange(lo, max(lo, hi), device=DEV)])
                ok = j[None] <= p[:, None]
                if c["kind"] == "window":
                    ok &= (j[None] + c["window"] > p[:, None]) | (j[None] < c["sinks"])
                logit = torch.einsum("gqd,kd->gqk", q[:, a:z], k[j]) / math.sqrt(d)
                logit = torch.where(ok[None], logit, torch.full_like(logit, -math.inf))
                values = v[j]
                if c["kind"] == "prefix":
                    logit = torch.cat([torch.einsum("gqd,kd->gqk", q[:, a:z], st["pk"][n].double()) / math.sqrt(d), logit], 2)
                    values = torch.cat([st["pv"][n].double(), values])
                if logit.shape[2]:
                    out[i, n * g:(n + 1) * g, a:z] = torch.nan_to_num(torch.softmax(logit, 2), nan=0.0) @ values
    return out


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["kind"] in ("window", "prefix"):
        return _exact_attention(c, st)
    results = []
    step = max(1, (1 << 26) // c["classes"])
    for a in range(0, c["rows"], step):
        x, t = st["logits"][a:a + step].double(), st["targets"][a:a + step].long()
        lse = torch.logsumexp(x, 1)
        logp = x - lse[:, None]
        p = torch.exp(logp)
        plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
        scored = (t >= 0).double()
        if c["kind"] == "logprobs":
            row = [logp.gather(1, t.clamp(min=0)[:, None])[:, 0] * scored, -plogp.sum(1), lse]
            if c["top"]:
                row.append(torch.sort(logp, 1, descending=True)[0][:, : c["top"]])
            results.append(row)
        else:
            d = -p * (st["g_logprob"][a:a + step].double() * scored)[:, None]
            d[torch.arange(x.shape[0], device=DEV), t.clamp(min=0)] += st["g_logprob"][a:a + step].double() * scored
            if st["g_entropy"] is not None:
                h = -plogp.sum(1, keepdim=True)
                d -= st["g_entropy"][a:a + step].double()[:, None] * (plogp + p * h)
            results.append([d])
    whole = [torch.cat(parts) for parts in zip(*results)]
    if c["kind"] == "gradient":
        return whole[0]
    out = dict(logprob=whole[0], entropy=whole[1], logsumexp=whole[2])
    if c["top"]:
        out["top_index"], out["top_logprob"] = None, whole[3]
    return out
