"""The attention core of the decoder layer, as measurable cases: appending to the paged key/value cache,
attention of one new token over it, and attention over whole prompts.

``own`` false runs the operators in plain torch, in 32 bits, rounded once at the end; ``own`` true makes
the calls a user makes of colizig_b200.attn.

Shapes.  The cache holds ``k`` and ``v`` as [pages, kv_heads, page_size, head_dim], bf16 or E4M3 with one
f32 multiplier per head.  32 query heads on 4 key/value heads of 128 is this repository's decoder layer;
the others are generic head layouts (one key/value head for all, one for each, groups of 2, 6, 7 and 8).
"""

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
EPS = 1e-6

# (query heads, key/value heads, head size)
HEADS = [(32, 4, 128), (16, 16, 64), (28, 4, 128), (12, 2, 128), (64, 8, 128), (8, 1, 64), (16, 8, 128)]


# ---------------------------------------------------------------- cases


def listed():
    return [
        # one new token of one conversation: what every layer pays per step, all latency
        {"name": "append token", "op": "append", "tokens": 1, "q_heads": 32, "kv_heads": 4, "dim": 128, "rot": 128,
         "page": 64, "kv": "bf16", "x": "f32", "norm": True, "packed": False},
        # one step of a full batch on an 8-bit cache
        {"name": "append batch e4m3", "op": "append", "tokens": 96, "q_heads": 32, "kv_heads": 4, "dim": 128,
         "rot": 128, "page": 64, "kv": "e4m3", "x": "f32", "norm": True, "packed": False},
        # a long prompt, with the packed copies that prompt attention reads
        {"name": "append prompt", "op": "append", "tokens": 8192, "q_heads": 32, "kv_heads": 4, "dim": 128,
         "rot": 128, "page": 64, "kv": "bf16", "x": "f32", "norm": True, "packed": True},
        # a ragged chunk of bf16 projections, partly rotated heads without norms, small pages
        {"name": "append chunk bf16", "op": "append", "tokens": 1531, "q_heads": 16, "kv_heads": 16, "dim": 64,
         "rot": 32, "page": 16, "kv": "bf16", "x": "bf16", "norm": False, "packed": True},
        # the first words of one conversation
        {"name": "decode short", "op": "decode", "batch": 1, "longest": 97, "spread": "same", "q_heads": 32,
         "kv_heads": 4, "dim": 128, "page": 64, "kv": "bf16"},
        # one long conversation: all of the card has to work on four key/value heads
        {"name": "decode long", "op": "decode", "batch": 1, "longest": 32781, "spread": "same", "q_heads": 32,
         "kv_heads": 4, "dim": 128, "page": 64, "kv": "bf16"},
        # a served batch, lengths of every size, an empty one among them, 8-bit cache
        {"name": "decode ragged e4m3", "op": "decode", "batch": 48, "longest": 8190, "spread": "ragged", "q_heads": 32,
         "kv_heads": 4, "dim": 128, "page": 64, "kv": "e4m3"},
        # a full batch of long conversations: the largest cache
        {"name": "decode full batch", "op": "decode", "batch": 96, "longest": 8192, "spread": "near", "q_heads": 32,
         "kv_heads": 4, "dim": 128, "page": 64, "kv": "bf16"},
        # one head each, half-size heads, small pages
        {"name": "decode single heads", "op": "decode", "batch": 13, "longest": 2051, "spread": "ragged",
         "q_heads": 16, "kv_heads": 16, "dim": 64, "page": 16, "kv": "bf16"},
        # one short question
        {"name": "prompt short", "op": "prefill", "batch": 1, "tokens": 77, "before": 0, "q_heads": 32, "kv_heads": 4,
         "dim": 128, "fused": False},
        # prompts of different lengths packed together, read out of the fused projection, keys before the queries
        {"name": "prompts packed", "op": "prefill", "batch": 11, "tokens": 5003, "before": 1200, "q_heads": 28,
         "kv_heads": 4, "dim": 128, "fused": True},
        # one long prompt
        {"name": "prompt long", "op": "prefill", "batch": 1, "tokens": 8192, "before": 0, "q_heads": 32, "kv_heads": 4,
         "dim": 128, "fused": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hk, d = rng.choice(HEADS)
    op = rng.choice(["append", "decode", "prefill"])
    c = {"op": op, "q_heads": hq, "kv_heads": hk, "dim": d}
    if op == "append":
        width = (hq + 2 * hk) * d
        c.update(tokens=_log(rng, 1, 8192 * 5120 // max(width, 5120)), rot=rng.choice([d, d // 2]),
                 page=rng.choice([16, 32, 64, 128]), kv=rng.choice(["bf16", "e4m3"]), x=rng.choice(["f32", "bf16"]),
                 norm=rng.random() < 0.7, packed=rng.random() < 0.4)
    elif op == "decode":
        c.update(batch=_log(rng, 1, 128), spread=rng.choice(["same", "near", "ragged"]),
                 page=rng.choice([16, 32, 64, 128]), kv=rng.choice(["bf16", "e4m3"]))
        # at most the cache (and the padded scores) of the largest listed case
        c["longest"] = _log(rng, 1, min(65536, 96 * 8192 * 4 * 128 // (c["batch"] * hk * d)))
    else:
        c.update(batch=_log(rng, 1, 24), before=rng.choice([0, 0, 1]), fused=rng.random() < 0.5)
        most = int(math.sqrt(8192 * 8192 * 32 * 128 / (hq * d)))
        c["tokens"] = max(c["batch"], _log(rng, 1, min(most, 8192)))
        if c["before"]:
            c["before"] = _log(rng, 1, max(1, 8192 - c["tokens"]))
    return c


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _lengths(case):
    """Tokens in each sequence's cache; the same for every seed, so that cases cost the same."""
    b, longest, spread = case["batch"], case["longest"], case["spread"]
    if spread == "same":
        return [longest] * b
    if spread == "near":  # the last eighth: conversations that filled up together
        return [max(1, longest - (i * 2654435761 % 1000) * longest // 8000) for i in range(b)]
    out = [int(longest * ((i * 2654435761 % 997) / 997.0) ** 2) for i in range(b)]  # many short, few long
    out[0] = longest
    if b > 3:
        out[3] = 0
    return out


def _cuts(total, parts):
    """total split into `parts` uneven whole numbers of at least 1."""
    w = [1 + (i * 2654435761 % 89) for i in range(parts)]
    out = [1 + (total - parts) * x // sum(w) for x in w]
    out[0] += total - sum(out)
    return out


def _cache(case, pages, gen):
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    k = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    ks = vs = None
    if case["kv"] == "e4m3":
        ks = 0.01 + 0.01 * torch.rand(case["kv_heads"], generator=gen, device="cuda")
        vs = 0.01 + 0.01 * torch.rand(case["kv_heads"], generator=gen, device="cuda")
        k = (k * 60).to(E4M3)  # codes well inside the type's range: values of about 1 under these multipliers
        v = (v * 60).to(E4M3)
    return k, v, ks, vs


def _rope(positions, rot):
    """[positions, rot] f32: the cosines of rot/2 angles, then their sines, from 64-bit angles."""
    inv = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _prepare_append(case, gen):
    t, hq, hk, d, page = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    dt = torch.float32 if case["x"] == "f32" else torch.bfloat16
    qkv = torch.randn((t, (hq + 2 * hk) * d), generator=gen, device="cuda", dtype=dt) * 1.5
    pages = -(-t // page) + 3
    k, v, ks, vs = _cache(case, pages, gen)
    s = {"q": qkv[:, : hq * d].unflatten(1, (hq, d)), "k": qkv[:, hq * d: (hq + hk) * d].unflatten(1, (hk, d)),
         "v": qkv[:, (hq + hk) * d:].unflatten(1, (hk, d))}
    first = 5000 % (4 * t + 1)
    s["positions"] = torch.arange(t, device="cuda", dtype=torch.int32) + first
    # the sequence's pages lie anywhere in the cache; every 37th token (a padded one) is not kept
    order = torch.randperm(pages, generator=gen, device="cuda")
    i = torch.arange(t, device="cuda")
    slots = order[i // page] * page + i % page
    s["slots"] = torch.where(i % 37 == 36, torch.full_like(slots, -1), slots)
    s["rope"] = _rope(first + t, case["rot"])
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"] = 1 + 0.2 * torch.randn(d, generator=gen, device="cuda")
        s["k_norm"] = 1 + 0.2 * torch.randn(d, generator=gen, device="cuda")
    s["ck"], s["cv"], s["ks"], s["vs"] = k, v, ks, vs
    return s


def _prepare_decode(case, gen):
    hq, d, page = case["q_heads"], case["dim"], case["page"]
    lens = _lengths(case)
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + 2, max(1, max(need))
    k, v, ks, vs = _cache(case, pages, gen)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    need_t = torch.tensor(need, device="cuda")
    start = torch.cumsum(need_t, 0) - need_t
    at = torch.arange(width, device="cuda")[None, :]
    # rows past a sequence's pages name page 0, as a zeroed table does
    table = torch.where(at < need_t[:, None], order[(start[:, None] + at).clamp(max=pages - 1)],
                        torch.zeros((), dtype=torch.int32, device="cuda")).contiguous()
    q = torch.randn((case["batch"], hq, d), generator=gen, device="cuda", dtype=torch.bfloat16) * 2
    return {"q": q, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "ck": k, "cv": v,
            "ks": ks, "vs": vs, "scale": d ** -0.5}


def _prepare_prefill(case, gen):
    hq, hk, d, t, before = case["q_heads"], case["kv_heads"], case["dim"], case["tokens"], case["before"]
    nq = _cuts(t, case["batch"])
    nk = [n + (before if i % 3 == 0 else 0) * (i + 1) // case["batch"] for i, n in enumerate(nq)]
    s = {"scale": d ** -0.5}
    if case["fused"] and nk == nq:  # q, k, v as columns of one projection
        qkv = torch.randn((t, (hq + 2 * hk) * d), generator=gen, device="cuda", dtype=torch.bfloat16)
        s["q"] = qkv[:, : hq * d].unflatten(1, (hq, d))
        s["k"] = qkv[:, hq * d: (hq + hk) * d].unflatten(1, (hk, d))
        s["v"] = qkv[:, (hq + hk) * d:].unflatten(1, (hk, d))
    elif case["fused"]:  # k and v as columns of one buffer (keys of earlier chunks in it)
        kv = torch.randn((sum(nk), 2 * hk * d), generator=gen, device="cuda", dtype=torch.bfloat16)
        s["q"] = torch.randn((t, hq, d), generator=gen, device="cuda", dtype=torch.bfloat16)
        s["k"] = kv[:, : hk * d].unflatten(1, (hk, d))
        s["v"] = kv[:, hk * d:].unflatten(1, (hk, d))
    else:
        s["q"] = torch.randn((t, hq, d), generator=gen, device="cuda", dtype=torch.bfloat16)
        s["k"] = torch.randn((sum(nk), hk, d), generator=gen, device="cuda", dtype=torch.bfloat16)
        s["v"] = torch.randn((sum(nk), hk, d), generator=gen, device="cuda", dtype=torch.bfloat16)
    s["q"] *= 2
    zero = torch.zeros(1, dtype=torch.int64)
    s["cu_q"] = torch.cat([zero, torch.tensor(nq).cumsum(0)]).to("cuda", torch.int32)
    s["cu_k"] = torch.cat([zero, torch.tensor(nk).cumsum(0)]).to("cuda", torch.int32)
    return s


def prepare(case, seed):
    gen = _gen(seed)
    s = {"append": _prepare_append, "decode": _prepare_decode, "prefill": _prepare_prefill}[case["op"]](case, gen)
    s["case"] = dict(case)
    if own:
        from colizig_b200 import attn, gpu

        if not gpu.available():
            gpu.init()
        if case["op"] != "prefill":
            s["cache"] = attn.KvCache(s["ck"], s["cv"], k_scale=s["ks"], v_scale=s["vs"])
        if case["op"] == "decode":
            s["plan"] = attn.DecodePlan(s["cache"], case["q_heads"], case["batch"], scale=s["scale"])
    return s


# ---------------------------------------------------------------- plain forms


def _normed_rotated(x, w, cs, rot):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    h = rot // 2
    c, s = cs[:, None, :h], cs[:, None, h:]
    a, b = x[..., :h], x[..., h:rot]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)


def _store(cache, scale, x, page, row):
    if scale is not None:
        code = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
        cache.view(torch.uint8)[page, :, row] = code.view(torch.uint8)
    else:
        cache[page, :, row] = x.to(torch.bfloat16)


def _plain_append(s):
    case = s["case"]
    cs = s["rope"][s["positions"]]
    q = _normed_rotated(s["q"], s["q_norm"], cs, case["rot"]).to(torch.bfloat16)
    k = _normed_rotated(s["k"], s["k_norm"], cs, case["rot"])
    v = s["v"].float()
    kept = s["slots"] >= 0
    slots = s["slots"][kept]
    page, row = slots // case["page"], slots % case["page"]
    _store(s["ck"], s["ks"], k[kept], page, row)
    _store(s["cv"], s["vs"], v[kept], page, row)
    out = {"q": q, "cache_k": s["ck"], "cache_v": s["cv"]}
    if case["packed"]:
        out["k"], out["v"] = k.to(torch.bfloat16), v.to(torch.bfloat16)
    return out


def _gathered(cache, scale, table, hk, d):
    """[batch, kv_heads, table width * page, d] f32: each sequence's cached rows in order."""
    if scale is not None:
        x = cache.view(torch.uint8)[table].view(E4M3).float() * scale[:, None, None]
    else:
        x = cache[table].float()
    return x.transpose(1, 2).reshape(table.shape[0], hk, -1, d)


def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v over the keys that `seen` allows; 0 where it allows none."""
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v)
    return torch.where(total > 0, o / total, torch.zeros_like(o))


def _plain_decode(s):
    case = s["case"]
    b, hq, hk, d = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
    table = s["table"].long()
    k = _gathered(s["ck"], s["ks"], table, hk, d)
    v = _gathered(s["cv"], s["vs"], table, hk, d)
    seen = torch.arange(k.shape[2], device="cuda")[None, :] < s["lens"][:, None]
    o = _attend(s["q"].float().view(b, hk, hq // hk, d), k, v, seen[:, None, None, :], s["scale"])
    return o.reshape(b, hq, d).to(torch.bfloat16)


def _plain_prefill(s):
    case = s["case"]
    t, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
    nk = s["k"].shape[0]
    cq, ck = s["cu_q"].long(), s["cu_k"].long()
    iq, ik = torch.arange(t, device="cuda"), torch.arange(nk, device="cuda")
    bq, bk = torch.bucketize(iq, cq[1:], right=True), torch.bucketize(ik, ck[1:], right=True)
    # places counted from the end of the sequence: a query sees keys that are not nearer to the end than itself
    seen = (bq[:, None] == bk[None, :]) & ((cq[bq + 1] - iq)[:, None] <= (ck[bk + 1] - ik)[None, :])
    q = s["q"].float().view(t, hk, hq // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
    k, v = s["k"].float().transpose(0, 1), s["v"].float().transpose(0, 1)
    o = _attend(q, k, v, seen.repeat(hq // hk, 1), s["scale"])
    return o.view(hk, hq // hk, t, d).permute(2, 0, 1, 3).reshape(t, hq, d).to(torch.bfloat16)


# ---------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill}[case["op"]](state)
    from colizig_b200 import attn

    if case["op"] == "decode":
        return state["plan"].run(state["q"], state["table"], state["lens"])
    if case["op"] == "prefill":
        return attn.prefill(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"], scale=state["scale"])
    q, k, v = attn.append(state["cache"], state["q"], state["k"], state["v"], state["positions"], state["slots"],
                          state["rope"], q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS,
                          packed=case["packed"])
    out = {"q": q, "cache_k": state["ck"], "cache_v": state["cv"]}
    if case["packed"]:
        out["k"], out["v"] = k, v
    return out


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        t, w = case["tokens"], (hq + 2 * hk) * d
        kept = t - t // 37
        one = 2 if case["kv"] == "bf16" else 1
        n = t * w * (4 if case["x"] == "f32" else 2) + t * (4 + 8) + t * case["rot"] * 4
        n += t * hq * d * 2 + kept * 2 * hk * d * one + (t * 2 * hk * d * 2 if case["packed"] else 0)
        return {"bytes": n, "flops": t * (hq + hk) * (4 * d + 3 * case["rot"])}
    if case["op"] == "decode":
        lens = _lengths(case)
        one = 2 if case["kv"] == "bf16" else 1
        tokens = sum(lens)
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": tokens * 2 * hk * d * one + pages * 4 + len(lens) * (4 + 2 * hq * d * 2),
                "flops": 4 * tokens * hq * d}
    nq = _cuts(case["tokens"], case["batch"])
    nk = [n + (case["before"] if i % 3 == 0 else 0) * (i + 1) // case["batch"] for i, n in enumerate(nq)]
    pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(nq, nk))
    return {"bytes": 2 * d * (2 * case["tokens"] * hq + 2 * sum(nk) * hk), "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------- the definitions in 64 bits


def _exact_append(case, s):
    d, rot, page = case["dim"], case["rot"], case["page"]

    def heads(x, w):
        y = x.double().clone()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        z = y.clone()
        for i in range(rot // 2):  # pair (i, i + rot/2) turned by its angle
            c, sn = (s["rope"][s["positions"].long()][:, j].double()[:, None] for j in (i, i + rot // 2))
            z[..., i] = y[..., i] * c - y[..., i + rot // 2] * sn
            z[..., i + rot // 2] = y[..., i] * sn + y[..., i + rot // 2] * c
        return z

    q, k, v = heads(s["q"], s["q_norm"]), heads(s["k"], s["k_norm"]), s["v"].double()
    out = {"q": q}
    for name, cache, scale, x in (("cache_k", s["ck"], s["ks"], k), ("cache_v", s["cv"], s["vs"], v)):
        full = cache.double()
        flat = full.transpose(1, 2).reshape(-1, case["kv_heads"], d)
        val = x if scale is None else (x / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        keep = (s["slots"] >= 0).nonzero()[:, 0]
        flat[s["slots"][keep]] = val[keep]
        out[name] = flat.view(-1, page, case["kv_heads"], d).transpose(1, 2)
    if case["packed"]:
        out["k"], out["v"] = k, v
    return out


def _exact_rows(q, k, v, scale, allowed):
    w = (q @ k.mT) * scale
    w[~allowed.expand_as(w)] = -math.inf
    return torch.softmax(w, -1) @ v


def _exact_decode(case, s):
    hq, hk, d, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(case["batch"], hq, d, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        rows = s["table"][b, : -(-n // page)].long()
        kv = []
        for cache, scale in ((s["ck"], s["ks"]), (s["cv"], s["vs"])):
            x = cache.view(torch.uint8)[rows].view(E4M3) if scale is not None else cache[rows]
            x = x.double() * (1.0 if scale is None else scale.double()[:, None, None])
            kv.append(x.transpose(0, 1).reshape(hk, -1, d)[:, :n])
        every = torch.ones(1, n, dtype=torch.bool, device="cuda")
        out[b] = _exact_rows(s["q"][b].double().view(hk, hq // hk, d), kv[0], kv[1], s["scale"], every).view(hq, d)
    return out


def _exact_prefill(case, s):
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(case["tokens"], hq, d, dtype=torch.float64, device="cuda")
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b in range(case["batch"]):
        q, k, v = s["q"][cq[b]:cq[b + 1]], s["k"][ck[b]:ck[b + 1]], s["v"][ck[b]:ck[b + 1]]
        nq, nk = q.shape[0], k.shape[0]
        allowed = torch.ones(nq, nk, dtype=torch.bool, device="cuda").tril(nk - nq)
        for h in range(hq):
            out[cq[b]:cq[b + 1], h] = _exact_rows(q[:, h].double(), k[:, h * hk // hq].double(),
                                                  v[:, h * hk // hq].double(), s["scale"], allowed)
    return out


def exact(case, seed):
    gen = _gen(seed)
    if case["op"] == "append":
        return _exact_append(case, _prepare_append(case, gen))
    if case["op"] == "decode":
        return _exact_decode(case, _prepare_decode(case, gen))
    return _exact_prefill(case, _prepare_prefill(case, gen))
