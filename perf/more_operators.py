"""What the operators of serving several requests over a paged cache are measured on.

A step takes new tokens of many requests (one each, a chain of drafts, or a
chunk of a prompt).  The operators: step (block tables and slot maps from the
requests' lengths), append (per-head q/k norm, rotation, rows into pages),
attention (every new token over its request's pages), verify (drafted tokens
against the target's probabilities, from given random numbers).  ``run``
computes them in plain torch, or -- ``own`` -- through odiengine_b200.paged.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # block tables of a few requests, one token each: the smallest, latency counts
        {"name": "step 8", "op": "step", "requests": 8, "page": 16, "most": 4096, "new_lo": 1, "new_hi": 1, "mix": 1},
        # a full server: chains of drafts, prompts' chunks and idle places in one step
        {"name": "step 512", "op": "step", "requests": 512, "page": 16, "most": 4096, "new_lo": 0, "new_hi": 61, "mix": 2},
        # one token of each of 8 requests, 32 heads over 8, normed q and k
        {"name": "append 8x1 f16 32/8", "op": "append", "requests": 8, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "dtype": "f16", "page": 16, "past_lo": 100, "past_hi": 4000, "new_lo": 1, "new_hi": 1, "theta": 10000.0,
         "norm": True, "mix": 3},
        # chunks of prompts, about 4096 tokens in all, far positions, the 64/8-head shape
        {"name": "append 5x~820 bf16 64/8", "op": "append", "requests": 5, "heads": 64, "kv_heads": 8, "head_dim": 128,
         "dtype": "bf16", "page": 64, "past_lo": 90000, "past_hi": 100003, "new_lo": 600, "new_hi": 1040,
         "theta": 500000.0, "norm": False, "mix": 4},
        # one request, one token, 32 heads each with its own keys, short context
        {"name": "attention 1x1 f16 32/32 518", "op": "attention", "requests": 1, "heads": 32, "kv_heads": 32,
         "head_dim": 128, "dtype": "f16", "page": 16, "past_lo": 517, "past_hi": 517, "new_lo": 1, "new_hi": 1,
         "cap": 0.0, "bias": False, "prefix": False, "mix": 5},
        # a batch of decoding requests of ragged lengths
        {"name": "attention 64x1 bf16 64/8", "op": "attention", "requests": 64, "heads": 64, "kv_heads": 8,
         "head_dim": 128, "dtype": "bf16", "page": 64, "past_lo": 300, "past_hi": 8100, "new_lo": 1, "new_hi": 1,
         "cap": 0.0, "bias": False, "prefix": False, "mix": 6},
        # chains of drafts of several requests, capped scores
        {"name": "attention 16x2-5 f16 32/8 cap", "op": "attention", "requests": 16, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "dtype": "f16", "page": 16, "past_lo": 500, "past_hi": 6000, "new_lo": 2, "new_hi": 5,
         "cap": 50.0, "bias": False, "prefix": False, "mix": 7},
        # whole prompts of odd lengths, distance bias, part of each visible both ways
        {"name": "attention 7x~700 f16 32/32 hd64 bias prefix", "op": "attention", "requests": 7, "heads": 32,
         "kv_heads": 32, "head_dim": 64, "dtype": "f16", "page": 32, "past_lo": 0, "past_hi": 0, "new_lo": 333,
         "new_hi": 1201, "cap": 0.0, "bias": True, "prefix": True, "mix": 8},
        # a chunk of a long prompt over what is in the cache: the most arithmetic
        {"name": "attention 1x2048 bf16 64/8 over 14001", "op": "attention", "requests": 1, "heads": 64, "kv_heads": 8,
         "head_dim": 128, "dtype": "bf16", "page": 64, "past_lo": 14001, "past_hi": 14001, "new_lo": 2048,
         "new_hi": 2048, "cap": 0.0, "bias": False, "prefix": False, "mix": 9},
        # the drafts of one request, a greedy drafter, vocabulary of 32000
        {"name": "verify 1x5 32000", "op": "verify", "requests": 1, "drafts_lo": 4, "drafts_hi": 4, "vocab": 32000,
         "temperature": 0.8, "probs": False, "mix": 10},
        # the drafts of 16 requests with the drafter's probabilities, large odd vocabulary
        {"name": "verify 16x~5 128259", "op": "verify", "requests": 16, "drafts_lo": 0, "drafts_hi": 7, "vocab": 128259,
         "temperature": 1.0, "probs": True, "mix": 11},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "append", "attention", "attention", "attention", "attention", "verify", "verify"])
    c = {"op": op, "mix": rng.randrange(1 << 30)}
    if op == "step":
        hi = _log(rng, 1, 61)
        return {**c, "requests": _log(rng, 1, 512), "page": rng.choice([16, 32, 64, 128]), "most": _log(rng, 64, 4096),
                "new_lo": rng.choice([0, 1, hi]), "new_hi": hi}
    if op == "verify":
        V = _log(rng, 100, 128259)
        hi = rng.randint(0, 7)
        return {**c, "requests": _log(rng, 1, 16), "drafts_lo": rng.randint(0, hi), "drafts_hi": hi, "vocab": V,
                "temperature": rng.choice([0.3, 0.8, 1.0, 1.7]), "probs": rng.random() < 0.5}
    kv = rng.choice([1, 2, 4, 8, 8, 16, 32])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8) if kv * g <= 64])
    c |= {"heads": heads, "kv_heads": kv, "head_dim": rng.choice([64, 128, 128]), "dtype": rng.choice(["f16", "bf16"]),
          "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        rows = _log(rng, 1, 4000)
        B = _log(rng, 1, min(rows, 64))
        n = max(1, rows // B)
        past = _log(rng, 1, 100003) - 1
        return {**c, "requests": B, "past_lo": past // 2, "past_hi": past, "new_lo": max(1, n // 2), "new_hi": n,
                "theta": rng.choice([10000.0, 500000.0]), "norm": rng.random() < 0.5}
    kind = rng.choice(["decode", "drafts", "chunk"])
    if kind == "chunk":
        n, B = _log(rng, 9, 2048), _log(rng, 1, 8)
        n = max(1, n // B)
    else:
        B = _log(rng, 1, 64)
        n = 1 if kind == "decode" else rng.randint(2, 8)
    # what the longest listed batch holds in its pages, and what the largest listed chunk multiplies
    most = min(131000, 8 * 64 * 8100 // (kv * B), 2048 * 64 * 15000 // (heads * B * n))
    past = _log(rng, 1, max(1, most)) - 1
    return {**c, "requests": B, "past_lo": past // rng.choice([1, 2, 20]), "past_hi": past, "new_lo": max(1, n // 2),
            "new_hi": n, "cap": rng.choice([0.0, 0.0, 30.0]), "bias": rng.random() < 0.3, "prefix": rng.random() < 0.2}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _lengths(c):
    """(past, new) of each request; they belong to the case, not to the seed."""
    r = random.Random(c["mix"])
    if c["op"] == "step":
        past, new = [], []
        for _ in range(c["requests"]):
            total = 0 if c["requests"] > 8 and r.random() < 0.1 else r.randint(1, c["most"])  # some places are idle
            n = min(total, r.randint(c["new_lo"], c["new_hi"]))
            past.append(total - n)
            new.append(n)
        return past, new
    if c["op"] == "verify":
        return None, [1 + r.randint(c["drafts_lo"], c["drafts_hi"]) for _ in range(c["requests"])]
    past = [r.randint(c["past_lo"], c["past_hi"]) for _ in range(c["requests"])]
    return past, [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["requests"])]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def _tables(s, c, g, past, new, P, spare):
    """Every request's pages, scattered over the pool, and the free rest; the
    pages of the new tokens are there from the step before, whose drafts the
    next step drops."""
    B = len(new)
    count = [-(-(a + b) // P) for a, b in zip(past, new)]
    used = sum(count)
    pages = used + spare
    perm = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    wide = max(1, max(count))
    j = torch.arange(wide, device=DEV)
    held = j < _ints(count)[:, None]
    s["table"] = torch.full((B, wide), -1, dtype=torch.int32, device=DEV)
    s["table"][held] = perm[:used]
    s["lens"] = _ints([a + b for a, b in zip(past, new)])
    s["free"] = torch.zeros(pages, dtype=torch.int32, device=DEV)
    s["free"][:spare] = perm[used:]
    s["free_count"] = _ints([spare])
    s["keep"], s["new"] = _ints(past), _ints(new)
    s["pages"] = pages


def prepare(case, seed):
    c = dict(case)
    op = c["op"]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"c": c}
    past, new = _lengths(c)
    rows, B = sum(new), len(new)
    if op == "verify":
        V = c["vocab"]
        s["logits"] = _randn(g, rows, V, std=3.0)
        draft = s["logits"] + _randn(g, rows, V, std=1.0)  # a drafter that often agrees
        if c["probs"]:
            s["probs"] = torch.softmax(draft, -1)
            chosen = torch.multinomial(s["probs"], 1, generator=g)[:, 0]
        else:
            s["probs"], chosen = None, draft.argmax(-1)
        s["tokens"] = chosen.roll(1).to(torch.int32)  # row r's choice is the token of row r + 1
        s["starts"] = _ints(np.concatenate([[0], np.cumsum(new)]).tolist())
        s["u_accept"] = torch.rand(rows, device=DEV, generator=g)
        s["u_next"] = torch.rand(B, device=DEV, generator=g)
        s["accepted"] = torch.empty(B, dtype=torch.int32, device=DEV)
        s["next"] = torch.empty_like(s["accepted"])
    else:
        P = c["page"]
        _tables(s, c, g, past, new, P, 7 + B)
        s["rows"] = rows
        if op == "step":
            heads = kv = 8
            s["most_new"] = max(1, c["new_hi"])
            s["starts"] = torch.empty(B + 1, dtype=torch.int32, device=DEV)
        else:
            heads, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
            dt = torch.float16 if c["dtype"] == "f16" else torch.bfloat16
            s["most_new"] = max(new)
            s["longest"] = max(a + b for a, b in zip(past, new))
            # the whole pool, pages that no request holds included
            s["k"] = _randn(g, s["pages"], kv, P, hd, dtype=dt)
            s["v"] = _randn(g, s["pages"], kv, P, hd, dtype=dt)
            s["row_request"] = torch.repeat_interleave(torch.arange(B, device=DEV), s["new"].long())
            s["row_offset"] = torch.arange(rows, device=DEV) - torch.repeat_interleave(
                (torch.cumsum(s["new"], 0) - s["new"]).long(), s["new"].long())
            s["positions"] = s["keep"].long()[s["row_request"]] + s["row_offset"]
            s["q"] = torch.empty((rows, heads * hd), dtype=dt, device=DEV)
        if op == "append":
            s["qkv"] = _randn(g, rows, (heads + 2 * kv) * hd, std=1.5)
            s["q_norm"] = 1.0 + _randn(g, hd, std=0.1) if c["norm"] else None
            s["k_norm"] = 1.0 + _randn(g, hd, std=0.1) if c["norm"] else None
        if op == "attention":
            s["q"].normal_(0.0, 1.7, generator=g)
            s["out"] = torch.empty_like(s["q"])
            # 2^(-8 h / heads), the usual fall of distance biases
            s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, heads + 1, device=DEV) / heads)).float() if c["bias"] else None
            s["prefix"] = (s["lens"] // 3) if c["prefix"] else None
    if own:  # the handles that a program keeps
        from odiengine_b200 import paged

        if op == "verify":
            s["scratch"] = paged.verify_scratch(rows, B, c["vocab"])
        else:
            s["tables"] = paged.PageTables(s["table"], s["lens"], s["free"], s["free_count"], P)
            s["batch"] = paged.PagedBatch(s["tables"], max_rows=max(1, rows), max_new=s["most_new"], heads=heads, kv_heads=kv)
            if op != "step":
                s["cache"] = paged.PagedCache(s["k"], s["v"])
                paged.paged_step(s["tables"], s["batch"], s["new"], keep=s["keep"], prefix=s.get("prefix"))
                s["scratch"] = paged.attention_paged_scratch(s["cache"], s["batch"])
    return s


# ---- one pass --------------------------------------------------------------------------------------------------

def run(s):
    c = s["c"]
    if own:
        return _OWN[c["op"]](s, c)
    return _PLAIN[c["op"]](s, c)


def _own_step(s, c):
    from odiengine_b200 import paged

    b = s["batch"]
    paged.paged_step(s["tables"], b, s["new"], keep=s["keep"])
    return s["table"], s["lens"], s["free"], s["free_count"], b.starts, b.positions[:s["rows"]], b.slots[:s["rows"]]


def _own_append(s, c):
    from odiengine_b200 import paged

    paged.qk_rope_append_paged(s["qkv"], s["cache"], s["batch"], s["q"], heads=c["heads"], theta=c["theta"],
                               q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    return s["q"], s["k"], s["v"]


def _own_attention(s, c):
    from odiengine_b200 import paged

    return paged.attention_paged(s["q"], s["cache"], s["tables"], s["batch"], s["out"],
                                 scale=1.0 / math.sqrt(c["head_dim"]), softcap=c["cap"], slopes=s["slopes"],
                                 scratch=s["scratch"])


def _own_verify(s, c):
    from odiengine_b200 import paged

    return paged.verify_sampled(s["logits"], s["tokens"], s["starts"], s["u_accept"], s["u_next"], s["accepted"], s["next"],
                                temperature=c["temperature"], draft_probs=s["probs"], scratch=s["scratch"])


_OWN = {"step": _own_step, "append": _own_append, "attention": _own_attention, "verify": _own_verify}


def _plain_step(s, c):
    P, table, n = c["page"], s["table"], s["free_count"]
    B, wide = table.shape
    had, kept = (s["lens"] + P - 1) // P, (s["keep"] + P - 1) // P
    wants = (s["keep"] + s["new"] + P - 1) // P
    j = torch.arange(wide, device=DEV)
    drop = (j >= kept[:, None]) & (j < had[:, None])
    take = (j >= kept[:, None]) & (j < wants[:, None])
    # dropped pages go on the free list so that the first dropped is the first taken again
    order = torch.cumsum(drop.flatten().int(), 0, dtype=torch.int32).view(B, wide)
    dropped = order[-1, -1]
    at = torch.where(drop, n + dropped - order, len(s["free"]))
    free = torch.cat([s["free"], s["free"][:1]])
    free[at.long()] = table
    n = n + dropped
    rank = torch.cumsum(take.flatten().int(), 0, dtype=torch.int32).view(B, wide)
    got = free[(n - rank).clamp_(min=0).long()]
    table.copy_(torch.where(take, got, torch.where(drop, -1, table)))
    s["free"].copy_(free[:-1])
    s["free_count"].copy_(n - rank[-1, -1])
    s["lens"].copy_(s["keep"] + s["new"])
    ends = torch.cumsum(s["new"], 0, dtype=torch.int32)
    s["starts"][:1] = 0
    s["starts"][1:] = ends
    r = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(ends, r, right=True)
    pos = (s["keep"][b] + (r - (ends - s["new"])[b])).int()
    return (table, s["lens"], s["free"], s["free_count"], s["starts"], pos,
            (table[b, (pos // P).long()] * P + pos % P).int())


def _plain_append(s, c):
    H, kv, hd, P, T = c["heads"], c["kv_heads"], c["head_dim"], c["page"], s["rows"]
    x = s["qkv"].view(T, H + 2 * kv, hd)
    q, k, v = x[:, :H], x[:, H:H + kv], x[:, H + kv:]
    if c["norm"]:
        q = q / torch.sqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    # far positions need 64 bits before the sine
    i = torch.arange(hd // 2, dtype=torch.float64, device=DEV)
    a = s["positions"].double()[:, None] * torch.pow(c["theta"], -2.0 * i / hd)
    cs, sn = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]

    def turn(u):
        a, b = u[..., :hd // 2], u[..., hd // 2:]
        return torch.cat([a * cs - b * sn, a * sn + b * cs], -1)

    page = s["table"][s["row_request"], s["positions"] // P].long()
    s["k"][page, :, s["positions"] % P] = turn(k).to(s["k"].dtype)
    s["v"][page, :, s["positions"] % P] = v.to(s["v"].dtype)
    s["q"].copy_(turn(q).reshape(T, H * hd))
    return s["q"], s["k"], s["v"]


def _plain_attention(s, c):
    """All requests at once, padded to the longest."""
    H, kv, hd, P, T = c["heads"], c["kv_heads"], c["head_dim"], c["page"], s["rows"]
    B, G, N = len(s["new"]), H // kv, s["most_new"]
    pages = s["table"][:, :-(-s["longest"] // P)].clamp(min=0).long()
    L = pages.shape[1] * P

    def rows(pool):
        return pool[pages].transpose(1, 2).reshape(B, kv, L, hd).float()

    at = (s["row_request"] * N + s["row_offset"])
    x = torch.zeros((B * N, kv, G, hd), dtype=torch.float32, device=DEV)
    x[at] = s["q"].view(T, kv, G, hd).float()
    x = x.view(B, N, kv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, kv, N * G, hd)
    p = torch.matmul(x, rows(s["k"]).transpose(2, 3)).view(B, kv, N, G, L)
    p *= 1.0 / math.sqrt(hd)
    if c["cap"]:
        p = c["cap"] * torch.tanh(p / c["cap"])
    j = torch.arange(L, device=DEV)
    i = s["keep"][:, None] + torch.arange(N, device=DEV)  # [B, N]
    if c["bias"]:
        away = (i[:, :, None] - j).abs().float()
        p -= s["slopes"].view(kv, 1, G, 1) * away[:, None, :, None]
    most = i + 1 if s["prefix"] is None else torch.maximum(i + 1, s["prefix"][:, None])
    most = torch.minimum(most, s["lens"][:, None])
    p.masked_fill_((j >= most[:, :, None])[:, None, :, None], -math.inf)
    p -= p.amax(-1, keepdim=True)
    p.exp_()
    o = torch.matmul(p.view(B, kv, N * G, L), rows(s["v"])) / p.sum(-1).view(B, kv, N * G, 1)
    o = o.view(B, kv, N, G, hd).permute(0, 2, 1, 3, 4).reshape(B * N, H * hd)
    return o[at].to(s["q"].dtype)


def _plain_verify(s, c):
    """In 64 bits: a decision next to its border has to fall the same way."""
    V, starts = c["vocab"], s["starts"].long()
    R, B = len(s["tokens"]), len(starts) - 1
    p = s["logits"].double()
    p = torch.exp((p - p.amax(-1, keepdim=True)) / c["temperature"])
    p /= p.sum(-1, keepdim=True)
    r = torch.arange(R, device=DEV)
    seq = torch.searchsorted(starts[1:], r, right=True)
    draft = s["tokens"].long().roll(-1)[:, None]  # what row r is followed by
    last = r == starts[1:][seq] - 1
    px = p.gather(1, draft)[:, 0]
    qx = torch.ones_like(px) if s["probs"] is None else s["probs"].gather(1, draft)[:, 0].double()
    stop = last | ~(s["u_accept"].double() * qx < px)
    at = torch.full((B,), R, device=DEV).scatter_reduce_(0, seq, torch.where(stop, r, R), "amin")  # the first row that stops
    w = p[at]
    whole = last[at][:, None]
    if s["probs"] is None:
        q = torch.zeros_like(w).scatter_(1, draft[at], 1.0)
    else:
        q = s["probs"][at].double()
    rest = (w - q).clamp_(min=0)
    w = torch.where(whole | (rest.sum(-1, keepdim=True) <= 0), w, rest)
    sums = w.cumsum(-1)
    first = sums > s["u_next"].double()[:, None] * sums[:, -1:]
    token = torch.where(first, torch.arange(V, device=DEV), V).amin(-1)
    return (at - starts[:-1]).int(), token.int()


_PLAIN = {"step": _plain_step, "append": _plain_append, "attention": _plain_attention, "verify": _plain_verify}


# ---- 64 bits ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    if op in ("step", "verify"):
        return None  # whole numbers
    s = prepare(case, seed)
    c = s["c"]
    past, new = _lengths(c)
    H, kv, hd, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    G = H // kv
    table = s["table"].cpu().tolist()
    if op == "append":
        half = hd // 2
        x = s["qkv"].double().view(-1, H + 2 * kv, hd)
        where = [(table[b][(past[b] + j) // P], (past[b] + j) % P) for b in range(len(new)) for j in range(new[b])]
        page = torch.tensor([a for a, _ in where], device=DEV)
        off = torch.tensor([b for _, b in where], device=DEV)
        pos = torch.tensor([past[b] + j for b in range(len(new)) for j in range(new[b])], dtype=torch.float64, device=DEV)
        f = torch.tensor([c["theta"] ** (-2.0 * i / hd) for i in range(half)], dtype=torch.float64, device=DEV)
        z = torch.polar(torch.ones((len(pos), half), dtype=torch.float64, device=DEV), pos[:, None] * f)[:, None]

        def one(u, w):
            if w is not None:
                u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * w.double()
            r = torch.complex(u[..., :half].contiguous(), u[..., half:].contiguous()) * z
            return torch.cat([r.real, r.imag], -1)

        k, v = s["k"].double(), s["v"].double()
        k[page, :, off] = one(x[:, H:H + kv], s["k_norm"])
        v[page, :, off] = x[:, H + kv:]
        return one(x[:, :H], s["q_norm"]).reshape(-1, H * hd), k, v
    out, row = [], 0
    for b in range(len(new)):
        n, N = past[b] + new[b], new[b]
        pages = torch.tensor(table[b][:-(-n // P)], device=DEV)
        k = s["k"][pages].transpose(0, 1).reshape(kv, -1, hd)[:, :n]
        v = s["v"][pages].transpose(0, 1).reshape(kv, -1, hd)[:, :n]
        q = s["q"][row:row + N].view(N, kv, G, hd)
        o = torch.empty((N, kv, G, hd), dtype=torch.float64, device=DEV)
        j = torch.arange(n, device=DEV)
        i = torch.arange(past[b], n, device=DEV)
        limit = i + 1 if not c["prefix"] else torch.clamp(i + 1, min=n // 3)
        hide = j[None, :] >= limit[:, None]
        for h in range(kv):
            for a in range(G):
                w = (q[:, h, a].double() @ k[h].double().T) / math.sqrt(hd)
                if c["cap"]:
                    w = torch.tanh(w / c["cap"]) * c["cap"]
                if c["bias"]:
                    w = w - s["slopes"][h * G + a].double() * (i[:, None] - j[None, :]).abs()
                o[:, h, a] = torch.softmax(w.masked_fill(hide, -math.inf), -1) @ v[h].double()
        out.append(o.reshape(N, H * hd))
        row += N
    return torch.cat(out)


def work(case):
    c = case
    past, new = _lengths(c)
    rows, B = sum(new), len(new)
    if c["op"] == "verify":
        drafts = rows - B
        return {"bytes": 4 * c["vocab"] * (rows + (drafts if c["probs"] else 0)) + 4 * (2 * rows + 4 * B),
                "flops": 10 * rows * c["vocab"]}
    if c["op"] == "step":
        P = c["page"]
        pages = sum(-(-(a + n) // P) - -(-a // P) for a, n in zip(past, new))
        return {"bytes": 4 * (5 * B + 4 * pages + 2 * rows), "flops": 10 * rows}
    H, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "append":
        return {"bytes": 6 * rows * (H + 2 * kv) * hd, "flops": 6 * rows * (H + kv) * hd}
    held = sum(past) + rows
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(past, new))
    return {"bytes": 4 * held * kv * hd + 4 * rows * H * hd, "flops": 4 * H * hd * pairs}
