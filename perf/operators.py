"""What the operators of drafted-token verification are measured on.

A verification step checks T drafted tokens (a chain or a tree) in one pass
over a KV cache.  The operators: append (per-head q/k norm, rotation, cache
write), attention (a tree of queries over the cache), logits (penalties,
biases, masks, greedy token), read and move (cache rows out, accepted rows
into place).  ``run`` computes them in plain torch, or -- ``own`` -- through
odiengine_b200.draft.
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
        # one new token of a grouped-query model (32 heads over 8), int8 cache: the smallest, latency counts
        {"name": "append 1 i8 32/8", "op": "append", "cache": "i8", "tokens": 1, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "ctx": 4096, "pos": 2047, "theta": 10000.0, "norm": True},
        # a chunk of a prompt at a far position, the 64/8-head shape, fp16 cache
        {"name": "append 512 f16 64/8", "op": "append", "cache": "f16", "tokens": 512, "heads": 64, "kv_heads": 8,
         "head_dim": 128, "ctx": 131072, "pos": 100003, "theta": 500000.0, "norm": False},
        # a short odd range of a small cache read back as fp32
        {"name": "read 77 f32", "op": "read", "cache": "i8", "kv_heads": 8, "head_dim": 64, "ctx": 512,
         "start": 131, "count": 77, "out": "f32"},
        # a whole long int8 prefix handed on as fp16
        {"name": "read 32001 f16", "op": "read", "cache": "i8", "kv_heads": 8, "head_dim": 128, "ctx": 32768,
         "start": 5, "count": 32001, "out": "f16"},
        # the accepted path of a small tree, one layer
        {"name": "move 5 of 16 f16", "op": "move", "cache": "f16", "kv_heads": 8, "head_dim": 128, "ctx": 4096,
         "pos": 1001, "nodes": 16, "keep": 5},
        # a long accepted chain in a cache of all heads
        {"name": "move 100 of 256 i8", "op": "move", "cache": "i8", "kv_heads": 32, "head_dim": 128, "ctx": 4096,
         "pos": 2500, "nodes": 256, "keep": 100},
        # single-token form, 32 heads each with its own keys, short context
        {"name": "attention 1 f16 32/32 518", "op": "attention", "cache": "f16", "tokens": 1, "heads": 32,
         "kv_heads": 32, "head_dim": 128, "ctx": 4096, "past": 517},
        # an ordinary drafted tree over an ordinary context
        {"name": "attention 13 f16 32/8 4014", "op": "attention", "cache": "f16", "tokens": 13, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "ctx": 8192, "past": 4001},
        # single-token form over a very long int8 cache
        {"name": "attention 1 i8 64/8 131001", "op": "attention", "cache": "i8", "tokens": 1, "heads": 64,
         "kv_heads": 8, "head_dim": 128, "ctx": 131072, "past": 131000},
        # a large tree over a long int8 cache: the most arithmetic
        {"name": "attention 64 i8 64/8 32641", "op": "attention", "cache": "i8", "tokens": 64, "heads": 64,
         "kv_heads": 8, "head_dim": 128, "ctx": 32768, "past": 32577},
        # one row of a 32000-token vocabulary, penalties and a mask: latency
        {"name": "logits 1 32000", "op": "logits", "rows": 1, "vocab": 32000, "history": 64, "bias": 7,
         "mask": "shared"},
        # every node of a large tree over a large odd vocabulary, a mask of its own for each node
        {"name": "logits 64 128259", "op": "logits", "rows": 64, "vocab": 128259, "history": 1000, "bias": 300,
         "mask": "rows"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "move", "attention", "attention", "attention", "logits", "logits"])
    cache = rng.choice(["f16", "i8"])
    hd = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 8, 16, 32])
    if op == "append":
        heads = kv * rng.choice([g for g in (1, 2, 3, 4, 5, 8) if kv * g <= 64])
        ctx = _log(rng, 1024, 131072)
        T = _log(rng, 1, 512)
        return {"op": op, "cache": cache, "tokens": T, "heads": heads, "kv_heads": kv, "head_dim": hd, "ctx": ctx,
                "pos": rng.randrange(0, ctx - T + 1), "theta": rng.choice([10000.0, 500000.0]),
                "norm": rng.random() < 0.5}
    if op == "read":
        ctx = _log(rng, 64, 32768 * 8 // max(8, kv))
        count = rng.randint(1, ctx)
        return {"op": op, "cache": cache, "kv_heads": kv, "head_dim": hd, "ctx": ctx,
                "start": rng.randint(0, ctx - count), "count": count, "out": rng.choice(["f16", "f32"])}
    if op == "move":
        nodes = _log(rng, 2, 256)
        keep = rng.randint(1, max(1, nodes // 2))
        pos = rng.randint(0, 3800)
        return {"op": op, "cache": cache, "kv_heads": kv, "head_dim": hd, "ctx": 4096, "pos": pos, "nodes": nodes,
                "keep": keep}
    if op == "attention":
        heads = kv * rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8) if kv * g <= 64])
        T = _log(rng, 1, 64)
        most = min(131000, 8 * 131000 // kv, 64 * 64 * 32577 * 128 // (T * heads * hd))
        past = _log(rng, 1, most) - 1
        ctx = past + T + rng.randint(0, 300)
        return {"op": op, "cache": cache, "tokens": T, "heads": heads, "kv_heads": kv, "head_dim": hd, "ctx": ctx,
                "past": past}
    rows = _log(rng, 1, 64)
    return {"op": "logits", "rows": rows, "vocab": _log(rng, 100, 128259), "history": _log(rng, 1, 1000),
            "bias": rng.choice([0, 1, 30, 60]), "mask": rng.choice(["none", "shared", "rows"])}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=g)


def _cache_views(buf, kv, hd, ctx, dtype):
    """fp16: the [kv, ctx, hd] tensor.  int8: the codes [kv, ctx, hd] and, from the next multiple of 256 bytes,
    one fp32 scale for each row [kv, ctx]."""
    if dtype == "f16":
        return buf, None
    n = kv * ctx * hd
    off = -(-n // 256) * 256
    return buf[:n].view(torch.int8).view(kv, ctx, hd), buf[off:off + 4 * kv * ctx].view(torch.float32).view(kv, ctx)


def _make_cache(g, kv, hd, ctx, dtype, filled):
    """A cache half (K or V) whose first `filled` positions hold rows of about unit size."""
    if dtype == "f16":
        buf = torch.zeros((kv, ctx, hd), dtype=torch.float16, device=DEV)
        buf[:, :filled].normal_(0.0, 1.0, generator=g)
        return buf
    n = -(-kv * ctx * hd // 256) * 256
    buf = torch.zeros(n + 4 * kv * ctx, dtype=torch.uint8, device=DEV)
    codes, scales = _cache_views(buf, kv, hd, ctx, dtype)
    # rows of normal values quantised to their own largest magnitude: codes spread over +-127
    codes[:, :filled] = torch.empty((kv, filled, hd), dtype=torch.float16, device=DEV).normal_(
        0.0, 45.0, generator=g).round_().clamp_(-127, 127).to(torch.int8)
    scales[:, :filled].uniform_(0.012, 0.032, generator=g)
    return buf


def _tree(seed, T):
    """Parents of a random tree in topological order (node 0 the root), its depths and ancestor bit masks."""
    r = random.Random(seed)
    parent = [-1] + [r.randrange(max(0, i - 6), i) for i in range(1, T)]
    depth, sees = [], []
    for i, p in enumerate(parent):
        depth.append(0 if p < 0 else depth[p] + 1)
        sees.append((0 if p < 0 else sees[p]) | (1 << i))
    W = (T + 31) // 32
    words = np.array([[(s >> (32 * w)) & 0xFFFFFFFF for w in range(W)] for s in sees], dtype=np.uint32)
    return depth, words.view(np.int32)


def prepare(case, seed):
    c = dict(case)
    g = _gen(seed)
    s = {"c": c}
    op = c["op"]
    if op == "logits":
        rows, V, H = c["rows"], c["vocab"], c["history"]
        s["logits"] = _randn(g, rows, V, std=3.0)
        # recent tokens repeat: ids from a steep distribution over the vocabulary
        u = torch.rand((rows, H), device=DEV, generator=g)
        s["history"] = (u.pow(3) * V).to(torch.int32).clamp_(0, V - 1)
        s["lens"] = torch.randint(0, H + 1, (rows,), device=DEV, generator=g, dtype=torch.int32)
        s["bias_ids"] = torch.randperm(V, device=DEV, generator=g)[:c["bias"]].to(torch.int32)
        s["bias"] = _randn(g, c["bias"], std=2.0)
        W = (V + 31) // 32
        if c["mask"] == "none":
            s["mask"] = None
        else:
            shape = (1, W) if c["mask"] == "shared" else (rows, W)
            a = torch.randint(-2**31, 2**31, shape, device=DEV, generator=g)
            b = torch.randint(-2**31, 2**31, shape, device=DEV, generator=g)
            s["mask"] = (a & b).to(torch.int32)
        s["out"] = torch.empty_like(s["logits"])
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device=DEV)
    else:
        kv, hd, ctx, dt = c["kv_heads"], c["head_dim"], c["ctx"], c["cache"]
        filled = {"append": c.get("pos", 0), "read": ctx, "move": c.get("pos", 0) + c.get("nodes", 0),
                  "attention": c.get("past", 0) + c.get("tokens", 0)}[op]
        if op == "append":
            filled = 0  # what lies before the written slots is not touched
        s["k"] = _make_cache(g, kv, hd, ctx, dt, filled)
        s["v"] = _make_cache(g, kv, hd, ctx, dt, filled)
        pos = c.get("pos", c.get("past", 0))
        s["state"] = torch.tensor([1, pos, 0, 0], dtype=torch.int32, device=DEV)
    if op == "append":
        T, H = c["tokens"], c["heads"]
        s["qkv"] = _randn(g, T, (H + 2 * kv) * hd, std=1.5)
        s["depth"] = torch.tensor(_tree(seed, T)[0], dtype=torch.int32, device=DEV)
        s["q_norm"] = 1.0 + _randn(g, hd, std=0.1) if c["norm"] else None
        s["k_norm"] = 1.0 + _randn(g, hd, std=0.1) if c["norm"] else None
        s["q_out"] = torch.empty((T, H * hd), dtype=torch.float32, device=DEV)
        s["k_rows"] = torch.empty((kv, T, hd), dtype=torch.float16, device=DEV)
        s["v_rows"] = torch.empty_like(s["k_rows"])
    elif op == "read":
        t = torch.float16 if c["out"] == "f16" else torch.float32
        s["k_rows"] = torch.empty((kv, c["count"], hd), dtype=t, device=DEV)
        s["v_rows"] = torch.empty_like(s["k_rows"])
    elif op == "move":
        # the kept nodes are among the later half, so that a repeated move gives the same rows
        keep, nodes = c["keep"], c["nodes"]
        r = random.Random(seed)
        src = sorted(r.sample(range(keep, nodes), min(keep, nodes - keep)))
        c["kept"] = len(src)
        s["src"] = torch.tensor(src, dtype=torch.int32, device=DEV)
        s["dst"] = torch.arange(len(src), dtype=torch.int32, device=DEV)
        s["k_rows"] = torch.empty((kv, len(src), hd), dtype=torch.float16, device=DEV)
        s["v_rows"] = torch.empty_like(s["k_rows"])
    elif op == "attention":
        T, H = c["tokens"], c["heads"]
        s["q"] = _randn(g, T, H * hd, std=1.7)
        s["mask"] = torch.from_numpy(_tree(seed, T)[1]).to(DEV)
        s["out"] = torch.empty((T, H * hd), dtype=torch.float32, device=DEV)
    if own:  # the handles and scratch that a program keeps
        from odiengine_b200 import draft

        if op == "logits":
            s["scratch"] = draft.logits_scratch(rows)
        else:
            s["cache"] = draft.KVCache(s["k"], s["v"], dt, kv, hd, ctx)
            if op == "attention":
                s["scratch"] = draft.attention_tree_scratch(s["cache"], T, H)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------

def run(s):
    c = s["c"]
    if own:
        return _OWN[c["op"]](s, c)
    return _PLAIN[c["op"]](s, c)


def _own_append(s, c):
    from odiengine_b200 import draft

    draft.qk_rope_append(s["qkv"], s["cache"], s["state"], s["q_out"], heads=c["heads"], theta=c["theta"],
                         q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, depth=s["depth"])
    p, T = c["pos"], c["tokens"]
    if c["cache"] == "f16":  # the cache's own rows
        return s["q_out"], s["k"][:, p:p + T], s["v"][:, p:p + T]
    draft.kv_read(s["cache"], p, T, s["k_rows"], s["v_rows"])
    return s["q_out"], s["k_rows"], s["v_rows"]


def _own_read(s, c):
    from odiengine_b200 import draft

    draft.kv_read(s["cache"], c["start"], c["count"], s["k_rows"], s["v_rows"])
    return s["k_rows"], s["v_rows"]


def _own_move(s, c):
    from odiengine_b200 import draft

    draft.kv_move(s["cache"], s["src"], s["dst"], state=s["state"])
    p, n = c["pos"], c["kept"]
    if c["cache"] == "f16":
        return s["k"][:, p:p + n], s["v"][:, p:p + n]
    draft.kv_read(s["cache"], p, n, s["k_rows"], s["v_rows"])
    return s["k_rows"], s["v_rows"]


def _own_attention(s, c):
    from odiengine_b200 import draft

    return draft.attention_tree(s["q"], s["cache"], s["out"], s["state"], heads=c["heads"],
                                scale=1.0 / math.sqrt(c["head_dim"]), scratch=s["scratch"], mask=s["mask"])


def _own_logits(s, c):
    from odiengine_b200 import draft

    draft.logits_adjust(s["logits"], s["out"], s["tokens"], scratch=s["scratch"], history=s["history"],
                        history_lens=s["lens"], repeat_penalty=1.1, frequency_penalty=0.05, presence_penalty=0.2,
                        bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"])
    return s["out"], s["tokens"]


_OWN = {"append": _own_append, "read": _own_read, "move": _own_move, "attention": _own_attention,
        "logits": _own_logits}


def _angles(c, depth):
    """cos and sin of the rotation, [T, 1, hd/2]: far positions need 64 bits before the sine."""
    i = torch.arange(c["head_dim"] // 2, dtype=torch.float64, device=DEV)
    a = (c["pos"] + depth).double()[:, None] * torch.pow(c["theta"], -2.0 * i / c["head_dim"])
    return torch.cos(a)[:, None, :], torch.sin(a)[:, None, :]


def _quantise(x):
    """Rows to int8 codes and one fp32 scale each: d = max|x| / 127, codes round half away from zero."""
    d = x.abs().amax(-1, keepdim=True) / 127.0
    t = x * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
    return torch.trunc(t + torch.copysign(torch.full_like(t, 0.5), t)), d


def _store(buf, rows, start, c):
    """rows [kv, n, hd] fp32 into the cache half at start..; returns what the cache then holds."""
    view, scales = _cache_views(buf, c["kv_heads"], c["head_dim"], c["ctx"], c["cache"])
    n = rows.shape[1]
    if scales is None:
        view[:, start:start + n] = rows.half()
        return view[:, start:start + n]
    codes, d = _quantise(rows)
    view[:, start:start + n] = codes.to(torch.int8)
    scales[:, start:start + n] = d[..., 0]
    return (codes * d).half()


def _rows(buf, lo, hi, c):
    """Cache rows lo..hi-1 in 32 bits."""
    view, scales = _cache_views(buf, c["kv_heads"], c["head_dim"], c["ctx"], c["cache"])
    x = view[:, lo:hi].float()
    return x if scales is None else x * scales[:, lo:hi, None]


def _plain_append(s, c):
    T, H, kv, hd = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].view(T, H + 2 * kv, hd)
    q, k, v = x[:, :H], x[:, H:H + kv], x[:, H + kv:]
    if c["norm"]:
        q = q / torch.sqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    cs, sn = (a.float() for a in _angles(c, s["depth"]))

    def turn(u):
        a, b = u[..., :hd // 2], u[..., hd // 2:]
        return torch.cat([a * cs - b * sn, a * sn + b * cs], -1)

    kr, vr = turn(k).transpose(0, 1), v.transpose(0, 1)
    return turn(q).reshape(T, H * hd), _store(s["k"], kr, c["pos"], c), _store(s["v"], vr, c["pos"], c)


def _plain_read(s, c):
    lo, hi = c["start"], c["start"] + c["count"]
    t = torch.float16 if c["out"] == "f16" else torch.float32
    return _rows(s["k"], lo, hi, c).to(t), _rows(s["v"], lo, hi, c).to(t)


def _plain_move(s, c):
    got = []
    p, n = c["pos"], c["kept"]
    for buf in (s["k"], s["v"]):
        view, scales = _cache_views(buf, c["kv_heads"], c["head_dim"], c["ctx"], c["cache"])
        src = s["src"].long() + p
        view[:, p:p + n] = view[:, src]
        if scales is not None:
            scales[:, p:p + n] = scales[:, src]
        got.append(_rows(buf, p, p + n, c).half() if scales is not None else view[:, p:p + n])
    return tuple(got)


def _visible(s, c):
    """[T, len]: what each node sees: the whole past, and its bits of the tree."""
    T = c["tokens"]
    j = torch.arange(T, device=DEV)
    bits = (s["mask"][:, j // 32] >> (j % 32)) & 1
    return torch.cat([torch.ones((T, c["past"]), dtype=torch.bool, device=DEV), bits.bool()], 1)


def _attend(q, k, v, vis, c):
    T, H, kv, hd = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"]
    G = H // kv
    x = q.view(T, kv, G, hd).permute(1, 0, 2, 3).reshape(kv, T * G, hd)
    p = torch.matmul(x, k.transpose(1, 2))
    p *= 1.0 / math.sqrt(hd)
    p.masked_fill_(~vis.repeat_interleave(G, 0), -math.inf)
    p -= p.amax(-1, keepdim=True)
    p.exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(kv, T, G, hd).permute(1, 0, 2, 3).reshape(T, H * hd)


def _plain_attention(s, c):
    n = c["past"] + c["tokens"]
    return _attend(s["q"], _rows(s["k"], 0, n, c), _rows(s["v"], 0, n, c), _visible(s, c), c)


def _plain_logits(s, c):
    rows, V, H = c["rows"], c["vocab"], c["history"]
    live = torch.arange(H, device=DEV) < s["lens"][:, None]
    count = torch.zeros((rows, V), dtype=torch.int32, device=DEV)
    count.scatter_add_(1, s["history"].long(), live.int())
    x = s["logits"]
    seen = count > 0
    x = torch.where(seen, torch.where(x > 0, x / 1.1, x * 1.1), x)
    x = x - count.float() * 0.05
    x = torch.where(seen, x - 0.2, x)
    b = torch.zeros(V, dtype=torch.float32, device=DEV)
    b[s["bias_ids"].long()] = s["bias"]
    x = x + b
    if s["mask"] is not None:
        j = torch.arange(V, device=DEV)
        x = torch.where(((s["mask"][:, j // 32] >> (j % 32)) & 1).bool(), x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, torch.arange(V, device=DEV), V).amin(-1)  # ties: the lowest index
    return x, torch.where(top[:, 0] > -math.inf, first, -1).int()


_PLAIN = {"append": _plain_append, "read": _plain_read, "move": _plain_move, "attention": _plain_attention,
          "logits": _plain_logits}


# ---- 64 bits ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    op = c["op"]
    if op == "logits":
        x = s["logits"].double().cpu().numpy()
        hist, lens = s["history"].cpu().numpy(), s["lens"].cpu().numpy()
        for r in range(c["rows"]):
            ids, n = np.unique(hist[r, :lens[r]], return_counts=True)
            l = x[r, ids]
            # the penalties are fp32 arguments of the call
            x[r, ids] = (np.where(l > 0, l / float(np.float32(1.1)), l * float(np.float32(1.1)))
                         - n * float(np.float32(0.05)) - float(np.float32(0.2)))
        x[:, s["bias_ids"].cpu().numpy()] += s["bias"].double().cpu().numpy()
        if s["mask"] is not None:
            w = np.ascontiguousarray(s["mask"].cpu().numpy()).view(np.uint8)
            x[np.broadcast_to(np.unpackbits(w, axis=1, bitorder="little")[:, :c["vocab"]] == 0, x.shape)] = -np.inf
        return x, None
    kv, hd = c["kv_heads"], c["head_dim"]

    def rows64(buf, idx):
        view, scales = _cache_views(buf, kv, hd, c["ctx"], c["cache"])
        x = view[:, idx].double()
        return x if scales is None else x * scales[:, idx, None].double()

    if op == "read":
        idx = torch.arange(c["start"], c["start"] + c["count"], device=DEV)
        return rows64(s["k"], idx), rows64(s["v"], idx)
    if op == "move":
        idx = s["src"].long() + c["pos"]
        return rows64(s["k"], idx), rows64(s["v"], idx)
    T, H = c["tokens"], c["heads"]
    if op == "append":
        x = s["qkv"].double().view(T, H + 2 * kv, hd)
        p = torch.tensor(_tree(seed, T)[0], dtype=torch.float64, device=DEV) + c["pos"]
        half = hd // 2
        f = torch.tensor([c["theta"] ** (-2.0 * i / hd) for i in range(half)], dtype=torch.float64, device=DEV)
        z = torch.polar(torch.ones((T, half), dtype=torch.float64, device=DEV), p[:, None] * f)[:, None]

        def one(u, w):
            if w is not None:
                u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * w.double()
            r = torch.complex(u[..., :half].contiguous(), u[..., half:].contiguous()) * z
            return torch.cat([r.real, r.imag], -1)

        def held(u):
            u = u.transpose(0, 1)
            if c["cache"] == "f16":
                return u
            d = (u.abs().amax(-1, keepdim=True) / 127.0).float().double()  # the scale is kept in 32 bits
            return torch.sign(u) * torch.floor((u / d).abs() + 0.5) * d

        return (one(x[:, :H], s["q_norm"]).reshape(T, H * hd), held(one(x[:, H:H + kv], s["k_norm"])),
                held(x[:, H + kv:]))
    n = c["past"] + T
    idx = torch.arange(n, device=DEV)
    vis = _visible(s, c)
    q = s["q"].double().view(T, kv, H // kv, hd)
    out = torch.empty((T, H, hd), dtype=torch.float64, device=DEV)
    k, v = rows64(s["k"], idx), rows64(s["v"], idx)
    for h in range(kv):  # one key head after the other: the scores of all would not fit
        w = torch.einsum("tgd,nd->tgn", q[:, h], k[h]) / math.sqrt(hd)
        w = torch.softmax(w.masked_fill(~vis[:, None, :], -math.inf), -1)
        out[:, h * (H // kv):(h + 1) * (H // kv)] = torch.einsum("tgn,nd->tgd", w, v[h])
    return out.reshape(T, H * hd)


def work(case):
    c = case
    op = c["op"]
    if op == "logits":
        n = c["rows"] * c["vocab"]
        m = {"none": 0, "shared": (c["vocab"] + 31) // 32 * 4, "rows": c["rows"] * ((c["vocab"] + 31) // 32) * 4}
        return {"bytes": 8 * n + m[c["mask"]] + 4 * c["rows"] * (c["history"] + 2) + 8 * c["bias"], "flops": n}
    kv, hd = c["kv_heads"], c["head_dim"]
    row = 2 * hd if c["cache"] == "f16" else hd + 4
    if op == "append":
        T, H = c["tokens"], c["heads"]
        return {"bytes": 4 * T * (2 * H + 2 * kv) * hd + 2 * T * kv * row, "flops": 6 * T * (H + kv) * hd}
    if op == "read":
        out = 2 if c["out"] == "f16" else 4
        return {"bytes": 2 * c["count"] * kv * (row + out * hd), "flops": 2 * c["count"] * kv * hd}
    if op == "move":
        n = min(c["keep"], c["nodes"] - c["keep"])
        return {"bytes": 4 * n * kv * row, "flops": 0}
    T, H = c["tokens"], c["heads"]
    n = c["past"] + T
    return {"bytes": 8 * T * H * hd + 2 * n * kv * row + 4 * T * ((T + 31) // 32), "flops": 4 * T * H * hd * n}
