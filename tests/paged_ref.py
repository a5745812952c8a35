"""Plain restatements, in 64 bits and on the host, of the operators over a
paged cache (odiengine_b200.paged)."""
import math

import numpy as np
import torch


class Tables:
    """odi_cuda_paged_step on Python lists."""

    def __init__(self, table, lens, free, count):
        self.table, self.lens, self.free, self.count = [list(r) for r in table], list(lens), list(free), count

    def step(self, P, new, keep, max_new, max_rows):
        B, wide = len(self.lens), len(self.table[0])
        pages = lambda n: -(-n // P)  # noqa: E731
        status, had, kept = 0, [], []
        for b in range(B):
            n = self.lens[b]
            if n < 0 or n > wide * P:
                status, n = status | 32, min(max(n, 0), wide * P)
            k = n if keep is None else keep[b]
            if k < 0 or k > n:
                status, k = status | 16, min(max(k, 0), n)
            had.append(n)
            kept.append(k)
        dropped = []
        for b in range(B):
            for j in range(pages(kept[b]), pages(had[b])):
                dropped.append(self.table[b][j])
                self.table[b][j] = -1
        for i, p in enumerate(reversed(dropped)):
            self.free[self.count + i] = p
        self.count += len(dropped)
        starts, lens, positions, slots, asked, taken = [0], [], [-1] * max_rows, [-1] * max_rows, 0, 0
        for b in range(B):
            r0 = min(starts[-1], max_rows)
            rows = min(max(new[b], 0), max_rows)
            bad = 0
            if new[b] < 0 or new[b] > max_new:
                bad = 4
            elif kept[b] + new[b] > wide * P:
                bad = 2
            if rows and r0 + rows > max_rows:
                bad |= 8
            need = 0 if bad & 14 else pages(kept[b] + rows) - pages(kept[b])
            asked += need
            if need and asked > self.count:
                bad |= 1
            status |= bad
            starts.append(min(r0 + rows, max_rows))
            if bad & 15:
                self.lens[b] = kept[b]
                lens.append(0)
                continue
            for i in range(need):
                self.table[b][pages(kept[b]) + i] = self.free[self.count - 1 - (asked - need) - i]
            taken += need
            self.lens[b] = kept[b] + rows
            lens.append(self.lens[b])
            for j in range(rows):
                pos = kept[b] + j
                positions[r0 + j] = pos
                slots[r0 + j] = self.table[b][pos // P] * P + pos % P
        self.count -= taken
        return status, starts, lens, positions, slots


def attention(q, k, v, past, heads, scale, softcap=0.0, slopes=None, prefix=0):
    """One request: q [N, heads * hd], k and v [kv, n, hd] (n = past + N), any
    type; float64 rows [N, heads, hd], and for each value how far a kernel may
    be off whose weights are rounded to the cache's type.

    A weight is off by half a step of its type (below 2^-14 of the reference,
    fp16 has an absolute step: half of 2^-24), by its score's error and by 2^-20
    for exp2 and the sums.  A score's products are summed in fp32, by an adder
    that truncates: 2^-21 of the sum of magnitudes."""
    dt = k.dtype
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    kv, n, hd = k.shape
    N, G = q.shape[0], heads // kv
    x = q.view(N, kv, G, hd)
    s = torch.einsum("tkgd,knd->tkgn", x, k) * scale
    ds = torch.einsum("tkgd,knd->tkgn", x.abs(), k.nan_to_num().abs()) * scale * 2.0 ** -21
    if softcap:
        s = softcap * torch.tanh(s / softcap)
        ds = ds + softcap * 2.0 ** -21
    i = torch.arange(past, past + N)
    j = torch.arange(n)
    if slopes is not None:
        far = (i[:, None] - j[None]).abs().double()
        bias = slopes.detach().cpu().double().view(1, kv, G, 1) * far[:, None, None, :]
        s = s - bias
        ds = ds + (bias.abs() + s.abs()) * 2.0 ** -23
    see = j[None] < torch.clamp(i + 1, min=min(prefix, n))[:, None]
    s = s.masked_fill(~see[:, None, None], -math.inf)
    ds = ds.masked_fill(~see[:, None, None], 0.0)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    l = p.sum(-1, keepdim=True)
    vz = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    o = torch.einsum("tkgn,knd->tkgd", p, vz) / l.clamp(min=1e-300)
    half = torch.finfo(dt).eps / 2
    err = half + 2.0 ** -20 + ds
    tol = torch.einsum("tkgn,knd->tkgd", p * err, vz.abs()) / l.clamp(min=1e-300)
    tol = tol + o.abs() * ((p * (ds + 2.0 ** -20)).sum(-1, keepdim=True) / l.clamp(min=1e-300))
    if dt is torch.float16:
        tol = tol + 2.0 ** -25 * torch.einsum("tkgn,knd->tkgd", see[:, None, None].double().expand_as(p), vz.abs()) / l.clamp(min=1.0)
    # what is not finite reaches whoever sees it
    bad = ~torch.isfinite(v)
    if bad.any():
        plus = torch.einsum("tn,knd->tkd", see.double(), (v == math.inf).double()) > 0
        minus = torch.einsum("tn,knd->tkd", see.double(), (v == -math.inf).double()) > 0
        nan = (torch.einsum("tn,knd->tkd", see.double(), torch.isnan(v).double()) > 0) | (plus & minus)
        inf = torch.where(nan, math.nan, torch.where(plus, math.inf, torch.where(minus, -math.inf, 0.0)))
        o = o + inf[:, :, None]
    return o.reshape(N, heads * hd), tol.reshape(N, heads * hd)


def within(got, want, tol, out_dtype):
    """Whether got is within tol and the rounding of its own type of want; what is
    not finite has to be the same."""
    got = got.detach().cpu().double()
    fin = torch.isfinite(want)
    if not torch.equal(torch.isnan(got), torch.isnan(want)) or not torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]):
        return False
    step = torch.finfo(out_dtype).eps / 2 * (want.abs() + tol)
    if out_dtype is torch.float16:
        step = step.clamp(min=2.0 ** -25)
    return bool(((got - want).abs() <= tol + step)[fin].all())


def verify(logits, tokens, starts, u_accept, u_next, temperature, probs=None):
    """accepted and next of verify_sampled, in float64 numpy."""
    V = logits.shape[1]
    accepted, nxt = [], []
    for b in range(len(starts) - 1):
        a = 0
        tok = -1
        for r in range(starts[b], starts[b + 1]):
            x = logits[r].astype(np.float64)
            x = np.where(np.isposinf(x), np.finfo(np.float32).max, x)
            m = x.max() if not np.isnan(x).any() else np.nan
            if not m > -np.inf:
                break
            p = np.exp((x - m) / temperature)
            p /= p.sum()
            last = r + 1 == starts[b + 1]
            q = np.zeros(V)
            if not last:
                d = int(tokens[r + 1])
                ok = 0 <= d < V
                if probs is not None:
                    q = probs[r].astype(np.float64)
                elif ok:
                    q[d] = 1.0
                if ok and float(u_accept[r]) * q[d] < p[d]:
                    a += 1
                    continue
            w = np.maximum(p - q, 0.0)
            if last or w.sum() <= 0:
                w = p
            s = np.cumsum(w)
            over = np.nonzero(s > float(u_next[b]) * s[-1])[0]
            tok = int(over[0])
            break
        accepted.append(a)
        nxt.append(tok)
    return accepted, nxt
