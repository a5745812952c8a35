"""The drafted-token operators (odiengine_b200.draft) against plain float64
implementations.

u = 2^-24 below is half a step of fp32.  Tolerances:
  q rows        the norm's factor takes 11 roundings (a sum of squares through
                9 adds enters by its square root: 4.5; mean, eps, sqrt,
                reciprocal, weight, product), the rotation 3 (two products,
                their sum) and the sine and cosine 2 u each plus the angle's
                2^-26 turn = 1.6 u rad: |d| <= 20 u (|a| + |b|) of the pair
  fp16 rows     those 20 u, then half an fp16 step: 2^-11 |x| + 2^-25
  int8 rows     20 u, then half a code (0.5 d) and the 127 * 4 u d that scale,
                reciprocal, product and the border add
  reads         exact: one product, one rounding
  attention     a score is a sum of hd products in some order,
                |ds| <= hd u S with S = scale * sum |q_i k_i|, and a weight is
                off by |ds| + 8 u of itself (exp, sum, division): the output by
                2 (|ds| + 8 u) max|v|, a worst case.  The roundings are
                independent, so the 2-norm over all outputs is held to 1e-5.
  logits        exact: the same fp32 operations in the same order
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dr(cuda_lib):
    from odiengine_b200 import draft

    return draft


def dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def state(pos):
    import torch

    return torch.tensor([1, pos, 0, 0], dtype=torch.int32, device="cuda")


def halves(cache):
    """The cache's K and V as (values or codes, scales or None), numpy views of copies."""
    import torch

    out = []
    for t in (cache.k, cache.v):
        if cache.dtype == "f16":
            out.append((t.cpu().numpy().reshape(cache.kv_heads, cache.ctx, cache.head_dim), None))
        else:
            n = cache.kv_heads * cache.ctx * cache.head_dim
            off = (n + 255) // 256 * 256
            b = t.cpu()
            out.append((b[:n].view(torch.int8).numpy().reshape(cache.kv_heads, cache.ctx, cache.head_dim),
                        b[off:off + 4 * cache.kv_heads * cache.ctx].view(torch.float32).numpy()
                        .reshape(cache.kv_heads, cache.ctx)))
    return out


def quantise(x):
    """The int8 row quantiser in fp32, operation by operation."""
    x = x.astype(np.float32)
    d = (np.abs(x).max(-1, keepdims=True) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(d > 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
    t = (x * inv).astype(np.float32)
    # round half away from zero: exact in float64
    return (np.sign(t) * np.floor(np.abs(t.astype(np.float64)) + 0.5)).astype(np.int8), d[..., 0]


def fill(cache, rng, lo=0, hi=None, garbage=None):
    """Random rows lo..hi-1 (normal, of differing sizes); `garbage` bytes-level junk elsewhere."""
    import torch

    kv, ctx, hd = cache.kv_heads, cache.ctx, cache.head_dim
    hi = ctx if hi is None else hi
    for t in (cache.k, cache.v):
        x = rng.standard_normal((kv, ctx, hd)) * np.exp(0.3 * rng.standard_normal((kv, ctx, 1)))
        if cache.dtype == "f16":
            x = x.astype(np.float16)
            if garbage is not None:
                x[:, :lo] = garbage
                x[:, hi:] = garbage
            t.copy_(torch.from_numpy(x))
        else:
            q, d = quantise(x)
            if garbage is not None:
                q[:, hi:], d[:, hi:] = -128, garbage
                q[:, :lo], d[:, :lo] = -128, garbage
            n = kv * ctx * hd
            off = (n + 255) // 256 * 256
            t[:n].view(torch.int8).copy_(torch.from_numpy(q.reshape(-1)))
            t[off:off + 4 * kv * ctx].view(torch.float32).copy_(torch.from_numpy(d.reshape(-1)))


def values64(cache):
    return [x.astype(np.float64) if s is None else x.astype(np.float64) * s[..., None].astype(np.float64)
            for x, s in halves(cache)]


# ---- append ----------------------------------------------------------------------------------------------------

def rope64(x, p, theta):
    """x [T, heads, hd] float64 rotated at positions p [T]."""
    hd = x.shape[-1]
    h = hd // 2
    ang = p[:, None].astype(np.float64) * theta ** (-2.0 * np.arange(h) / hd)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = x[..., :h], x[..., h:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def pair_size(x):
    h = x.shape[-1] // 2
    m = np.abs(x[..., :h]) + np.abs(x[..., h:])
    return np.concatenate([m, m], -1)


APPEND = [  # hd, heads, kv_heads, T, ctx, pos, dtype, norm, theta, extra stride, offset
    (128, 32, 8, 1, 64, 17, "i8", True, 1e4, 0, 0),
    (128, 32, 8, 1, 64, 17, "f16", False, 1e4, 0, 0),
    (64, 4, 4, 1, 8, 0, "f16", True, 1e4, 0, 0),
    (64, 5, 1, 3, 7, 4, "i8", True, 5e5, 1, 1),
    (128, 9, 3, 17, 40, 20, "i8", False, 1e4, 3, 1),
    (128, 64, 8, 300, 513, 100, "f16", True, 5e5, 0, 0),
    (64, 12, 12, 129, 200, 60, "i8", True, 1e4, 2, 2),
    (128, 2, 2, 1, 5, 4, "i8", True, 1e4, 0, 0),
]


@pytest.mark.parametrize("hd,H,KV,T,ctx,pos,dt,norm,theta,extra,off", APPEND)
@pytest.mark.parametrize("tree", [False, True])
def test_append(dr, hd, H, KV, T, ctx, pos, dt, norm, theta, extra, off, tree):
    import torch

    rng = np.random.default_rng(hd + T + pos)
    W = (H + 2 * KV) * hd
    x = (1.7 * rng.standard_normal((T, W))).astype(np.float32)
    buf = torch.zeros(off + T * (W + extra), device="cuda")
    qkv = buf[off:].view(T, W + extra)[:, :W]
    qkv.copy_(dev(x))
    wq, wk = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    # a tree's depths; one node at a far position (the rotation only, not the slot)
    depth = rng.integers(0, T, T).astype(np.int32)
    depth[-1] = 1_000_003
    p = pos + (depth.astype(np.int64) if tree else np.arange(T))
    c = dr.KVCache.new(dt, KV, hd, ctx)
    fill(c, rng)
    before = halves(c)
    obuf = torch.full((off + T * (H * hd + extra),), 7.0, device="cuda")
    out = obuf[off:].view(T, H * hd + extra)[:, :H * hd]
    got = dr.qk_rope_append(qkv, c, state(pos), out, heads=H, theta=theta, q_norm=dev(wq) if norm else None,
                            k_norm=dev(wk) if norm else None, eps=1e-6, depth=dev(depth) if tree else None)
    assert got is out
    torch.cuda.synchronize()
    assert torch.equal(qkv, dev(x))
    r = x.astype(np.float64).reshape(T, H + 2 * KV, hd)
    q, k, v = r[:, :H], r[:, H:H + KV], r[:, H + KV:]
    if norm:
        q, k = (a / np.sqrt((a * a).mean(-1, keepdims=True) + 1e-6) * w for a, w in ((q, wq), (k, wk)))
    tq, tk = 20 * U * pair_size(q), 20 * U * pair_size(k)
    q, k = rope64(q, p, theta), rope64(k, p, theta)
    assert (np.abs(out.cpu().numpy().reshape(T, H, hd) - q) <= tq).all()
    if extra:  # what lies between the rows is left alone
        assert (obuf[off:].view(T, H * hd + extra)[:, H * hd:] == 7.0).all()
    n = min(T, ctx - pos)  # slots past the cache are not written
    after = halves(c)
    for (a, sa), (b, sb), ref, tol in ((before[0], after[0], k, tk), (before[1], after[1], v, 0 * tk)):
        keep = np.r_[0:pos, pos + n:ctx]
        assert np.array_equal(a[:, keep], b[:, keep])
        ref, tol = ref[:n].transpose(1, 0, 2), tol[:n].transpose(1, 0, 2)
        rows = b[:, pos:pos + n]
        if dt == "f16":
            assert (np.abs(rows.astype(np.float64) - ref) <= tol + np.abs(ref) * 2.0 ** -11 + 2.0 ** -25).all()
        else:
            assert np.array_equal(sa[:, keep], sb[:, keep])
            d = sb[:, pos:pos + n].astype(np.float64)
            big = np.abs(ref).max(-1)
            assert (np.abs(d - big / 127) <= tol.max(-1) / 127 + 2 * U * d).all()
            assert (np.abs(rows * d[..., None] - ref) <= tol + d[..., None] * (0.5 + 127 * 4 * U)).all()
            assert np.abs(rows).max() == 127
    if dt == "i8":  # v is stored as it came: the quantiser to the bit
        codes, d = quantise(x.reshape(T, -1, hd)[:n, H + KV:].transpose(1, 0, 2))
        assert np.array_equal(after[1][0][:, pos:pos + n], codes)
        assert np.array_equal(after[1][1][:, pos:pos + n], d)


def test_append_in_place_and_repeated(dr):
    import torch

    rng = np.random.default_rng(5)
    H, KV, hd, T = 6, 2, 128, 9
    x = dev(rng.standard_normal((T, (H + 2 * KV) * hd)).astype(np.float32))
    c = dr.KVCache.new("f16", KV, hd, 32)
    a = dr.qk_rope_append(x, c, state(3), heads=H, theta=1e4)
    k0 = c.k.clone()
    b = dr.qk_rope_append(x, c, state(3), heads=H, theta=1e4)
    assert torch.equal(a, b) and torch.equal(k0, c.k)
    y = x.clone()
    dr.qk_rope_append(y, c, state(3), y[:, :H * hd], heads=H, theta=1e4)
    torch.cuda.synchronize()
    assert torch.equal(y[:, :H * hd], a) and torch.equal(y[:, H * hd:], x[:, H * hd:]) and torch.equal(k0, c.k)


@pytest.mark.parametrize("dt", ["f16", "i8"])
def test_append_zero_tiny_and_nonfinite_rows(dr, dt):
    """A zero row, one too small for an fp32 reciprocal, and rows with NaN or
    infinity: int8 rows read back as 0, 0, NaN; the neighbours are untouched."""
    import torch

    hd, T = 64, 5
    x = np.ones((T, 3, hd), np.float32)
    x[0] = 0
    x[1] = 1e-39
    x[2, :, 7] = np.nan
    x[3, :, 9] = np.inf
    c = dr.KVCache.new(dt, 1, hd, 8)
    dr.qk_rope_append(dev(x.reshape(T, -1)), c, state(1), heads=1, theta=1e4, k_norm=None)
    k, v = dr.kv_read(c, 1, T)
    k, v = k.cpu().numpy()[0], v.cpu().numpy()[0]
    assert not v[:2].any() and not k[:2].any()
    if dt == "i8":
        assert np.isnan(v[2:4]).all() and np.isnan(k[2:4]).all()
    else:
        assert np.isnan(v[2, 7]) and np.isinf(v[3, 9]) and np.isfinite(v[2, :7]).all()
    assert np.allclose(v[4], 1.0, rtol=2.0 ** -11)


@pytest.mark.parametrize("pos", [-3, -1, 63, 64, 2**31 - 1])
def test_append_outside_the_cache(dr, pos):
    """Slots outside [0, ctx) are not written; q is rotated all the same."""
    import torch

    rng = np.random.default_rng(1)
    H, KV, hd, T, ctx = 2, 1, 64, 2, 64
    x = rng.standard_normal((T, (H + 2 * KV) * hd)).astype(np.float32)
    c = dr.KVCache.new("f16", KV, hd, ctx)
    q = dr.qk_rope_append(dev(x), c, state(pos), heads=H, theta=1e4)
    torch.cuda.synchronize()
    written = np.abs(halves(c)[1][0][0]).sum(-1) > 0
    want = np.zeros(ctx, bool)
    for t in range(T):
        if 0 <= pos + t < ctx:
            want[pos + t] = True
    assert np.array_equal(written, want)
    r = x[:, :H * hd].reshape(T, H, hd).astype(np.float64)
    assert (np.abs(q.cpu().numpy().reshape(T, H, hd) - rope64(r, pos + np.arange(T), 1e4)) <= 20 * U * pair_size(r)).all()


# ---- read and move ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("out", ["f16", "f32"])
@pytest.mark.parametrize("hd,KV,ctx,start,count", [(64, 1, 1, 0, 1), (64, 3, 77, 5, 33), (128, 2, 300, 0, 300),
                                                   (128, 8, 1031, 1030, 1), (128, 5, 999, 17, 901)])
def test_read(dr, dt, out, hd, KV, ctx, start, count):
    import torch

    c = dr.KVCache.new(dt, KV, hd, ctx)
    fill(c, np.random.default_rng(ctx))
    t = torch.float16 if out == "f16" else torch.float32
    bufs = [torch.full((KV * count * hd + 8,), 3.0, dtype=t, device="cuda") for _ in range(2)]
    k, v = (b[:KV * count * hd].view(KV, count, hd) for b in bufs)
    dr.kv_read(c, start, count, k, v)
    for (x, s), got, b in zip(halves(c), (k, v), bufs):
        f = x.astype(np.float32) if s is None else (x.astype(np.float32) * s[..., None]).astype(np.float32)
        want = f[:, start:start + count].astype(np.float16 if out == "f16" else np.float32)
        assert np.array_equal(got.cpu().numpy(), want)
        assert (b[KV * count * hd:] == 3.0).all()
    only = torch.empty_like(v)
    dr.kv_read(c, start, count, None, only)
    assert torch.equal(only, v)
    dr.kv_read(c, ctx, 0)


def moved(rows, src, dst, pos):
    new, ctx = rows.copy(), rows.shape[1]
    for a, b in zip(src, dst):  # in list order: a destination listed twice takes its last row
        if 0 <= pos + a < ctx and 0 <= pos + b < ctx:
            new[:, pos + b] = rows[:, pos + a]
    return new


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("KV,ctx,pos,src,dst", [
    (2, 40, 10, [0, 2, 5, 9], [0, 1, 2, 3]),             # an accepted path: sources and destinations overlap
    (1, 40, None, [3], [39]),
    (3, 64, 5, list(range(30, 0, -1)), list(range(30))),  # every row is a source and a destination
    (2, 16, 4, [0, 1, 2, 3], [7, 7, 8, 7]),               # listed twice
    (2, 16, 4, [0, 50, 2, -9, 3], [1, 2, -40, 5, 12]),    # ends outside the cache are skipped
    (2, 600, 100, list(range(255, -1, -1)), list(range(200, 456))),
    (1, 8, -3, [3, 4], [9, 10]),
])
def test_move(dr, dt, hd, KV, ctx, pos, src, dst):
    c = dr.KVCache.new(dt, KV, hd, ctx)
    fill(c, np.random.default_rng(7))
    before = halves(c)
    dr.kv_move(c, dev(np.array(src, np.int32)), dev(np.array(dst, np.int32)), None if pos is None else state(pos))
    for (a, sa), (b, sb) in zip(before, halves(c)):
        assert np.array_equal(moved(a, src, dst, pos or 0), b)
        if sa is not None:
            assert np.array_equal(moved(sa, src, dst, pos or 0), sb)


# ---- attention -------------------------------------------------------------------------------------------------

def random_tree(rng, T):
    par = [-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, T)]
    vis = np.zeros((T, T), bool)
    for i, p in enumerate(par):
        if p >= 0:
            vis[i] = vis[p]
        vis[i, i] = True
    return vis


def words(vis):
    T = vis.shape[0]
    W = (T + 31) // 32
    bits = np.zeros((T, W * 32), np.uint8)
    bits[:, :T] = vis
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32).reshape(T, W)


def attend64(q, K, V, vis, pos, scale):
    """q [T, H, hd], K and V [KV, ctx, hd] float64: outputs and the tolerance's S."""
    T, H, hd = q.shape
    KV, ctx = K.shape[:2]
    n = max(0, min(ctx, pos + T))
    out, S = np.zeros((T, H, hd)), np.zeros((T, H))
    seen = np.zeros((T, n), bool)
    seen[:, :max(0, min(pos, n))] = True
    for j in range(T):
        if 0 <= pos + j < n:
            seen[:, pos + j] = vis[:, j]
    for h in range(H):
        kh = h // (H // KV)
        for t in range(T):
            w = seen[t]
            if not w.any():
                continue
            k, v = K[kh, :n][w], V[kh, :n][w]
            s = scale * (k @ q[t, h])
            S[t, h] = abs(scale) * (np.abs(k) @ np.abs(q[t, h])).max()
            p = np.exp(s - s.max())
            out[t, h] = (p @ v) / p.sum()
    return out, S


def check_attention(dr, dt, hd, H, KV, T, pos, ctx, mask, seed=0, qstd=1.5, pad=0, garbage=np.nan):
    import torch

    rng = np.random.default_rng(seed + 1000 * T + pos)
    c = dr.KVCache.new(dt, KV, hd, ctx)
    n = max(0, min(ctx, pos + T))
    fill(c, rng, 0, n, garbage=garbage)
    q = (qstd * rng.standard_normal((T, H, hd))).astype(np.float32)
    vis = np.tril(np.ones((T, T), bool)) if mask is None else mask(rng, T)
    qb = torch.zeros((T, H * hd + pad), device="cuda")
    qb[:, :H * hd] = dev(q.reshape(T, -1))
    scr = dr.attention_tree_scratch(c, T, H)
    out = torch.full((T, H * hd), 9.0, device="cuda")
    scale = 1.0 / math.sqrt(hd)
    outs = []
    for _ in range(2):
        dr.attention_tree(qb[:, :H * hd], c, out, state(pos), heads=H, scale=scale, scratch=scr,
                          mask=None if mask is None else dev(words(vis)))
        outs.append(out.cpu().numpy().reshape(T, H, hd))
    assert np.array_equal(outs[0], outs[1])  # fixed order of every sum, scratch left reusable
    assert not scr[:256].cpu().numpy()[:4].any()
    K, V = values64(c)
    K, V = np.nan_to_num(K), np.nan_to_num(V)
    ref, S = attend64(q.astype(np.float64), K, V, vis, pos, scale)
    vmax = np.abs(V[:, :n]).max() if n else 0.0
    tol = 2 * (hd * U * S + 8 * U)[..., None] * vmax
    err = np.abs(outs[0] - ref)
    assert np.isfinite(outs[0]).all()
    assert (err <= tol).all(), (err.max(), tol.min())
    if np.linalg.norm(ref):
        assert np.linalg.norm(outs[0] - ref) <= 1e-5 * np.linalg.norm(ref), np.linalg.norm(outs[0] - ref) / np.linalg.norm(ref)
    return outs[0]


ATT = [  # hd, heads, kv_heads, T, pos, ctx
    (128, 8, 2, 1, 0, 8),        # one token, empty past
    (128, 8, 8, 1, 63, 64),      # every head its own keys, the cache full
    (64, 8, 1, 1, 127, 300),     # length 128: a whole block
    (64, 4, 4, 1, 128, 300),     # one past it
    (128, 32, 8, 13, 300, 400),
    (128, 6, 2, 5, 1000, 1005),  # ratio 3, the tree ends with the cache
    (64, 7, 1, 33, 77, 200),     # ratio 7, two mask words
    (128, 16, 2, 16, 250, 266),  # the tree straddles a block border
    (128, 64, 8, 64, 500, 700),
    (64, 5, 5, 256, 0, 256),     # the largest tree, no past
    (128, 8, 1, 200, 333, 600),
    (128, 4, 4, 3, 2500, 2600),
    (128, 40, 8, 7, 4090, 4200),
    (64, 40, 8, 31, 1023, 1100),
    (128, 32, 8, 13, 4001, 8192),
    # so much work that a CTA takes 64 rows
    (128, 8, 1, 200, 333, 5000),
    (128, 16, 2, 64, 1200, 7300),
    (128, 64, 8, 64, 1500, 2000),
    (128, 40, 1, 256, 0, 700),
    (128, 33, 1, 129, 77, 1600),
]


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("hd,H,KV,T,pos,ctx", ATT)
def test_attention(dr, dt, hd, H, KV, T, pos, ctx):
    check_attention(dr, dt, hd, H, KV, T, pos, ctx, random_tree, pad=4 * (T % 3))


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("T,pos,H,ctx", [(1, 5, 8, 300), (9, 0, 8, 300), (70, 200, 8, 300), (70, 200, 64, 2000)])
def test_attention_chain_without_a_mask(dr, dt, T, pos, H, ctx):
    check_attention(dr, dt, 128, H, 2, T, pos, ctx, None)


@pytest.mark.parametrize("dt", ["f16", "i8"])
def test_attention_nodes_that_see_nothing(dr, dt):
    """With no past, nodes with an empty mask row get zeros, whatever the others see."""
    def some(rng, T):
        v = rng.random((T, T)) < 0.3
        v[::3] = False
        return v

    for H, KV, ctx in ((8, 4, 64), (64, 1, 6000)):  # 32 and 64 rows per CTA
        out = check_attention(dr, dt, 128, H, KV, 20, 0, ctx, some)
        assert not out[::3].any()


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("pos,ctx,T", [(-2, 16, 5), (-9, 16, 5), (14, 16, 5), (16, 16, 5), (40, 16, 2),
                                        (41, 21, 2), (1000, 20, 3), (1000, 130, 40)])
def test_attention_slots_outside_the_cache(dr, dt, pos, ctx, T):
    """pos < 0 or a tree past the cache's end: those slots are not seen."""
    check_attention(dr, dt, 64, 4, 2, T, pos, ctx, lambda rng, t: np.ones((t, t), bool))
    check_attention(dr, dt, 128, 8, 1, T, pos, ctx, lambda rng, t: np.ones((t, t), bool))


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("pos", [-20, -100, 2890, 2900, 5000])
def test_attention_many_rows_outside_the_cache(dr, dt, pos):
    """The same with 64 rows per CTA."""
    check_attention(dr, dt, 128, 64, 1, 40, pos, 2900, lambda rng, t: np.ones((t, t), bool))


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("H,KV,ctx", [(8, 2, 256), (64, 1, 4900)])  # 32 and 64 rows per CTA
def test_attention_nonfinite_nodes_stay_with_who_sees_them(dr, dt, bad, H, KV, ctx):
    """K and V of one tree slot are not finite: nodes that do not see it get
    what they get without it; nodes that see it get NaN."""
    import torch

    rng = np.random.default_rng(3)
    hd, T, pos, j = 128, 24, 150, 4
    c = dr.KVCache.new(dt, KV, hd, ctx)
    fill(c, rng, 0, pos + T)
    q = dev((1.5 * rng.standard_normal((T, H * hd))).astype(np.float32))
    vis = random_tree(rng, T)
    scr = dr.attention_tree_scratch(c, T, H)
    kw = dict(heads=H, scale=0.1, scratch=scr, mask=dev(words(vis)))
    clean = dr.attention_tree(q, c, None, state(pos), **kw).cpu().numpy()
    for t in (c.k, c.v):
        if dt == "f16":
            t[:, pos + j, 5] = bad
        else:
            n = KV * ctx * hd
            off = (n + 255) // 256 * 256
            t[off:off + 4 * KV * ctx].view(torch.float32).view(KV, ctx)[:, pos + j] = bad
    got = dr.attention_tree(q, c, None, state(pos), **kw).cpu().numpy()
    blind = ~vis[:, j]
    assert blind.any() and vis[:, j].any()
    assert np.array_equal(got[blind], clean[blind])
    assert not np.isfinite(got[vis[:, j]]).any(axis=0).all()


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("qstd", [0.0, 1e-6, 40.0, 1e4])
@pytest.mark.parametrize("H,KV,T,ctx", [(8, 2, 6, 800), (256, 1, 9, 3400)])  # 32 and 64 rows per CTA
def test_attention_query_sizes(dr, dt, qstd, H, KV, T, ctx):
    """Equal scores, tiny ones, and scores of which one key takes all (the
    softmax tolerance then scales with S)."""
    import torch

    rng = np.random.default_rng(11)
    hd, pos = 128, 700
    c = dr.KVCache.new(dt, KV, hd, ctx)
    fill(c, rng, 0, pos + T, garbage=np.nan)
    q = (qstd * rng.standard_normal((T, H, hd))).astype(np.float32)
    out = dr.attention_tree(dev(q.reshape(T, -1)), c, None, state(pos), heads=H, scale=0.088,
                            scratch=dr.attention_tree_scratch(c, T, H)).cpu().numpy().reshape(T, H, hd)
    K, V = (np.nan_to_num(x) for x in values64(c))
    ref, S = attend64(q.astype(np.float64), K, V, np.tril(np.ones((T, T), bool)), pos, 0.088)
    w = np.minimum(1.0, 2 * (hd * U * S + 8 * U))[..., None]  # a weight cannot be off by more than itself
    assert np.isfinite(out).all()
    assert (np.abs(out - ref) <= 2 * w * np.abs(V).max()).all()


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("hd,T,H,KV,ctx", [(64, 9, 8, 2, 256), (128, 1, 8, 2, 256), (128, 9, 8, 2, 256), (128, 9, 256, 1, 3400)])
@pytest.mark.parametrize("scale", [0.0, -0.09, 1e-30])
def test_attention_any_scale(dr, dt, hd, T, scale, H, KV, ctx):
    """Zero (the mean of what is seen), negative and tiny scales, with nodes masked."""
    rng = np.random.default_rng(13)
    pos = 200
    c = dr.KVCache.new(dt, KV, hd, ctx)
    fill(c, rng, 0, pos + T, garbage=np.nan)
    q = (1.5 * rng.standard_normal((T, H, hd))).astype(np.float32)
    vis = random_tree(rng, T)
    out = dr.attention_tree(dev(q.reshape(T, -1)), c, None, state(pos), heads=H, scale=scale, mask=dev(words(vis)),
                            scratch=dr.attention_tree_scratch(c, T, H)).cpu().numpy().reshape(T, H, hd)
    K, V = (np.nan_to_num(x) for x in values64(c))
    ref, S = attend64(q.astype(np.float64), K, V, vis, pos, float(np.float32(scale)))
    assert (np.abs(out - ref) <= 2 * (hd * U * S + 8 * U)[..., None] * np.abs(V).max()).all()


def test_attention_two_caches_one_scratch_and_graph(dr):
    """One scratch serves the layers of a step; a captured step replays with
    another position."""
    import torch

    rng = np.random.default_rng(2)
    hd, H, KV, T, ctx = 128, 8, 2, 8, 500
    cs = [dr.KVCache.new(dt, KV, hd, ctx) for dt in ("f16", "f16", "i8")]
    for c in cs:
        fill(c, rng)
    q = dev(rng.standard_normal((T, H * hd)).astype(np.float32))
    st = state(100)
    scr = dr.attention_tree_scratch(cs[0], T, H)
    outs = [torch.zeros((T, H * hd), device="cuda") for _ in cs]

    def step():
        for c, o in zip(cs, outs):
            dr.attention_tree(q, c, o, st, heads=H, scale=0.1, scratch=scr)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for pos in (100, 333, 0):
        st.copy_(state(pos))
        g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for c, o in zip(cs, got):
            own = dr.attention_tree(q, c, None, state(pos), heads=H, scale=0.1,
                                    scratch=dr.attention_tree_scratch(c, T, H))
            assert torch.equal(own, o)


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_shapes_share_one_scratch(dr, hd):
    """Calls of different numbers of tokens, dtypes and lengths, one scratch,
    alternating: each as with a scratch of its own (the joins through it leave
    its counters zero whatever came before)."""
    import torch

    rng = np.random.default_rng(21)
    H, KV, ctx = 8, 2, 30000
    cs = [dr.KVCache.new(dt, KV, hd, ctx) for dt in ("f16", "i8")]
    for c in cs:
        fill(c, rng)
    scr = dr.attention_tree_scratch(cs[0], 1, H)
    assert scr.numel() == dr.attention_tree_scratch(cs[1], 256, 64).numel()
    for T, pos in ((1, 29000), (13, 29900), (1, 200), (70, 15000), (3, 29997), (256, 20000), (1, 29999), (2, 29000)):
        q = dev(rng.standard_normal((T, H * hd)).astype(np.float32))
        for c in cs:
            a = dr.attention_tree(q, c, None, state(pos), heads=H, scale=0.1, scratch=scr)
            b = dr.attention_tree(q, c, None, state(pos), heads=H, scale=0.1, scratch=dr.attention_tree_scratch(c, T, H))
            assert torch.equal(a, b), (T, pos)


def test_attention_long_offsets_past_32_bits(dr):
    """kv_heads * ctx * head_dim past 2^31 values: the last head's rows are the
    ones read."""
    import torch

    hd, H, KV, T, pos = 128, 20, 20, 2, 900
    ctx = 840_001
    c = dr.KVCache.new("i8", KV, hd, ctx)  # 2.15e9 codes each
    rng = np.random.default_rng(8)
    n = KV * ctx * hd
    off = (n + 255) // 256 * 256
    rows = rng.integers(-127, 128, (pos + T, hd)).astype(np.int8)
    for t, m in ((c.k, 1), (c.v, -1)):
        t[:n].view(torch.int8).view(KV, ctx, hd)[KV - 1, :pos + T] = dev(rows) * m
        t[off:off + 4 * KV * ctx].view(torch.float32).view(KV, ctx)[KV - 1, :pos + T] = 0.02
    q = rng.standard_normal((T, H, hd)).astype(np.float32)
    out = dr.attention_tree(dev(q.reshape(T, -1)), c, None, state(pos), heads=H, scale=0.1,
                            scratch=dr.attention_tree_scratch(c, T, H)).cpu().numpy().reshape(T, H, hd)
    x = rows.astype(np.float64) * float(np.float32(0.02))
    ref, S = attend64(q[:, -1:].astype(np.float64), x[None], -x[None], np.tril(np.ones((T, T), bool)), pos, 0.1)
    assert (np.abs(out[:, -1:] - ref) <= 2 * (hd * U * S + 8 * U)[..., None] * np.abs(x).max()).all()
    assert not out[:, :-1].any()  # the other heads hold zeros
    k, _ = dr.kv_read(c, 3, pos - 3)
    assert np.array_equal(k[KV - 1].cpu().numpy(), (rows[3:pos].astype(np.float32) * np.float32(0.02)).astype(np.float16))


# ---- logits ----------------------------------------------------------------------------------------------------

def adjust(x, hist=None, lens=None, rp=1.0, fp=0.0, pp=0.0, ids=None, bias=None, mask=None):
    """The same fp32 operations, row by row."""
    x = x.copy()
    rows, V = x.shape
    f = np.float32
    for r in range(rows):
        if hist is not None:
            h = hist[r % hist.shape[0]]
            h = h[:hist.shape[1] if lens is None else max(0, min(lens[r], hist.shape[1]))]
            h = h[(h >= 0) & (h < V)]
            i, n = np.unique(h, return_counts=True)
            l = x[r, i]
            with np.errstate(over="ignore", invalid="ignore"):
                l = np.where(l > 0, l / f(rp), l * f(rp)).astype(f)
                l = (l - (n.astype(f) * f(fp)).astype(f)).astype(f)
                x[r, i] = (l - f(pp)).astype(f)
        if ids is not None:
            last = {int(i): b for i, b in zip(ids, bias)}
            for i, b in last.items():
                if 0 <= i < V:
                    x[r, i] = f(x[r, i] + b)
        if mask is not None:
            bits = np.unpackbits(mask[r % mask.shape[0]].view(np.uint8), bitorder="little")[:V]
            x[r, bits == 0] = -np.inf
    tok = np.full(rows, -1, np.int32)
    for r in range(rows):
        y = np.where(np.isnan(x[r]), -np.inf, x[r])
        if y.max() > -np.inf:
            tok[r] = int(np.argmax(y))
    return x, tok


@pytest.mark.parametrize("rows,V,H,nb,mask", [
    (1, 1, 1, 1, 1), (1, 100, 5, 0, 0), (3, 31, 40, 3, 3), (2, 4093, 10, 7, 1), (5, 4096, 0, 0, 5), (4, 4097, 64, 9, 4),
    (7, 8191, 300, 33, 1), (64, 1003, 1000, 50, 64), (1, 32000, 64, 7, 1), (3, 128259, 2000, 300, 3)])
@pytest.mark.parametrize("pad", [0, 3])
def test_logits(dr, rows, V, H, nb, mask, pad):
    import torch

    rng = np.random.default_rng(V + rows)
    x = (3 * rng.standard_normal((rows, V))).astype(np.float32)
    x[0, V // 2] = 0.0
    hist = (V * rng.random((rows, H)) ** 3).astype(np.int32) if H else None
    if H > 4:
        hist[:, 0], hist[:, 1], hist[0, 2] = -1, V, V + 5  # ids outside the vocabulary are skipped
    lens = rng.integers(0, H + 1, rows).astype(np.int32) if H else None
    ids = rng.integers(-2, V + 2, nb).astype(np.int32) if nb else None  # some twice, some outside
    bias = rng.standard_normal(nb).astype(np.float32) if nb else None
    m = rng.integers(-2**31, 2**31, (mask, (V + 31) // 32)).astype(np.int32) if mask else None
    buf = torch.full((rows, V + pad), 5.0, device="cuda")
    xin = buf[:, :V]
    xin.copy_(dev(x))
    out = torch.full((rows, V + 2 * pad), 6.0, device="cuda")
    tok = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    scr = dr.logits_scratch(rows)
    kw = dict(scratch=scr, history=dev(hist) if H else None, history_lens=dev(lens) if H else None, repeat_penalty=1.3,
              frequency_penalty=0.1, presence_penalty=0.7, bias_ids=dev(ids) if nb else None,
              bias=dev(bias) if nb else None, mask=dev(m) if mask else None)
    want, wtok = adjust(x, hist, lens, 1.3, 0.1, 0.7, ids, bias, m)
    for _ in range(2):  # the scratch is left reusable
        tok.fill_(77)
        dr.logits_adjust(xin, out[:, :V], tok, **kw)
        assert np.array_equal(out[:, :V].cpu().numpy(), want)
        assert np.array_equal(tok.cpu().numpy(), wtok)
    assert not scr.any() and (out[:, V:] == 6.0).all() and (buf[:, V:] == 5.0).all()
    tok.fill_(77)
    dr.logits_adjust(xin, None, tok, **kw)      # the tokens alone
    assert np.array_equal(tok.cpu().numpy(), wtok) and torch.equal(xin, dev(x))
    dr.logits_adjust(xin, xin, **{**kw, "scratch": None})  # in place, no tokens
    assert np.array_equal(xin.cpu().numpy(), want) and (buf[:, V:] == 5.0).all()


def test_logits_ties_empty_rows_and_nonfinite(dr):
    import torch

    V = 9000
    x = np.zeros((6, V), np.float32)
    x[0, [4500, 8999, 77]] = 2.0          # a tie across CTAs: the lowest index
    x[1] = np.nan                         # nothing to choose
    x[2] = -np.inf
    x[2, 8000] = np.nan
    x[3, 100], x[3, 50] = np.inf, np.nan
    x[4] = -0.0
    x[4, 20] = 0.0                        # -0 and +0 are equal: index 0
    tok = torch.zeros(6, dtype=torch.int32, device="cuda")
    scr = dr.logits_scratch(6)
    dr.logits_adjust(dev(x), None, tok, scratch=scr)
    assert tok.cpu().tolist() == [77, -1, -1, 100, 0, 0]
    mask = np.zeros((6, (V + 31) // 32), np.int32)
    mask[0, 8999 // 32] = np.uint32(1 << (8999 % 32)).astype(np.int32)
    out = torch.empty((6, V), device="cuda")
    dr.logits_adjust(dev(x), out, tok, scratch=scr, mask=dev(mask))
    assert tok.cpu().tolist() == [8999, -1, -1, -1, -1, -1]
    o = out.cpu().numpy()
    assert (o[1:] == -np.inf).all() and o[0, 8999] == 2.0 and (o[0, :8999] == -np.inf).all()
    # a bias of -inf bans a token, a shared history counts for every row
    dr.logits_adjust(dev(x), out, tok, scratch=scr, bias_ids=dev(np.array([77], np.int32)),
                     bias=dev(np.array([-np.inf], np.float32)), history=dev(np.array([[4500, 4500]], np.int32)),
                     frequency_penalty=0.5)
    assert tok.cpu().tolist()[0] == 8999 and out[0, 4500].item() == 1.0 and out[5, 4500].item() == -1.0


# ---- other streams ---------------------------------------------------------------------------------------------

def test_calls_follow_their_stream(dr):
    """On a side stream the calls are ordered with that stream's work."""
    import torch

    rng = np.random.default_rng(4)
    hd, H, KV, T, ctx, pos = 128, 8, 2, 12, 300, 200
    x = dev(rng.standard_normal((T, (H + 2 * KV) * hd)).astype(np.float32))
    res = []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for how in ("current", "argument", "inline"):
        c = dr.KVCache.new("i8", KV, hd, ctx)
        scr = dr.attention_tree_scratch(c, T, H)
        q, out = torch.zeros((T, H * hd), device="cuda"), torch.zeros((T, H * hd), device="cuda")
        st = state(pos)
        y = torch.zeros_like(x)
        s.wait_stream(torch.cuda.current_stream())
        kw = dict(stream=s) if how == "argument" else {}
        ctxm = torch.cuda.stream(s) if how != "inline" else torch.cuda.stream(torch.cuda.current_stream())
        with ctxm:
            torch.cuda._sleep(2_000_000)  # the input arrives late
            y.copy_(x)
            dr.qk_rope_append(y, c, st, q, heads=H, theta=1e4, **kw)
            dr.attention_tree(q, c, out, st, heads=H, scale=0.1, scratch=scr, **kw)
        torch.cuda.synchronize()
        res.append(out.cpu())
    assert torch.equal(res[0], res[1]) and torch.equal(res[0], res[2]) and res[0].abs().sum() > 0
