"""Attention of drafted tokens where a number format could show: scales far
from the others, one key that outweighs all, rows beside rows that differ."""
import numpy as np
import pytest

from test_gpu_draft import attend64, dev, dr, fill, random_tree, state, values64, words  # noqa: F401

pytestmark = pytest.mark.gpu

# hd, heads, kv_heads, ctx of the shapes below: 64 dims; 8 and fewer, and more rows per kv head; 32 and 64 rows per CTA
SHAPES = [(64, 8, 4, 256, 24), (128, 8, 8, 256, 7), (128, 8, 2, 256, 24), (128, 64, 1, 4900, 24)]


def scales(cache, half):
    """The int8 cache's row scales [kv_heads, ctx], a view."""
    import torch

    n = cache.kv_heads * cache.ctx * cache.head_dim
    off = (n + 255) // 256 * 256
    return half[off:off + 4 * cache.kv_heads * cache.ctx].view(torch.float32).view(cache.kv_heads, cache.ctx)


@pytest.mark.parametrize("hd,H,KV,ctx,T", SHAPES)
@pytest.mark.parametrize("big", [1e30, 1e36, 3e38])
def test_a_large_scale_stays_with_who_sees_it(dr, hd, H, KV, ctx, T, big):  # noqa: F811
    """A finite V scale of any size in a slot that a node does not see changes nothing."""
    rng = np.random.default_rng(5)
    pos, j = 150, 2
    c = dr.KVCache.new("i8", KV, hd, ctx)
    fill(c, rng, 0, pos + T)
    q = dev((1.5 * rng.standard_normal((T, H * hd))).astype(np.float32))
    vis = random_tree(rng, T)
    vis[:, j] = False
    kw = dict(heads=H, scale=0.1, scratch=dr.attention_tree_scratch(c, T, H), mask=dev(words(vis)))
    clean = dr.attention_tree(q, c, None, state(pos), **kw).cpu().numpy()
    scales(c, c.v)[:, pos + j] = big
    assert np.array_equal(dr.attention_tree(q, c, None, state(pos), **kw).cpu().numpy(), clean)


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("hd,H,KV,ctx,T", SHAPES)
def test_nonfinite_rows_reach_all_of_who_sees_them(dr, dt, bad, which, hd, H, KV, ctx, T):  # noqa: F811
    """One value of a tree slot's K or V (int8: the row's scale) is not finite:
    every output of a node that sees it is NaN, of every head, and the others
    are what they are without it.  (An fp16 key's infinity stands against
    queries of either sign: exp(-inf) is a weight of 0, and the header allows NaN.)"""
    rng = np.random.default_rng(9)
    pos, j = 150, 3
    c = dr.KVCache.new(dt, KV, hd, ctx)
    fill(c, rng, 0, pos + T)
    q = dev((1.5 * rng.standard_normal((T, H * hd))).astype(np.float32))
    vis = random_tree(rng, T)
    vis[j + 1:, j] &= rng.random(T - j - 1) < 0.5
    vis[-1, j] = False
    kw = dict(heads=H, scale=0.1, scratch=dr.attention_tree_scratch(c, T, H), mask=dev(words(vis)))
    clean = dr.attention_tree(q, c, None, state(pos), **kw).cpu().numpy()
    half = getattr(c, which)
    if dt == "f16":
        half[:, pos + j, 5] = bad
    elif not (bad < 0):  # scales are not negative
        scales(c, half)[:, pos + j] = bad
    else:
        return
    got = dr.attention_tree(q, c, None, state(pos), **kw).cpu().numpy()
    nan = np.isnan(got.reshape(T, H, hd))
    if dt == "f16" and which == "k" and np.isinf(bad):
        sees = vis.copy()
        sees[:, j] = False
        without = dr.attention_tree(q, c, None, state(pos), **{**kw, "mask": dev(words(sees))}).cpu().numpy().reshape(T, H, hd)
        below = (q.cpu().numpy().reshape(T, H, hd)[..., 5] * bad < 0) & vis[:, j, None]  # scores of -inf
        assert (nan.all(-1) == nan.any(-1)).all()
        zero = below & ~nan.any(-1)
        assert np.array_equal(got.reshape(T, H, hd)[zero], without[zero])
        nan[zero] = True
    assert nan[vis[:, j]].all()
    assert vis[:, j].any() and not vis[:, j].all() and np.array_equal(got[~vis[:, j]], clean[~vis[:, j]])


@pytest.mark.parametrize("hd,H,KV,ctx,T", SHAPES)
@pytest.mark.parametrize("big", [1e27, 3e38])
def test_a_large_scale_of_no_weight(dr, hd, H, KV, ctx, T, big):  # noqa: F811
    """A row that all see, of any finite V scale, whose weight is below 2^-150 (0
    in fp32): nobody's outputs change, nor the bits that other rows keep."""
    rng = np.random.default_rng(15)
    pos, j = 150, 100
    c = dr.KVCache.new("i8", KV, hd, ctx)
    fill(c, rng, 0, pos + T)
    q = dev(np.abs(rng.standard_normal((T, H * hd))).astype(np.float32) + 0.5)
    c.k[:KV * ctx * hd].view(KV, ctx, hd)[:, j] = 256 - 127  # codes of -127: scores of -0.1 * 4 * 127 * 64 * 0.5 and below
    scales(c, c.k)[:, j] = 4.0
    kw = dict(heads=H, scale=0.1, scratch=dr.attention_tree_scratch(c, T, H))
    before = dr.attention_tree(q, c, None, state(pos), **kw).cpu().numpy()
    scales(c, c.v)[:, j] = big
    after = dr.attention_tree(q, c, None, state(pos), **kw).cpu().numpy()
    assert np.isfinite(before).all() and np.array_equal(before, after)


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("hd,H,KV,ctx,T", SHAPES)
@pytest.mark.parametrize("size", [1e38, 3.4e38])
def test_queries_of_any_finite_size(dr, dt, hd, H, KV, ctx, T, size):  # noqa: F811
    """Queries up to fp32's largest, with a scale that brings the scores back: q
    enters to within 2^-20 (int8; 2^-22 fp16) of its largest value, so a score of
    hd such products is off by at most hd 2^-20 of the largest, and the rest as in
    test_gpu_draft."""
    rng = np.random.default_rng(31)
    pos = 150
    c = dr.KVCache.new(dt, KV, hd, ctx)
    fill(c, rng, 0, pos + T)
    q = rng.uniform(-1, 1, (T, H, hd))
    q /= np.abs(q).max(-1, keepdims=True)
    q = (q * size).astype(np.float32)
    scale = 0.2 / size
    vis = random_tree(rng, T)
    out = dr.attention_tree(dev(q.reshape(T, -1)), c, None, state(pos), heads=H, scale=scale, mask=dev(words(vis)),
                            scratch=dr.attention_tree_scratch(c, T, H)).cpu().numpy().reshape(T, H, hd)
    K, V = values64(c)
    ref, S = attend64(q.astype(np.float64), K, V, vis, pos, float(np.float32(scale)))
    ds = hd * 2.0 ** -24 * S + 0.2 * hd * 2.0 ** -20 * np.abs(K).max()
    assert (np.abs(out - ref) <= 2 * (ds + 8 * 2.0 ** -24)[..., None] * np.abs(V).max()).all()


def attend64_gpu(q, k, v, pos, scale):
    """q [T, H, hd], k and v [KV, pos + T, hd], float64 on the GPU, a chain."""
    import torch

    T, H, hd = q.shape
    KV, n = k.shape[:2]
    vis = torch.arange(n, device="cuda")[None] <= pos + torch.arange(T, device="cuda")[:, None]
    out = torch.empty_like(q)
    for h in range(KV):
        g = slice(h * (H // KV), (h + 1) * (H // KV))
        s = torch.einsum("tgd,nd->tgn", q[:, g], k[h]) * scale
        out[:, g] = torch.einsum("tgn,nd->tgd", torch.softmax(s.masked_fill(~vis[:, None], -np.inf), -1), v[h])
    return out


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("hd,H,KV,T", [(128, 8, 1, 1), (128, 32, 4, 2), (128, 8, 1, 64), (64, 8, 2, 13)])
@pytest.mark.parametrize("at", [0, 20001])
@pytest.mark.parametrize("gap", [6, 10, 14, 18])
def test_one_key_outweighs_all(dr, dt, hd, H, KV, T, at, gap):  # noqa: F811
    """One key `gap` nats above the mean of 30,000 others (in real models the first
    position is one), its values ordinary, small or 0, the others' with and
    without a mean.  The 2-norm is held to 1e-5, as for ordinary scores.

    A weight of an fp16 cache enters to within half of fp16's last 2^-24, against a
    largest of more than 2^11: 2^-36 of the key's.  Where that key's values are 0
    this is not small against the output: N such roundings, each of its own sign,
    of values of size 1."""
    import torch

    rng = np.random.default_rng(17 * gap + T)
    n, ctx, scale = 30_000, 30_100, hd ** -0.5
    pos = n - T
    k0, v0 = rng.standard_normal((2, KV, n, hd))
    q = rng.standard_normal((T, H, hd))
    q[..., 5], k0[..., 5] = 4.0, 0.0
    k0[:, at], k0[:, at, 5] = 0.0, gap / (4.0 * scale)
    qd = dev(q.astype(np.float32))
    c = dr.KVCache.new(dt, KV, hd, ctx)
    scr = dr.attention_tree_scratch(c, T, H)
    for size, mean in ((1.0, 0.0), (0.02, 0.0), (0.02, 0.5), (1.0, 0.5), (0.0, 0.0)):
        v = v0 + mean
        v[:, at] *= size
        rows = []
        for half, x in ((c.k, k0), (c.v, v)):
            x = torch.from_numpy(x).cuda()
            if dt == "f16":
                half[:, :n] = x.half()
                rows.append(half[:, :n].double())
            else:
                d = (x.abs().amax(-1, keepdim=True) / 127).float()
                codes = torch.round(x / torch.where(d > 0, d, 1.0).double())
                half[:KV * ctx * hd].view(torch.int8).view(KV, ctx, hd)[:, :n] = codes.to(torch.int8)
                scales(c, half)[:, :n] = d[..., 0]
                rows.append(codes * d.double())
        out = dr.attention_tree(qd.view(T, -1), c, None, state(pos), heads=H, scale=scale, scratch=scr)
        ref = attend64_gpu(qd.double(), *rows, pos, scale)
        err, norm = float((out.view(T, H, hd).double() - ref).norm()), float(ref.norm())
        tol = 1e-5 * norm
        if dt == "f16" and size == 0.0:
            tol += 2.0 ** -36 * (n * ref.numel()) ** 0.5
        assert err <= tol, (size, mean, err / norm, tol / norm)


@pytest.mark.parametrize("dt", ["f16", "i8"])
@pytest.mark.parametrize("hd,H,KV,T,n", [(128, 8, 8, 7, 5000), (128, 32, 8, 8, 30000), (128, 64, 8, 64, 9000), (64, 8, 1, 9, 6000)])
def test_rows_do_not_depend_on_each_other(dr, dt, hd, H, KV, T, n):  # noqa: F811
    """Every other node's queries are other ones, of other sizes: the bits of the
    nodes between them stay, over many blocks of positions per CTA."""
    rng = np.random.default_rng(23)
    c = dr.KVCache.new(dt, KV, hd, n + 64)
    fill(c, rng, 0, n + T)
    q = (1.7 * rng.standard_normal((T, H * hd))).astype(np.float32)
    kw = dict(heads=H, scale=hd ** -0.5, scratch=dr.attention_tree_scratch(c, T, H))
    want = dr.attention_tree(dev(q), c, None, state(n), **kw).cpu().numpy()
    for size in (0.0, 6.0, 40.0, np.nan):
        other = q.copy()
        other[1::2] = size * rng.standard_normal((T // 2, H * hd))
        got = dr.attention_tree(dev(other), c, None, state(n), **kw).cpu().numpy()
        assert np.array_equal(got[::2], want[::2])
        assert not np.array_equal(got[1::2], want[1::2])


# ---- streams ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("op", ["append", "read", "attention"])
def test_outputs_are_allocated_on_the_stream_that_writes_them(dr, op):  # noqa: F811
    """A block that was freed while work of the current stream still reads it is
    not what a call on another stream writes to."""
    import torch

    rng = np.random.default_rng(6)
    hd, H, KV, T, ctx = 128, 16, 16, 128, 256
    c = dr.KVCache.new("f16", KV, hd, ctx)
    fill(c, rng)
    x = dev(rng.standard_normal((T, (H + 2 * KV) * hd)).astype(np.float32))
    q = dev(rng.standard_normal((T, H * hd)).astype(np.float32))
    scr, st = dr.attention_tree_scratch(c, T, H), state(10)
    s = torch.cuda.Stream()

    def call(**kw):
        if op == "append":
            return dr.qk_rope_append(x, c, st, heads=H, theta=1e4, **kw)
        if op == "read":
            return torch.cat([t.flatten() for t in dr.kv_read(c, 3, T, **kw)])
        return dr.attention_tree(q, c, None, st, heads=H, scale=0.1, scratch=scr, **kw)

    want = call()
    torch.cuda.synchronize()
    # two blocks of the outputs' size (both outputs of a read), and a reader of them that comes late
    n, dt = (T * H * hd, torch.float32) if op != "read" else (KV * T * hd, torch.float16)
    blocks = [torch.full((n,), 3.0, dtype=dt, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    late = [b * 2 for b in blocks]
    del blocks
    if op == "read":
        k, v = dr.kv_read(c, 3, T, stream=s)
        s.synchronize()
        got = torch.cat([k.flatten(), v.flatten()])
    else:
        got = call(stream=s)
        s.synchronize()
    torch.cuda.synchronize()
    assert all((x == 6.0).all() for x in late)
    assert torch.equal(got, want)
