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
