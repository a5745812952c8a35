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
