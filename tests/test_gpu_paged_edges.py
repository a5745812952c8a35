"""The operators over a paged cache where they are easily wrong: logits so large
that nothing else counts, a key that outweighs all others, far positions, single
tiles, tables and batches that do not fit, lanes that part ways before an
instruction that wants them together."""
import math

import numpy as np
import pytest
import torch

import paged_ref
from test_gpu_paged import Setup, cuda_lib_status, ints

pytestmark = pytest.mark.gpu


# ---- verify -------------------------------------------------------------------------------------------------------

LARGEST = torch.finfo(torch.float32).max
# (largest logit, temperature): where it is +inf; where its neighbours in fp32 lie further
# apart than a weight reaches, or about as far; where nothing below it is finite
TOPS = [(math.inf, 1.0), (math.inf, 1e-6), (math.inf, 1e6), (LARGEST, 1.0), (3e9, 1.0), (2e10, 1.0), (2.2e9, 1.0), (2.2e6, 1e-3),
        (2.2e4, 1e-5), (1500.0, 1e-6), (1060.0, 1e-6), (1.7e7, 1e-3), (-1500.0, 1e-6), (-LARGEST, 1.0)]


@pytest.mark.parametrize("top,temperature", TOPS)
@pytest.mark.parametrize("V", [5, 3001, 40000])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_rows_whose_largest_logits_have_it_all(cuda_lib, top, temperature, V, probs):
    """One or two ids share a row, and the draft is one of them, or is not: what is
    kept and what is drawn are what p = 1, or 1/2 each, gives."""
    from odiengine_b200 import paged

    rng = np.random.default_rng(V)
    B = 8
    logits = (3 * rng.standard_normal((2 * B, V))).astype(np.float32)
    if top < 0:
        logits = np.full_like(logits, -np.inf) if top == -LARGEST else logits + np.float32(2 * top)
    tokens, ua = np.zeros(2 * B, np.int32), np.zeros(2 * B, np.float32)
    for b in range(B):
        ids = rng.choice(V, 3, replace=False)
        logits[2 * b:2 * b + 2, ids[:1 + b % 2]] = top
        tokens[2 * b + 1] = ids[2] if b == 6 else ids[b % 2]
        ua[2 * b] = (0.9, 0.3, 0.999, 0.7)[b % 4]
    un = rng.random(B).astype(np.float32)
    q = torch.softmax(torch.from_numpy(rng.standard_normal((2 * B, V)).astype(np.float32)), -1) if probs else None
    starts = list(range(0, 2 * B + 1, 2))
    got = paged.verify_sampled(torch.from_numpy(logits).cuda(), ints(tokens.tolist()), ints(starts), torch.from_numpy(ua).cuda(),
                               torch.from_numpy(un).cuda(), temperature=temperature, draft_probs=None if q is None else q.cuda(),
                               scratch=paged.verify_scratch(2 * B, B, V))
    want = paged_ref.verify(logits, tokens.tolist(), starts, ua.tolist(), un.tolist(), temperature, None if q is None else q.numpy())
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1], (got, want)
    assert want[0][0] == want[0][2] == 1 and want[0][6] == 0  # p = 1 is kept, p = 0 is not


# ---- attention ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("new,heads,kv,hd", [(1, 4, 4, 128), (1, 8, 1, 64), (1, 128, 128, 64), (3, 8, 1, 128), (70, 2, 2, 128), (40, 8, 1, 64), (300, 4, 2, 64)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nats", [12.0, 17.0, 18.0, 20.0])
@pytest.mark.parametrize("own", [0.0, 0.001])
@pytest.mark.parametrize("out32", [True, False])
def test_a_key_that_outweighs_the_rest(cuda_lib, new, heads, kv, hd, dtype, nats, own, out32):
    """One key some nats above all others, whose values are 0 or small: what the
    others add is there.  A weight is off by half a step of its type, 2^-20 and its
    score's error; in fp16, whose steps end, by 2^-32 of the row's largest weight: half of
    2^-24, that weight standing at 2^7 or above.  Weights of two parts (an fp32 output): one
    and a half of 2^-24, the second part's last bit and rounding.  Then the output's own."""
    from odiengine_b200 import paged

    past = 3000 - new
    s = Setup([past], [new], heads, kv, hd, dtype, 64, seed=int(nats))
    scale = 1 / math.sqrt(hd)
    g = torch.Generator(device="cuda").manual_seed(7)
    base = torch.randn(hd, device="cuda", generator=g)
    base = base / base.norm() * math.sqrt(hd)
    # every query along one direction, the keys but one across it or nearly so
    s.q.copy_((base * (1 + 0.01 * torch.randn((new, heads, 1), device="cuda", generator=g))).reshape(new, -1))
    keys = torch.randn(s.cache.k.shape, device="cuda", generator=g)
    keys -= (keys @ base)[..., None] * base / hd
    s.cache.k.copy_(keys * 0.3)
    s.cache.v.copy_(1 + 0.5 * torch.randn(s.cache.v.shape, device="cuda", generator=g))
    slot = int(s.tables.table[0, 1500 // 64]) * 64 + 1500 % 64
    s.cache.k[slot // 64, :, slot % 64] = base * (nats / (scale * hd))
    s.cache.v[slot // 64, :, slot % 64] = own
    out = torch.empty((new, heads * hd), dtype=torch.float32 if out32 else s.q.dtype, device="cuda")
    paged.attention_paged(s.q, s.cache, s.tables, s.batch, out, scale=scale, scratch=s.scratch)
    q, k, v = (t.cpu().double() for t in (s.q, s.rows(s.cache.k, 0), s.rows(s.cache.v, 0)))
    x = q.view(new, kv, heads // kv, hd)
    see = (torch.arange(past + new)[None] <= torch.arange(past, past + new)[:, None])[:, None, None]
    sc = torch.einsum("tkgd,knd->tkgn", x, k) * scale
    ds = torch.einsum("tkgd,knd->tkgn", x.abs(), k.abs()) * scale * 2.0 ** -21
    p = torch.exp((sc - sc.masked_fill(~see, -math.inf).amax(-1, keepdim=True)).masked_fill(~see, -math.inf))
    l = p.sum(-1, keepdim=True)
    want = torch.einsum("tkgn,knd->tkgd", p, v) / l
    err = p * (torch.finfo(s.cache.dtype).eps / 2 + 2.0 ** -20 + ds) + ((1.5 * 2.0 ** -31 if out32 else 2.0 ** -32) * see if dtype == "f16" else 0.0)
    tol = torch.einsum("tkgn,knd->tkgd", err, v.abs()) / l + want.abs() * ((p * (ds + 2.0 ** -20)).sum(-1, keepdim=True) / l + 2.0 ** -23)
    own_step = torch.finfo(out.dtype).eps / 2 * (want.abs() + tol)
    tol = tol + (own_step.clamp(min=2.0 ** -25) if out.dtype is torch.float16 else own_step)
    off = (out.cpu().double().view(want.shape) - want).abs()
    assert (off <= tol).all(), (off.max(), (off / tol).max())
    assert cuda_lib_status(s.scratch) == 0


def close_attention(s, b, row, scale, softcap=0.0, slopes=None):
    """Request b in 64 bits, and how far an fp32 output may be off.  A weight is off by its
    two parts: the first is cut off at a step of its type (2^-7 or 2^-10 of it), the second off
    by half a step of that, 2^-16, or in fp16, whose last bit is set, by one and a half,
    1.5 * 2^-20, or of fp16's smallest steps (2^-24, the largest weight standing at 2^7 or
    above); by 2^-20 and its score's error; a sum by a step of fp32 per product of 16
    positions, of which each part makes one."""
    past, N = s.past[b], s.new[b]
    n, parts = past + N, 1.5 * 2.0 ** -20 if s.cache.dtype is torch.float16 else 2.0 ** -16
    q, k, v = (t.cpu().double() for t in (s.q[row:row + N], s.rows(s.cache.k, b), s.rows(s.cache.v, b)))
    x = q.view(N, s.kv, s.heads // s.kv, s.hd)
    far = (torch.arange(past, n)[:, None] - torch.arange(n)[None])[:, None, None].double()
    sc = torch.einsum("tkgd,knd->tkgn", x, k) * scale
    ds = torch.einsum("tkgd,knd->tkgn", x.abs(), k.abs()) * scale * 2.0 ** -21
    if softcap:
        sc, ds = softcap * torch.tanh(sc / softcap), ds + softcap * 2.0 ** -21
    if slopes is not None:
        bias = slopes.cpu().double().view(1, s.kv, -1, 1) * far.abs()
        sc, ds = sc - bias, ds + (bias + (sc - bias).abs()) * 2.0 ** -23
    sc = sc.masked_fill(far < 0, -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    ds = ds.masked_fill(far < 0, 0.0)
    l = p.sum(-1, keepdim=True)
    want = torch.einsum("tkgn,knd->tkgd", p, v) / l
    rel = parts + 2.0 ** -20 + 2 * (n // 16 + 8) * 2.0 ** -23
    tiny = 1.5 * 2.0 ** -31 * (far >= 0).double().expand_as(p) if s.cache.dtype is torch.float16 else 0.0
    tol = torch.einsum("tkgn,knd->tkgd", p * (rel + ds) + tiny, v.abs()) / l
    return want.reshape(N, -1), (tol + want.abs() * ((p * (ds + rel)).sum(-1, keepdim=True) / l)).reshape(N, -1)


@pytest.mark.parametrize("past,new,heads,kv,hd,P", [
    ([99], [1], 4, 4, 128, 16), ([150, 3, 0], [1, 1, 1], 8, 1, 64, 32), ([120, 40], [3, 2], 16, 2, 128, 16), ([100, 0], [90, 200], 4, 2, 128, 64),
    ([0, 33], [129, 40], 8, 1, 64, 16), ([60], [300], 3, 3, 64, 128)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("option", ["plain", "cap", "slopes", "both"])
def test_an_fp32_output_is_more_than_16_bits(cuda_lib, past, new, heads, kv, hd, P, dtype, option):
    """Weights enter in two parts, so that what an fp32 output is off by is not their
    rounding to the cache's type."""
    from odiengine_b200 import paged

    s = Setup(past, new, heads, kv, hd, dtype, P)
    slopes = torch.linspace(0.01, 0.3, heads, device="cuda") if option in ("slopes", "both") else None
    cap, scale = 3.0 if option in ("cap", "both") else 0.0, 1 / math.sqrt(hd)
    out = torch.empty(s.q.shape, dtype=torch.float32, device="cuda")
    paged.attention_paged(s.q, s.cache, s.tables, s.batch, out, scale=scale, softcap=cap, slopes=slopes, scratch=s.scratch)
    row = 0
    for b, N in enumerate(new):
        want, tol = close_attention(s, b, row, scale, cap, slopes)
        off = (out[row:row + N].cpu().double() - want).abs()
        assert (off <= tol).all(), (b, off.max(), (off / tol).max())
        row += N
    assert cuda_lib_status(s.scratch) == 0


@pytest.mark.parametrize("past,new,heads,kv,hd", [([200], [1], 4, 4, 128), ([300], [3], 8, 1, 64), ([150], [70], 4, 2, 128), ([200], [129], 3, 3, 64)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("out32", [False, True])
@pytest.mark.parametrize("even", [False, True])
def test_infinities_that_all_rows_see(cuda_lib, past, new, heads, kv, hd, dtype, out32, even):
    """Infinite values of positions that every row sees stay infinities of their sign, and
    both signs a NaN: also where all weights are powers of two (queries of zero), which
    one 16-bit part holds whole."""
    from odiengine_b200 import paged

    s = Setup(past, new, heads, kv, hd, dtype, 32)
    if even:
        s.q.zero_()
    for j, d, x in ((0, 1, math.inf), (40, 2, -math.inf), (99, 3, math.inf), (100, 3, -math.inf), (140, 5, math.inf), (141, 5, math.inf)):
        slot = int(s.tables.table[0, j // 32]) * 32 + j % 32
        s.cache.v[slot // 32, :, slot % 32, d] = x
    out = torch.empty(s.q.shape, dtype=torch.float32 if out32 else s.q.dtype, device="cuda")
    paged.attention_paged(s.q, s.cache, s.tables, s.batch, out, scale=0.1, scratch=s.scratch)
    s.check(out, 0.1)
    assert cuda_lib_status(s.scratch) == 0


@pytest.mark.parametrize("past,new,heads,kv,hd", [([200], [1], 4, 4, 128), ([3000], [2], 8, 1, 64), ([150], [70], 4, 2, 128), ([2000], [129], 3, 3, 64)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("out32", [False, True])
@pytest.mark.parametrize("values", ["finite", "inf", "nan"])
def test_rows_all_of_whose_scores_are_minus_infinity_are_zero(cuda_lib, past, new, heads, kv, hd, dtype, out32, values):
    """Keys of -inf in one dim that the first head's queries look at and the others' do not;
    whatever values stand there."""
    from odiengine_b200 import paged

    s = Setup(past, new, heads, kv, hd, dtype, 64)
    T, G = sum(new), heads // kv
    q = s.q.view(T, kv, G, hd)
    s.cache.k[..., 7] = -math.inf
    q[..., 7] = 0.0  # 0 * -inf is NaN: the other heads' queries see NaN
    q[:, :, 0, 7] = 2.0
    if values != "finite":
        slot = int(s.tables.table[0, 1]) * 64 + 5
        s.cache.v[slot // 64, :, slot % 64, 3] = math.inf if values == "inf" else math.nan
    out = torch.full(s.q.shape, 9.0, dtype=torch.float32 if out32 else s.q.dtype, device="cuda")
    paged.attention_paged(s.q, s.cache, s.tables, s.batch, out, scale=0.1, scratch=s.scratch)
    got = out.view(T, kv, G, hd)
    assert (got[:, :, 0] == 0).all()
    assert G == 1 or torch.isnan(got[:, :, 1:]).all()
    assert cuda_lib_status(s.scratch) == 0


@pytest.mark.parametrize("new", [[1], [3], [40]])
def test_distances_behind_16_million_positions(cuda_lib, new):
    """Distances count whole positions where fp32 no longer tells two neighbouring
    positions apart."""
    from odiengine_b200 import paged

    past, heads, hd, P, near = (1 << 24) + 5, 4, 64, 128, 4096
    n = past + new[0]
    pages = -(-n // P)
    pools = [torch.zeros((pages, 1, P, hd), dtype=torch.float16, device="cuda") for _ in range(2)]
    cache = paged.PagedCache(*pools)
    t = paged.PageTables(torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous(), ints([past]),
                         torch.zeros(pages, dtype=torch.int32, device="cuda"), ints([0]), P)
    t.lens.fill_(n)  # the new tokens' pages are there
    batch = paged.PagedBatch(t, max_rows=new[0], max_new=new[0], heads=heads, kv_heads=1)
    paged.paged_step(t, batch, ints(new), keep=ints([past]))
    assert batch.status() == 0
    g = torch.Generator(device="cuda").manual_seed(3)
    for pool in pools:
        pool.view(-1, hd)[n - near:n] = torch.randn((near, hd), device="cuda", generator=g).half()
    q = torch.randn((new[0], heads * hd), device="cuda", generator=g).half()
    slopes = torch.tensor([0.25, 0.5, 1.0, 2.0], device="cuda")
    scratch = paged.attention_paged_scratch(cache, batch)
    out = paged.attention_paged(q, cache, t, batch, scale=0.125, slopes=slopes, scratch=scratch)
    k, v = (pool.view(-1, hd)[n - near:n][None] for pool in pools)  # beyond, the weights are below e^-900
    want, tol = paged_ref.attention(q, k, v, near - new[0], heads, 0.125, 0.0, slopes)
    assert paged_ref.within(out, want, tol, out.dtype), (out.cpu().double() - want).abs().max()
    assert cuda_lib_status(scratch) == 0


@pytest.mark.parametrize("past,new,heads,kv,hd,P", [
    ([40000], [1], 8, 1, 128, 128), ([30000, 70], [5, 1], 16, 2, 128, 16), ([9000], [3], 16, 2, 64, 32), ([20000], [16], 16, 2, 128, 64),
    ([0, 4000], [1500, 129], 4, 4, 64, 16), ([8100], [300], 8, 1, 128, 128)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_tile_counts_once(cuda_lib, past, new, heads, kv, hd, P, dtype):
    """Queries of zero weigh all positions alike, and a position's values are 1 in the
    dim that its run of 16 has: the outputs count positions, exactly but for the division."""
    from odiengine_b200 import paged

    s = Setup(past, new, heads, kv, hd, dtype, P)
    s.q.zero_()
    s.cache.v.zero_()
    for b in range(len(new)):
        j = torch.arange(past[b] + new[b], device="cuda")
        slot = s.tables.table[b].long()[j // P] * P + j % P
        s.cache.v[slot // P, :, slot % P, j // 16 % hd] = 1.0
    out = torch.empty(s.q.shape, dtype=torch.float32, device="cuda")
    paged.attention_paged(s.q, s.cache, s.tables, s.batch, out, scale=0.1, scratch=s.scratch)
    row = 0
    for b, N in enumerate(new):
        n = past[b] + N
        ones = torch.zeros((n, hd), dtype=torch.float64)
        ones[torch.arange(n), torch.arange(n) // 16 % hd] = 1.0
        upto = torch.arange(past[b] + 1, n + 1)
        want = ones.cumsum(0)[upto - 1] / upto[:, None]
        got = out[row:row + N].cpu().double().view(N, heads, hd)
        # a reciprocal and a product, each off by 2^-24; sums of whole numbers are exact
        assert ((got - want[:, None]).abs() <= 2.0 ** -22 * want[:, None]).all()
        row += N


# ---- lanes that part ways ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("past,new,heads,kv,hd", [([70], [45], 3, 3, 64), ([0, 130], [77, 40], 5, 1, 64), ([300], [260], 3, 3, 64),
                                                  ([90], [45], 3, 3, 128)])
@pytest.mark.parametrize("out32", [False, True])
def test_rows_that_end_inside_a_warp(cuda_lib, past, new, heads, kv, hd, out32):
    """Values that are not finite, which each row gets back for the positions that it
    sees, in items whose last warp has rows and lanes without one."""
    from odiengine_b200 import paged

    s = Setup(past, new, heads, kv, hd, "f16", 32)
    row = 0
    for N in new:
        for j, x in ((1, math.nan), (N // 3, math.inf), (N - 2, -math.inf)):
            slot = int(s.batch.slots[row + j])
            s.cache.v[slot // 32, :, slot % 32, (7 * j) % hd] = x
        row += N
    out = torch.empty(s.q.shape, dtype=torch.float32 if out32 else s.q.dtype, device="cuda")
    paged.attention_paged(s.q, s.cache, s.tables, s.batch, out, scale=0.1, scratch=s.scratch)
    s.check(out, 0.1)
    assert cuda_lib_status(s.scratch) == 0


@pytest.mark.parametrize("B,drops", [(300, 1), (300, 37), (1500, 9001), (2048, 8191)])
def test_steps_that_drop_any_number_of_pages(cuda_lib, B, drops):
    """Pages dropped by some lanes of some warps of a cluster, before the barrier that
    all of them share."""
    from odiengine_b200 import paged

    P, wide = 16, 8
    t = paged.PageTables.new(B, wide, B * wide, P)
    batch = paged.PagedBatch(t, max_rows=B * wide * P, max_new=wide * P, heads=4, kv_heads=4)
    ref = paged_ref.Tables(t.table.tolist(), t.lens.tolist(), t.free.tolist(), B * wide)
    full, each = [wide * P] * B, [drops // B + (b < drops % B) for b in range(B)]
    for new, keep in ((full, None), ([P + 1 if d > 1 else 0 for d in each], [(wide - min(d, wide)) * P for d in each]),
                      ([1] * B, [0] * B)):
        status, starts, lens, pos, slots = ref.step(P, new, keep, wide * P, B * wide * P)
        paged.paged_step(t, batch, ints(new), keep=None if keep is None else ints(keep))
        assert batch.status() == status == 0
        assert t.table.tolist() == ref.table and t.free.tolist() == ref.free and t.free_count.item() == ref.count
        assert batch.starts.tolist() == starts and batch.positions.tolist() == pos and batch.slots.tolist() == slots


# ---- tables that are not the step's ----------------------------------------------------------------------------------

@pytest.mark.parametrize("new", [[3, 1], [70, 40]])
@pytest.mark.parametrize("nan", [False, True])
def test_tables_narrower_than_the_steps(cuda_lib, new, nan):
    """A step made with tables of more pages per request: the pages that these do not
    have read as zeros, as ones that they do not name, and the error word says so."""
    from odiengine_b200 import paged

    heads, kv, hd, P, wide = 4, 1, 64, 32, 3
    s = Setup([200, 40], new, heads, kv, hd, "f16", P)
    assert s.tables.max_pages > wide
    if nan:  # a value behind the narrow table's end, and one before it
        for r in (1, new[0]):
            slot = int(s.batch.slots[r])
            s.cache.v[slot // P, :, slot % P, 5] = math.nan
    t = paged.PageTables(s.tables.table[:, :wide].contiguous(), s.tables.lens, s.tables.free, s.tables.free_count, P)
    out = paged.attention_paged(s.q, s.cache, t, s.batch, scale=0.1, scratch=s.scratch)
    assert cuda_lib_status(s.scratch) != 0
    s.scratch[:4].zero_()
    row = 0
    for b, N in enumerate(new):
        k, v = (s.rows(pool, b).clone() for pool in (s.cache.k, s.cache.v))
        k[:, wide * P:], v[:, wide * P:] = 0, 0
        want, tol = paged_ref.attention(s.q[row:row + N], k, v, s.past[b], heads, 0.1)
        assert paged_ref.within(out[row:row + N], want, tol, out.dtype)
        row += N


# ---- columns of one buffer -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("new", [[2, 1], [50, 20]])
def test_inputs_and_outputs_in_columns_of_one_buffer(cuda_lib, new):
    """Rows that lie between one another without sharing a byte are no overlap."""
    from odiengine_b200 import paged

    heads, kv, hd, T = 4, 2, 64, sum(new)
    s = Setup([100, 3], new, heads, kv, hd, "bf16", 32)
    w = heads * hd
    both = torch.full((T, 2 * w), math.nan, dtype=s.q.dtype, device="cuda")
    for q, out in ((both[:, :w], both[:, w:]), (both[:, w:], both[:, :w])):
        q.copy_(s.q)
        paged.attention_paged(q, s.cache, s.tables, s.batch, out, scale=0.1, scratch=s.scratch)
        assert torch.equal(q, s.q)
        s.check(out, 0.1)
    W = (heads + 2 * kv) * hd
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn((T, W), device="cuda", generator=g)
    want = paged.qk_rope_append_paged(qkv, s.cache, s.batch, heads=heads, theta=1e4)
    wide = torch.empty((T, W + w // 2), device="cuda")  # q as 16-bit values behind each row
    wide[:, :W] = qkv
    got = wide.view(torch.bfloat16)[:, 2 * W:]
    paged.qk_rope_append_paged(wide[:, :W], s.cache, s.batch, got, heads=heads, theta=1e4)
    assert torch.equal(got, want) and torch.equal(wide[:, :W], qkv)


# ---- who gets pages --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("B", [4, 300])
def test_requests_behind_one_without_pages(cuda_lib, B):
    """Five pages are free: the first request wants two, the second ten, and those after
    it one each or none.  The second is refused and with it who needs a page."""
    from odiengine_b200 import paged

    P = 16
    t = paged.PageTables.new(B, 12, 5 + B, P)
    batch = paged.PagedBatch(t, max_rows=1000 if B == 4 else 6000, max_new=160, heads=2, kv_heads=2)
    paged.paged_step(t, batch, ints([1 if b > 2 else 0 for b in range(B)]))
    free = 5 + B - (B - 3)
    t.free_count.fill_(5)
    new = [2 * P, 10 * P, 1] + [P - 1 if b % 2 else P for b in range(3, B)]  # the odd ones' page is there
    paged.paged_step(t, batch, ints(new))
    assert batch.status() == paged.NO_PAGES and free >= 5
    assert t.free_count.item() == 3
    served = [b == 0 or b > 2 and b % 2 == 1 for b in range(B)]
    had = [1 if b > 2 else 0 for b in range(B)]
    assert batch.lens.tolist() == [had[b] + new[b] if served[b] else 0 for b in range(B)]
    assert t.lens.tolist() == [had[b] + (new[b] if served[b] else 0) for b in range(B)]
    starts, slots = batch.starts.tolist(), batch.slots.tolist()
    for b in range(B):
        assert all((s >= 0) == served[b] for s in slots[starts[b]:starts[b + 1]]) and starts[b + 1] - starts[b] == new[b]


# ---- streams -----------------------------------------------------------------------------------------------------------

def test_the_status_of_a_step_on_another_stream(cuda_lib):
    """Read on the step's stream it is the step's, however late that runs."""
    from odiengine_b200 import paged

    t = paged.PageTables.new(2, 2, 3, 16)
    batch = paged.PagedBatch(t, max_rows=64, max_new=32, heads=1, kv_heads=1)
    side = torch.cuda.Stream()
    new = ints([20, 20])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    paged.paged_step(t, batch, new, stream=side)
    assert batch.status(side) == paged.NO_PAGES
