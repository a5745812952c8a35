"""The operators over a paged cache (odiengine_b200.paged) against plain
restatements on the host in 64 bits (paged_ref.py): one token to long chunks,
every page size, odd group sizes, ragged batches, requests that are refused,
values that are not finite where nobody looks, graphs and streams."""
import math

import numpy as np
import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Setup:
    """Tables, pages and one step of requests of the given past and new lengths."""

    def __init__(self, past, new, heads, kv, hd, dtype, P, seed=0, max_new=None, max_rows=None, spare=5, prefix=None, wide=0):
        from odiengine_b200 import paged

        g = torch.Generator(device="cuda").manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.past, self.new, self.heads, self.kv, self.hd, self.P = past, new, heads, kv, hd, P
        B, T = len(new), sum(new)
        count = [-(-(a + n) // P) for a, n in zip(past, new)]
        pages = sum(count) + spare
        dt = DTYPES[dtype]
        mk = lambda: torch.randn((pages, kv, P, hd), device="cuda", generator=g).to(dt)  # noqa: E731
        self.cache = paged.PagedCache(mk(), mk())
        self.tables = paged.PageTables.new(B, max(1, wide, max(count)), pages, P)
        self.tables.free.copy_(ints(rng.permutation(pages).tolist()))
        self.batch = paged.PagedBatch(self.tables, max_rows=max_rows or max(1, T), max_new=max_new or max(1, max(new)),
                                      heads=heads, kv_heads=kv)
        self.prefix = prefix
        # the past comes in a step of its own
        first = paged.PagedBatch(self.tables, max_rows=max(1, sum(past)), max_new=max(1, max(past)), heads=heads, kv_heads=kv)
        paged.paged_step(self.tables, first, ints(past))
        assert first.status() == 0
        paged.paged_step(self.tables, self.batch, ints(new), prefix=None if prefix is None else ints(prefix))
        assert self.batch.status() == 0
        self.q = (torch.randn((T, heads * hd), device="cuda", generator=g) * 1.5).to(dt)
        self.scratch = paged.attention_paged_scratch(self.cache, self.batch)

    def rows(self, pool, b):
        n = self.past[b] + self.new[b]
        at = self.tables.table[b, :-(-n // self.P)].long() if n else torch.zeros(0, dtype=torch.long, device="cuda")
        return pool[at].transpose(0, 1).reshape(self.kv, -1, self.hd)[:, :n]

    def check(self, out, scale, softcap=0.0, slopes=None, only=None):
        row = 0
        for b, N in enumerate(self.new):
            if N and (only is None or b in only):
                want, tol = paged_ref.attention(self.q[row:row + N], self.rows(self.cache.k, b), self.rows(self.cache.v, b),
                                                self.past[b], self.heads, scale, softcap, slopes,
                                                0 if self.prefix is None else self.prefix[b])
                got = out[row:row + N]
                assert paged_ref.within(got, want, tol, got.dtype), (b, (got.cpu().double() - want).abs().max(), tol.max())
            row += N


# ---- step -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("B,P,wide,max_new,max_rows,seed", [
    (1, 16, 4, 40, 40, 0), (5, 32, 3, 9, 30, 1), (40, 16, 20, 33, 700, 2), (130, 128, 3, 300, 5000, 3), (1500, 16, 9, 60, 40000, 4),
    (2048, 64, 2, 1, 2048, 5), (7, 16, 40, 600, 2500, 6)])
def test_steps_follow_the_lists(cuda_lib, B, P, wide, max_new, max_rows, seed):
    """Steps of random lengths, with requests that are too long, too many, keep
    what they do not have, or find no page: tables, free list, rows and status
    are those of the plain lists, step after step."""
    from odiengine_b200 import paged

    rng = np.random.default_rng(seed)
    pages = max(2, B * wide * 2 // 3)
    t = paged.PageTables.new(B, wide, pages, P)
    batch = paged.PagedBatch(t, max_rows=max_rows, max_new=max_new, heads=8, kv_heads=2)
    ref = paged_ref.Tables(t.table.tolist(), t.lens.tolist(), t.free.tolist(), pages)
    seen = 0
    for step in range(8):
        new = rng.integers(0, max_new + 1, B)
        new[rng.random(B) < 0.3] = 0
        keep = np.array([rng.integers(0, n + 1) if rng.random() < 0.5 else n for n in ref.lens])
        if step % 2:
            new[rng.random(B) < 0.05] = max_new + 1
            new[rng.random(B) < 0.05] = -3
            keep[rng.random(B) < 0.1] = wide * P + 7
            keep[rng.random(B) < 0.05] = -1
        use = None if step == 4 else keep.tolist()
        status, starts, lens, pos, slots = ref.step(P, new.tolist(), use, max_new, max_rows)
        paged.paged_step(t, batch, ints(new.tolist()), keep=None if use is None else ints(use))
        assert batch.status() == status
        seen |= status
        assert t.table.tolist() == ref.table and t.lens.tolist() == ref.lens
        assert t.free_count.item() == ref.count and t.free.tolist() == ref.free
        assert batch.starts.tolist() == starts and batch.lens.tolist() == lens
        assert batch.positions.tolist() == pos and batch.slots.tolist() == slots
        held = [p for r in ref.table for p in r if p >= 0] + ref.free[:ref.count]
        assert sorted(held) == list(range(pages))  # no page is lost or held twice
    assert B < 40 or (seen & 4 and seen & 16)


def test_lengths_out_of_range_are_brought_in(cuda_lib):
    from odiengine_b200 import paged

    t = paged.PageTables.new(3, 2, 9, 16)
    b = paged.PagedBatch(t, max_rows=9, max_new=9, heads=1, kv_heads=1)
    t.lens.copy_(ints([-5, 0, 1000]))
    t.free_count.fill_(6)
    ref = paged_ref.Tables(t.table.tolist(), [-5, 0, 1000], t.free.tolist(), 6)
    want = ref.step(16, [3, 3, 3], [0, 0, 0], 9, 9)
    paged.paged_step(t, b, ints([3, 3, 3]), keep=ints([0, 0, 0]))
    assert b.status() == want[0] == 32 and t.lens.tolist() == [3, 3, 3] and b.lens.tolist() == [3, 3, 3]
    # the third request's table named no pages (-1): two of them went onto the list and came back first
    assert b.slots.tolist() == [s if s >= 0 else -1 for s in want[4]]


# ---- append -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("past,new,heads,kv,hd,dtype,P,norm,theta", [
    ([0], [1], 4, 4, 128, "f16", 16, True, 1e4), ([7, 0, 100], [3, 5, 1], 6, 2, 64, "bf16", 32, True, 1e4),
    ([5000, 15], [200, 33], 16, 8, 128, "bf16", 128, False, 5e5), ([0, 0, 130000], [64, 1, 17], 8, 1, 64, "f16", 64, False, 5e5),
    ([31], [2], 5, 5, 128, "f16", 16, True, 1e4)])
@pytest.mark.parametrize("padded", [False, True])
def test_append(cuda_lib, past, new, heads, kv, hd, dtype, P, norm, theta, padded):
    """Against 64 bits.  fp32 arithmetic leaves 2e-6 of a pair's length (angle
    2^-24 of a turn, its sine, the norm's sum and root); then one rounding."""
    from odiengine_b200 import paged

    T, W = sum(new), (heads + 2 * kv) * hd
    s = Setup(past, new, heads, kv, hd, dtype, P, max_rows=T + 3)
    g = torch.Generator(device="cuda").manual_seed(1)
    extra = 3 if padded else 0
    wide = torch.randn((T + extra, W + (5 if padded else 0)), device="cuda", generator=g) * 1.5
    qkv = wide[:, :W]
    qn, kn = ((1 + 0.1 * torch.randn(hd, device="cuda", generator=g)) if norm else None for _ in range(2))
    q_wide = torch.full((T + extra, heads * hd + (2 if padded else 0)), 7.0, dtype=s.cache.dtype, device="cuda")
    q = q_wide[:, :heads * hd]
    k0, v0 = s.cache.k.clone(), s.cache.v.clone()
    paged.qk_rope_append_paged(qkv, s.cache, s.batch, q, heads=heads, theta=theta, q_norm=qn, k_norm=kn, eps=1e-6)
    pos = torch.tensor([past[b] + j for b in range(len(new)) for j in range(new[b])], dtype=torch.float64)
    x = qkv[:T].cpu().double().view(T, heads + 2 * kv, hd)
    i = torch.arange(hd // 2, dtype=torch.float64)
    a = (pos[:, None] * float(np.float32(theta)) ** (-2.0 * i / hd))[:, None]

    def turn(u, w):
        if w is not None:
            u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + float(np.float32(1e-6))) * w.cpu().double()
        lo, hi = u[..., :hd // 2], u[..., hd // 2:]
        out = torch.cat([lo * torch.cos(a) - hi * torch.sin(a), lo * torch.sin(a) + hi * torch.cos(a)], -1)
        size = torch.hypot(lo, hi)
        return out, 2e-6 * torch.cat([size, size], -1)

    want, tol = turn(x[:, :heads], qn)
    assert paged_ref.within(q[:T].reshape(T, heads, hd), want, tol, q.dtype)
    if padded:  # rows behind the last, and the gaps, are as they were
        assert (q_wide[T:] == 7).all() and (q_wide[:, heads * hd:] == 7).all()
    slots = s.batch.slots[:T].long()
    kw, kt = turn(x[:, heads:heads + kv], kn)
    got_k = s.cache.k[slots // P, :, slots % P]
    got_v = s.cache.v[slots // P, :, slots % P]
    assert paged_ref.within(got_k, kw, kt, q.dtype)
    assert torch.equal(got_v.cpu(), x[:, heads + kv:].to(q.dtype))
    # no other row of the pool changed
    other = torch.ones(s.cache.num_pages * P, dtype=torch.bool, device="cuda")
    other[slots] = False
    for now, was in ((s.cache.k, k0), (s.cache.v, v0)):
        flat = lambda t: t.transpose(1, 2).reshape(-1, kv, hd)[other]  # noqa: E731
        assert torch.equal(flat(now), flat(was))


# ---- attention ----------------------------------------------------------------------------------------------------

SHAPES = [
    # past, new, heads, kv, hd, dtype, page
    ([0], [1], 1, 1, 64, "f16", 16),
    ([517], [1], 32, 32, 128, "f16", 16),
    ([63, 64, 65, 0, 1000], [1, 1, 1, 1, 1], 8, 2, 128, "bf16", 64),
    ([15, 300], [4, 1], 12, 4, 64, "bf16", 32),
    ([100, 7], [5, 2], 21, 3, 128, "f16", 128),
    ([40000], [1], 8, 1, 128, "bf16", 128),
    ([9, 2000], [3, 5], 16, 4, 64, "f16", 16),
    ([0, 200, 31], [40, 70, 9], 10, 2, 128, "f16", 32),
    ([0], [129], 4, 4, 64, "bf16", 16),
    ([250, 0, 77], [300, 513, 130], 8, 1, 128, "bf16", 64),
    ([3, 120], [257, 31], 7, 7, 128, "f16", 128),
    ([1000, 0], [64, 0], 64, 1, 64, "f16", 16),
    ([2900], [150], 6, 2, 64, "bf16", 32),
]


@pytest.mark.parametrize("past,new,heads,kv,hd,dtype,P", SHAPES)
@pytest.mark.parametrize("option", ["plain", "cap", "slopes", "prefix", "all", "out32"])
def test_attention(cuda_lib, past, new, heads, kv, hd, dtype, P, option):
    from odiengine_b200 import paged

    prefix = [(a + n) // 2 + 1 for a, n in zip(past, new)] if option in ("prefix", "all") else None
    s = Setup(past, new, heads, kv, hd, dtype, P, prefix=prefix)
    slopes = (0.3 * torch.rand(heads, device="cuda") + 0.01) if option in ("slopes", "all") else None
    cap = 3.0 if option in ("cap", "all") else 0.0
    scale = 1 / math.sqrt(hd)
    out = torch.empty((sum(new), heads * hd), dtype=torch.float32 if option == "out32" else s.cache.dtype, device="cuda")
    paged.attention_paged(s.q, s.cache, s.tables, s.batch, out, scale=scale, softcap=cap, slopes=slopes, scratch=s.scratch)
    s.check(out, scale, cap, slopes)
    again = torch.empty_like(out)
    paged.attention_paged(s.q, s.cache, s.tables, s.batch, again, scale=scale, softcap=cap, slopes=slopes, scratch=s.scratch)
    assert torch.equal(out, again)  # bit for bit
    assert cuda_lib_status(s.scratch) == 0


@pytest.mark.parametrize("past,new,heads,kv,hd,dtype,P", [([4000], [200], 64, 64, 64, "f16", 16), ([3500], [70], 96, 48, 128, "bf16", 64)])
@pytest.mark.parametrize("option", ["slopes", "all"])
def test_attention_long_pieces_with_a_bias(cuda_lib, past, new, heads, kv, hd, dtype, P, option):
    """Steep and flat biases over runs of tiles long enough to go from the last tile
    to the first; a NaN among the new tokens' values."""
    from odiengine_b200 import paged

    s = Setup(past, new, heads, kv, hd, dtype, P, prefix=[past[0] + 20] if option == "all" else None)
    slot = int(s.batch.slots[new[0] // 2])
    s.cache.v[slot // P, :, slot % P, 3] = math.nan
    slopes = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
    out = paged.attention_paged(s.q, s.cache, s.tables, s.batch, scale=1 / math.sqrt(hd), slopes=slopes, scratch=s.scratch)
    s.check(out, 1 / math.sqrt(hd), 0.0, slopes)
    assert cuda_lib_status(s.scratch) == 0


@pytest.mark.parametrize("new", [[2, 1], [9, 5], [40, 90]])
@pytest.mark.parametrize("heads", [4, 6])
@pytest.mark.parametrize("shift,pad", [(2, 0), (0, 6), (2, 2)])
def test_attention_of_rows_that_are_not_aligned(cuda_lib, new, heads, shift, pad):
    """Queries and outputs on 4-byte boundaries, at odd strides."""
    from odiengine_b200 import paged

    s = Setup([100, 3], new, heads, 2, 128, "bf16", 32)
    T, w = s.q.shape
    wide = torch.full((T, w + shift + pad), math.nan, dtype=s.q.dtype, device="cuda")
    q = wide[:, shift:shift + w]
    q.copy_(s.q)
    out = torch.full((T, w + shift + pad), 5.0, dtype=s.q.dtype, device="cuda")
    paged.attention_paged(q, s.cache, s.tables, s.batch, out[:, shift:shift + w], scale=0.09, scratch=s.scratch)
    s.check(out[:, shift:shift + w], 0.09)
    assert (out[:, :shift] == 5).all() and (out[:, shift + w:] == 5).all()


@pytest.mark.parametrize("new,heads,kv", [(1, 3, 3), (2, 8, 1), (3, 8, 1), (9, 10, 1), (40, 8, 1), (1, 1, 1)])
@pytest.mark.parametrize("hd,dtype", [(64, "bf16"), (128, "f16")])
@pytest.mark.parametrize("past", [3300, 9000])
def test_attention_of_many_pieces(cuda_lib, new, heads, kv, hd, dtype, past):
    """One request whose few heads are cut into dozens of pieces, which join in
    groups; a NaN that the last rows see, and calls that follow one another."""
    from odiengine_b200 import paged

    s = Setup([past], [new], heads, kv, hd, dtype, 64, seed=past + new)
    slopes = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
    scale = 1 / math.sqrt(hd)
    for option in (None, slopes):
        out = torch.empty((new, heads * hd), dtype=torch.float32, device="cuda")
        paged.attention_paged(s.q, s.cache, s.tables, s.batch, out, scale=scale, slopes=option, scratch=s.scratch)
        s.check(out, scale, 0.0, option)
        again = torch.empty_like(out)
        paged.attention_paged(s.q, s.cache, s.tables, s.batch, again, scale=scale, slopes=option, scratch=s.scratch)
        assert torch.equal(out, again)
    slot = int(s.batch.slots[new - 1])
    s.cache.v[slot // 64, :, slot % 64, 5] = math.nan
    paged.attention_paged(s.q, s.cache, s.tables, s.batch, again, scale=scale, slopes=slopes, scratch=s.scratch)
    assert torch.equal(out[:-1], again[:-1])
    assert again[-1].view(heads, hd)[:, 5].isnan().all() and again[-1].isnan().sum() == heads
    assert cuda_lib_status(s.scratch) == 0 and not s.scratch[-4 * kv:].any()


def cuda_lib_status(scratch):
    return int(scratch[:4].view(torch.int32).item())


@pytest.mark.parametrize("past,new,heads,kv,hd,P", [
    ([100, 30], [6, 1], 4, 2, 128, 16), ([5, 400], [90, 200], 8, 2, 128, 64), ([70], [9], 16, 1, 64, 32), ([300], [260], 3, 3, 64, 128)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_values_that_are_not_finite_reach_only_who_sees_them(cuda_lib, past, new, heads, kv, hd, P, dtype):
    """NaN and infinities in every row that no request holds, and V's of some new
    tokens: rows before those tokens do not change."""
    from odiengine_b200 import paged

    s = Setup(past, new, heads, kv, hd, dtype, P)
    held = torch.zeros(s.cache.num_pages * P, dtype=torch.bool, device="cuda")
    for b in range(len(new)):
        n = past[b] + new[b]
        j = torch.arange(n, device="cuda")
        held[s.tables.table[b].long()[j // P] * P + j % P] = True
    for pool in (s.cache.k, s.cache.v):
        flat = pool.transpose(1, 2).reshape(-1, kv, hd)
        junk = torch.tensor([math.nan, math.inf, -math.inf], device="cuda").to(pool.dtype)[torch.randint(0, 3, flat.shape, device="cuda")]
        flat = torch.where(held[:, None, None], flat, junk)
        pool.copy_(flat.view(-1, P, kv, hd).transpose(1, 2))
    row = 0
    for b, N in enumerate(new):  # the middle and last new tokens' values
        for j, x in ((N // 2, math.nan), (N - 1, math.inf), (max(0, N - 2), -math.inf)):
            slot = int(s.batch.slots[row + j])
            s.cache.v[slot // P, :, slot % P, j % hd] = x
        row += N
    scale = 1 / math.sqrt(hd)
    out = paged.attention_paged(s.q, s.cache, s.tables, s.batch, scale=scale, scratch=s.scratch)
    s.check(out, scale)


def test_scores_that_are_not_finite(cuda_lib):
    """A NaN query, a key of NaN and one of infinity: as softmax has it, for the
    rows that meet them and no others."""
    from odiengine_b200 import paged

    for new in ([4, 3, 2], [40, 50, 20]):
        s = Setup([50, 60, 70], new, 4, 2, 64, "bf16", 16)
        s.q[1] = math.nan
        slot = int(s.batch.slots[new[0] + new[1] - 1])  # the second request's last key
        s.cache.k[slot // 16, :, slot % 16] = math.nan
        out = paged.attention_paged(s.q, s.cache, s.tables, s.batch, scale=0.125, scratch=s.scratch).float()
        bad = torch.isnan(out).all(1)
        want = torch.zeros(sum(new), dtype=torch.bool, device="cuda")
        want[1] = want[new[0] + new[1] - 1] = True
        assert torch.equal(bad, want) and torch.equal(torch.isnan(out).any(1), want)
        s.check(out.to(s.cache.dtype), 0.125, only=[2])


@pytest.mark.parametrize("new", [[1, 0, 2], [40, 0, 33]])
def test_rows_behind_the_last_and_of_refused_requests_are_left(cuda_lib, new):
    from odiengine_b200 import paged

    heads, kv, hd, P = 8, 4, 64, 16
    s = Setup([20, 0, 33], new, heads, kv, hd, "f16", P, max_rows=sum(new) + 90, max_new=60, spare=0, wide=8)
    T = sum(new)
    q = torch.cat([s.q, torch.full((4, heads * hd), math.nan, dtype=s.q.dtype, device="cuda")])
    out = torch.full((T + 4, heads * hd + 2), 5.0, dtype=s.q.dtype, device="cuda")
    paged.attention_paged(q, s.cache, s.tables, s.batch, out[:, :-2], scale=0.125, scratch=s.scratch)
    s.check(out[:T, :-2], 0.125)
    assert (out[T:] == 5).all() and (out[:, -2:] == 5).all()
    # the same lengths again, and a request for pages that are not there
    held = [a + n for a, n in zip(s.past, new)]
    paged.paged_step(s.tables, s.batch, ints([new[0], 50, new[2]]), keep=ints([20, 0, 33]))
    assert s.batch.status() == paged.NO_PAGES
    assert s.batch.lens.tolist() == [held[0], 0, 0 if -(-held[2] // P) > -(-33 // P) else held[2]]
    out.fill_(5.0)
    T = new[0] + 50 + new[2]
    q = torch.zeros((T, heads * hd), dtype=s.q.dtype, device="cuda")
    q[:new[0]] = s.q[:new[0]]
    out = torch.full((T, heads * hd), 5.0, dtype=s.q.dtype, device="cuda")
    paged.attention_paged(q, s.cache, s.tables, s.batch, out, scale=0.125, scratch=s.scratch)
    s.check(out, 0.125, only=[0])
    assert (out[new[0]:new[0] + 50] == 5).all()
    # fewer rows handed in than the batch has: the others are not touched
    few = torch.full((2, heads * hd), 5.0, dtype=s.q.dtype, device="cuda")
    paged.attention_paged(q[:1], s.cache, s.tables, s.batch, few[:1], scale=0.125, scratch=s.scratch)
    assert (few[1] == 5).all() and torch.equal(few[0], out[0])


@pytest.mark.parametrize("new", [[3], [70]])
def test_pages_that_a_table_does_not_name_read_as_zeros(cuda_lib, new):
    from odiengine_b200 import paged

    s = Setup([100], new, 4, 1, 128, "bf16", 32)
    s.tables.table[0, 1] = s.cache.num_pages + 3
    s.tables.table[0, 2] = -7
    out = paged.attention_paged(s.q, s.cache, s.tables, s.batch, scale=0.1, scratch=s.scratch)
    assert cuda_lib_status(s.scratch) != 0
    s.scratch[:4].zero_()
    k, v = (torch.cat([p, torch.zeros_like(p[:1])]) for p in (s.cache.k, s.cache.v))
    s.tables.table[0, 1:3] = s.cache.num_pages
    want, tol = paged_ref.attention(s.q, s.rows(k, 0), s.rows(v, 0), 100, 4, 0.1)
    assert paged_ref.within(out, want, tol, out.dtype)


@pytest.mark.parametrize("new", [[1, 2, 1], [20, 90, 33]])
def test_steps_captured_and_replayed(cuda_lib, new):
    """Step, append and attention in one graph, replayed with other lengths; two
    graphs over one scratch; another stream."""
    from odiengine_b200 import paged

    heads, kv, hd, P = 8, 2, 128, 16
    past = [10, 0, 64]
    s = Setup(past, new, heads, kv, hd, "bf16", P, max_rows=200, max_new=100, spare=60)
    t = paged.PageTables.new(3, 40, 120, P)
    batch = paged.PagedBatch(t, max_rows=200, max_new=100, heads=heads, kv_heads=kv)
    cache = paged.PagedCache.new(torch.bfloat16, 120, kv, P, hd)
    scratch = paged.attention_paged_scratch(cache, batch)
    keep, fresh = ints([0, 0, 0]), ints(new)
    qkv = torch.randn((200, (heads + 2 * kv) * hd), device="cuda")
    q = torch.zeros((200, heads * hd), dtype=torch.bfloat16, device="cuda")
    outs = [torch.zeros_like(q) for _ in range(2)]

    def work(out):
        paged.paged_step(t, batch, fresh, keep=keep)
        paged.qk_rope_append_paged(qkv, cache, batch, q, heads=heads, theta=1e4)
        paged.attention_paged(q, cache, t, batch, out, scale=0.09, scratch=scratch)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        work(outs[0])
        for out in outs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                work(out)
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    for k0, n0 in (([0, 0, 0], new), ([5, 0, 1], [min(100, n + 3) for n in new]), ([1, 1, 1], [1, 0, 1])):
        paged.paged_step(t, batch, ints(k0), keep=ints([0, 0, 0]))  # that many positions hold what they hold
        keep.copy_(ints(k0))
        fresh.copy_(ints(n0))
        got = []
        for g, out in zip(graphs, outs):
            out.fill_(3.0)
            g.replay()
            got.append(out.clone())
        torch.cuda.synchronize()
        ref = torch.full_like(q, 3.0)
        work(ref)
        assert torch.equal(got[0], ref) and torch.equal(got[1], ref)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            other = torch.full_like(q, 3.0)
            paged.attention_paged(q, cache, t, batch, other, scale=0.09, scratch=scratch, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(other, ref)
        s.past, s.new, s.tables, s.cache, s.batch, s.q = k0, n0, t, cache, batch, q
        s.check(ref[:sum(n0)], 0.09)
    assert cuda_lib_status(scratch) == 0


def test_pools_past_32_bits(cuda_lib):
    """A pool of more than 2^31 values, the last pages in use."""
    from odiengine_b200 import paged

    P, kv, hd = 128, 8, 128
    pages = (1 << 31) // (P * kv * hd) + 40
    cache = paged.PagedCache(*(torch.zeros((pages, kv, P, hd), dtype=torch.float16, device="cuda") for _ in range(2)))
    for new in ([2], [150]):
        t = paged.PageTables.new(1, 8, pages, P)
        t.free.copy_(torch.arange(pages, dtype=torch.int32, device="cuda"))  # the last page first
        b = paged.PagedBatch(t, max_rows=1000, max_new=500, heads=8, kv_heads=kv)
        small = paged.PagedBatch(t, max_rows=new[0], max_new=new[0], heads=8, kv_heads=kv)
        paged.paged_step(t, b, ints([300]))
        g = torch.Generator(device="cuda").manual_seed(3)
        q = torch.empty((300, 8 * hd), dtype=torch.float16, device="cuda")
        paged.qk_rope_append_paged(torch.randn((300, 24 * hd), device="cuda", generator=g), cache, b, q, heads=8, theta=1e4)
        paged.paged_step(t, small, ints(new))
        q = torch.randn((new[0], 8 * hd), device="cuda", generator=g).half()
        paged.qk_rope_append_paged(torch.randn((new[0], 24 * hd), device="cuda", generator=g), cache, small, torch.empty_like(q), heads=8, theta=1e4)
        assert int(small.slots.max()) * kv * hd > 1 << 31
        out = paged.attention_paged(q, cache, t, small, scale=0.09, scratch=paged.attention_paged_scratch(cache, small))
        n = 300 + new[0]
        rows = [p[t.table[0, :-(-n // P)].long()].transpose(0, 1).reshape(kv, -1, hd)[:, :n] for p in (cache.k, cache.v)]
        want, tol = paged_ref.attention(q, *rows, 300, 8, 0.09)
        assert rows[0].abs().min(-1)[0].max() > 0 and paged_ref.within(out, want, tol, out.dtype)


# ---- verify -------------------------------------------------------------------------------------------------------

def verify_case(R, V, seed, probs, sharp=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn((R, V), device="cuda", generator=g) * 3
    draft = logits + torch.randn((R, V), device="cuda", generator=g) * sharp
    p = torch.softmax(draft, -1) if probs else None
    chosen = torch.multinomial(p, 1, generator=g)[:, 0] if probs else draft.argmax(-1)
    u = torch.rand(R, device="cuda", generator=g), torch.rand(R, device="cuda", generator=g)
    return logits, chosen.roll(1).int(), p, u


@pytest.mark.parametrize("new,V", [([1], 7), ([5], 100), ([3, 1, 8, 2], 2047), ([4, 0, 6], 2048), ([9, 17], 2049), ([2, 40], 32000),
                                   ([6, 5, 1], 128259)])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temperature", [0.3, 1.0, 1.7])
def test_verify(cuda_lib, new, V, probs, temperature):
    from odiengine_b200 import paged

    R, B = sum(new), len(new)
    starts = [sum(new[:i]) for i in range(B + 1)]
    scratch = paged.verify_scratch(R, B, V)
    kept = 0
    for seed in range(4):
        logits, tokens, p, (ua, un) = verify_case(R, V, seed, probs, sharp=0.3)
        if seed == 1:
            un = torch.zeros_like(un)
        if seed == 2:  # the largest number below 1, and drafts outside the vocabulary
            un = torch.full_like(un, 1 - 2.0 ** -24)
            tokens[::3] = -1
            tokens[1::3] = V
        got = paged.verify_sampled(logits, tokens, ints(starts), ua, un[:B].contiguous(), temperature=temperature, draft_probs=p, scratch=scratch)
        want = paged_ref.verify(logits.cpu().numpy(), tokens.tolist(), starts, ua.tolist(), un.tolist(), temperature,
                                None if p is None else p.cpu().numpy())
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1], (seed, got, want)
        kept += sum(want[0])
    assert kept or temperature > 1 or max(new) < 3


def test_verify_odd_rows(cuda_lib):
    """Masked rows, rows of one token, infinities, NaN, p equal to q, a padded
    batch, strides; a scratch that larger calls used before."""
    from odiengine_b200 import paged

    V, inf = 3001, math.inf
    scratch = paged.verify_scratch(64, 8, 50000)
    big = verify_case(64, 50000, 0, False)
    paged.verify_sampled(big[0], big[1], ints([0, 10, 64]), big[3][0], big[3][1][:2].contiguous(), scratch=scratch)
    logits, tokens, p, (ua, un) = verify_case(16, V, 5, True)
    logits[2, 1:] = -inf                 # one token
    logits[4] = -inf                     # none
    logits[6, 17] = math.nan
    logits[8, 40] = logits[8, 2900] = inf
    p[10] = torch.softmax(logits[10], -1)  # nothing left but rounding
    tokens[11] = int(p[10].argmax())
    ua[10] = 0.999
    tokens[3] = 0
    starts = [0, 2, 4, 6, 8, 10, 13, 13, 15]
    wide = torch.full((16, V + 6), 9.0, device="cuda")
    wide[:, 1:V + 1] = logits
    for q in (None, p):
        got = paged.verify_sampled(wide[:, 1:V + 1], tokens, ints(starts), ua, un[:8].contiguous(), draft_probs=q, scratch=scratch)
        want = paged_ref.verify(logits.cpu().numpy(), tokens.tolist(), starts, ua.tolist(), un.tolist(), 1.0,
                                None if q is None else q.cpu().numpy())
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1], (got, want)
        assert got[1].tolist()[2] == -1 and got[1].tolist()[6] == -1


def test_verify_keeps_the_targets_distribution(cuda_lib):
    """40,000 first tokens after a draft from another distribution: their counts
    are the target's within five standard deviations of each."""
    from odiengine_b200 import paged

    n, V = 8000, 11
    g = torch.Generator(device="cuda").manual_seed(1)
    target, drafter = torch.randn(V, device="cuda", generator=g), torch.softmax(torch.randn(V, device="cuda", generator=g), -1)
    scratch = paged.verify_scratch(2 * n, n, V)
    counts = torch.zeros(V, dtype=torch.long)
    logits, probs = target.repeat(2 * n, 1).contiguous(), drafter.repeat(2 * n, 1).contiguous()
    for _ in range(5):
        draft = torch.multinomial(drafter.expand(n, V), 1, generator=g)[:, 0].int()
        tokens = torch.stack([torch.zeros_like(draft), draft], 1).flatten().contiguous()
        acc, nxt = paged.verify_sampled(logits, tokens, 2 * torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                                        torch.rand(2 * n, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g),
                                        draft_probs=probs, scratch=scratch)
        counts += torch.bincount(torch.where(acc > 0, draft, nxt).cpu().long(), minlength=V)
    p = torch.softmax(target, -1).cpu().double()
    N = 5 * n
    assert ((counts - N * p).abs() <= 5 * torch.sqrt(N * p * (1 - p))).all(), (counts, N * p)


def test_verify_captured(cuda_lib):
    from odiengine_b200 import paged

    logits, tokens, p, (ua, un) = verify_case(12, 5000, 9, True)
    starts, un = ints([0, 4, 4, 12]), un[:3].contiguous()
    scratch = paged.verify_scratch(12, 3, 5000)
    acc, nxt = ints([0] * 3), ints([0] * 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            paged.verify_sampled(logits, tokens, starts, ua, un, acc, nxt, draft_probs=p, scratch=scratch)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (9, 10):
        fresh = verify_case(12, 5000, seed, True)
        logits.copy_(fresh[0]), tokens.copy_(fresh[1]), p.copy_(fresh[2]), ua.copy_(fresh[3][0]), un.copy_(fresh[3][1][:3])
        for _ in range(3):
            g.replay()
        want = paged_ref.verify(logits.cpu().numpy(), tokens.tolist(), [0, 4, 4, 12], ua.tolist(), un.tolist(), 1.0, p.cpu().numpy())
        assert acc.tolist() == want[0] and nxt.tolist() == want[1]
