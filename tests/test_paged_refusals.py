"""The operators over a paged cache refuse what they cannot do, on the host and
before any launch: sizes, types, strides, alignment, overlaps.  No GPU needed
(the pointers below are never followed)."""
import ctypes

import pytest
import torch

import odiengine_b200 as ob
from odiengine_b200 import paged

INVALID, DTYPE = 2, 202
A, B, C = 0x10000, 0x20000000, 0x40000000  # aligned addresses of nothing


def cache(k=A, v=B, dtype=0, kv_heads=2, head_dim=128, page_size=16, num_pages=10):
    return paged._CacheStruct(k, v, dtype, kv_heads, head_dim, page_size, num_pages)


def tables(table=A, lens=A, free=A, count=A, requests=3, max_pages=4, page_size=16, num_pages=10):
    return paged._TablesStruct(table, lens, free, count, requests, max_pages, page_size, num_pages)


def batch(starts=A, lens=A, positions=A, slots=A, work=A, requests=3, max_rows=40, max_new=20, heads=6, kv_heads=2, page_size=16):
    return paged._BatchStruct(starts, lens, positions, slots, work, requests, max_rows, max_new, heads, kv_heads, page_size)


def refused(rc, code=INVALID, word=None):
    assert rc == code
    msg = ob.lib().odi_cuda_last_error().decode()
    assert msg and (word is None or word in msg), msg


BAD_BATCHES = [dict(starts=None), dict(lens=None), dict(positions=None), dict(slots=None), dict(work=None), dict(work=A + 4),
               dict(starts=A + 2), dict(slots=A + 1), dict(requests=0), dict(requests=2049), dict(max_rows=0), dict(max_rows=262145),
               dict(max_new=0), dict(max_new=41), dict(heads=5), dict(heads=0), dict(kv_heads=0), dict(heads=130), dict(page_size=24),
               dict(kv_heads=1025, heads=1025)]
BAD_CACHES = [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(k=A + 8), INVALID), (dict(dtype=2), DTYPE), (dict(dtype=-1), DTYPE),
              (dict(head_dim=96), INVALID), (dict(head_dim=256), INVALID), (dict(kv_heads=0), INVALID), (dict(page_size=8), INVALID),
              (dict(page_size=48), INVALID), (dict(num_pages=0), INVALID), (dict(num_pages=1 << 30), INVALID), (dict(v=A), INVALID),
              (dict(v=A + 10 * 2 * 16 * 128 * 2 - 16), INVALID)]


def step(t=None, b=None, keep=None, new=A, prefix=None):
    t, b = tables() if t is None else t, batch() if b is None else b
    return ob.lib().odi_cuda_paged_step(ctypes.byref(t), ctypes.byref(b), keep, new, prefix, None)


def append(c=None, b=None, qkv=A, ld=1280, out=C, ldq=768, T=4, H=6, theta=1e4, qn=None, kn=None):
    c, b = cache() if c is None else c, batch() if b is None else b
    return ob.lib().odi_cuda_qk_rope_append_paged(qkv, ld, qn, kn, 1e-6, out, ldq, ctypes.byref(c), ctypes.byref(b), T, H, theta, None)


NEED = ob.lib().odi_cuda_attention_paged_scratch_bytes(3, 40, 20, 6, 2, 128)


def attend(c=None, t=None, b=None, q=A, ld=768, out=C, ldo=768, kind=0, T=4, scale=1.0, cap=0.0, slopes=None, scr=A, n=None):
    c, t, b = cache() if c is None else c, tables() if t is None else t, batch() if b is None else b
    return ob.lib().odi_cuda_attention_paged(q, ld, ctypes.byref(c), ctypes.byref(t), ctypes.byref(b), out, ldo, kind, T, scale, cap,
                                             slopes, scr, NEED if n is None else n, None)


def test_work_and_scratch_bytes():
    L = ob.lib()
    assert L.odi_cuda_paged_work_bytes(3, 40, 20, 6, 2) > 0 and NEED > 0
    for a in ((0, 40, 20, 6, 2), (2049, 40, 20, 6, 2), (3, 0, 1, 6, 2), (3, 40, 41, 6, 2), (3, 40, 20, 5, 2), (3, 40, 20, 6, 0),
              (3, 262145, 1, 6, 2), (3, 40, 0, 6, 2), (3, 40, 20, 65, 1)):
        assert L.odi_cuda_paged_work_bytes(*a) == 0 and L.odi_cuda_attention_paged_scratch_bytes(*a, 128) == 0
    assert L.odi_cuda_attention_paged_scratch_bytes(3, 40, 20, 6, 2, 96) == 0
    # the largest batch there is: every item has its words
    assert L.odi_cuda_paged_work_bytes(2048, 262144, 262144, 64, 1) >= 4 * 3 * (262144 * 64 // 256)
    for a in ((0, 1, 10), (65536, 1, 10), (1, 0, 10), (1, 16385, 10), (1, 1, 0), (1, 1, 0x7fff0001)):
        assert L.odi_cuda_verify_scratch_bytes(*a) == 0
    assert L.odi_cuda_verify_scratch_bytes(65535, 16384, 200000) == 65536 + 16 * 98 * (65535 + 16384)


def test_every_operator_refuses_a_bad_batch():
    for bad in BAD_BATCHES:
        b = batch(**bad)
        refused(step(b=b))
        refused(append(b=b))
        refused(attend(b=b))
    L, t, c = ob.lib(), ctypes.byref(tables()), ctypes.byref(cache())
    refused(L.odi_cuda_paged_step(t, None, None, A, None, None))
    refused(L.odi_cuda_paged_step(None, ctypes.byref(batch()), None, A, None, None))
    refused(L.odi_cuda_qk_rope_append_paged(A, 1280, None, None, 1e-6, C, 768, c, None, 4, 6, 1e4, None))


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_a_bad_cache_is_refused(bad, code):
    refused(append(c=cache(**bad)), code)
    refused(attend(c=cache(**bad)), code)


def test_step_refusals():
    for bad in (dict(table=None), dict(lens=None), dict(free=None), dict(count=None), dict(table=A + 2), dict(lens=A + 1),
                dict(free=A + 3), dict(count=A + 2), dict(requests=2), dict(max_pages=0), dict(page_size=32), dict(page_size=20),
                dict(num_pages=0), dict(num_pages=1 << 28), dict(max_pages=1 << 29)):
        refused(step(t=tables(**bad)))
    # more tiles than a work list can count
    refused(step(t=tables(requests=2048, max_pages=1 << 18, page_size=16), b=batch(requests=2048, max_rows=262144, max_new=262144, heads=64, kv_heads=1)),
            word="tiles")
    refused(step(new=None))
    for k in ("keep", "new", "prefix"):
        refused(step(**{k: A + 2}))


def test_append_refusals():
    for kw in (dict(qkv=None), dict(out=None), dict(T=-1), dict(T=41), dict(H=0), dict(H=65536), dict(ld=1279), dict(ldq=767), dict(ldq=769),
               dict(theta=0.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(qkv=A + 2), dict(out=C + 2), dict(qn=A + 1),
               dict(kn=A + 2), dict(out=A), dict(out=A + 4 * 1280 * 4 - 4), dict(c=cache(page_size=32)), dict(ld=1 << 41)):
        refused(append(**kw))
    assert append(T=0) == 0


def test_attention_refusals():
    for kw in (dict(q=None), dict(out=None), dict(scr=None), dict(T=-1), dict(T=41), dict(ld=767), dict(ld=769), dict(ldo=767), dict(ldo=769),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0),
               dict(cap=float("nan")), dict(cap=float("inf")), dict(q=A + 2), dict(out=C + 2), dict(slopes=A + 1), dict(scr=A + 8),
               dict(n=NEED - 1), dict(out=A), dict(out=A + 2 * 768 * 4 - 4), dict(out=A - 4, kind=1), dict(c=cache(kv_heads=3)),
               dict(c=cache(page_size=32)), dict(t=tables(page_size=32)), dict(t=tables(requests=4)), dict(t=tables(table=None)),
               dict(t=tables(num_pages=11)), dict(t=tables(table=A + 2)), dict(ld=1 << 41)):
        refused(attend(**kw))
    refused(attend(kind=2), DTYPE)
    assert attend(T=0) == 0


def test_caps_out_of_range_are_refused():
    # scale / softcap past fp32, scale * log2(e) past fp32, a cap whose rounding the scores would show
    for kw in (dict(cap=1e-39), dict(cap=1e-30, scale=1e10), dict(scale=3e38), dict(cap=1024.5)):
        refused(attend(**kw))
    assert attend(T=0, cap=1024.0) == 0


def test_verify_refusals():
    n = ob.lib().odi_cuda_verify_scratch_bytes(5, 2, 100)

    def call(x=A, ld=100, tok=A, st=A, R=5, Bq=2, V=100, temp=1.0, p=None, ldp=0, ua=A, un=A, acc=A, nxt=A, scr=A, n=n):
        return ob.lib().odi_cuda_verify_sampled(x, ld, tok, st, R, Bq, V, temp, p, ldp, ua, un, acc, nxt, scr, n, None)

    for k in ("x", "tok", "st", "ua", "un", "acc", "nxt"):
        refused(call(**{k: None}))
        refused(call(**{k: A + 2}))
    for kw in (dict(scr=None), dict(scr=A + 4), dict(n=n - 1), dict(R=0), dict(R=65536), dict(Bq=0), dict(Bq=16385), dict(V=0),
               dict(V=0x7fff0001, ld=1 << 32), dict(ld=99), dict(p=A, ldp=99), dict(p=A + 1, ldp=100), dict(temp=0.0), dict(temp=-1.0),
               dict(temp=float("nan")), dict(temp=float("inf")), dict(temp=1e-7)):
        refused(call(**kw))


def test_tensors_that_do_not_fit_are_refused():
    z, i32 = torch.zeros, torch.int32
    with pytest.raises(TypeError):
        paged.PagedCache(z(2, 1, 16, 64), z(2, 1, 16, 64))
    with pytest.raises(ValueError):  # not on a CUDA device
        paged.PagedCache(z(2, 1, 16, 64, dtype=torch.float16), z(2, 1, 16, 64, dtype=torch.float16))
    with pytest.raises(ValueError):
        paged.PagedCache(z(2, 16, 64, dtype=torch.float16), z(2, 16, 64, dtype=torch.float16))
    with pytest.raises(ValueError):
        paged.PageTables(z(2, 3, dtype=i32), z(2, dtype=i32), z(5, dtype=i32), z(1, dtype=i32), 16)
    with pytest.raises(ValueError):
        paged.PageTables(z(2, 3, dtype=i32), z(2, dtype=i32), z(5, dtype=i32), z(1, dtype=i32), 20)
    with pytest.raises(ValueError):
        paged.verify_scratch(0, 1, 10)
    with pytest.raises(ValueError):
        paged.verify_sampled(z(2, 5), z(2, dtype=i32), z(2, dtype=i32), z(2), z(1), scratch=z(8, dtype=torch.uint8))
