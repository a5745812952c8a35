"""The drafted-token operators refuse what they cannot do, on the host and
before any launch: sizes, types, strides, alignment.  No GPU needed (the
pointers below are never followed)."""
import ctypes

import pytest
import torch

import odiengine_b200 as ob
from odiengine_b200 import draft

INVALID, DTYPE = 2, 202
A, B = 0x10000, 0x20000  # aligned addresses of nothing


def cache(k=A, v=B, dtype=0, kv_heads=2, head_dim=128, ctx=64):
    return draft._KvCacheStruct(k, v, dtype, kv_heads, head_dim, ctx)


def refused(rc, code=INVALID, word=None):
    assert rc == code
    msg = ob.lib().odi_cuda_last_error().decode()
    assert msg and (word is None or word in msg), msg


@pytest.mark.parametrize("dtype,kv,hd,ctx,want", [
    (0, 2, 128, 64, 2 * 64 * 128 * 2), (1, 2, 128, 64, 2 * 64 * 128 + 2 * 64 * 4),
    (1, 1, 64, 3, 256 + 3 * 4), (1, 3, 64, 5, 1024 + 15 * 4),
    (2, 2, 128, 64, 0), (0, 0, 128, 64, 0), (0, 2, 96, 64, 0), (1, 2, 64, 0, 0), (-1, 2, 64, 8, 0),
    (1, 8, 128, 1 << 22, (8 << 22) * 132)])  # past 32 bits
def test_cache_bytes(dtype, kv, hd, ctx, want):
    assert ob.lib().odi_cuda_kv_cache_bytes(dtype, kv, hd, ctx) == want


@pytest.mark.parametrize("bad,code", [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(k=A + 8), INVALID), (dict(dtype=2), DTYPE),
    (dict(head_dim=96), INVALID), (dict(head_dim=256), INVALID), (dict(kv_heads=0), INVALID),
    (dict(kv_heads=70000), INVALID), (dict(ctx=0), INVALID)])
def test_every_operator_refuses_a_bad_cache(bad, code):
    L, c = ob.lib(), ctypes.byref(cache(**bad))
    refused(L.odi_cuda_qk_rope_append(A, 768, None, None, 1e-6, B, 256, c, A, None, 1, 2, 1e4, None), code)
    refused(L.odi_cuda_kv_read(c, 0, 1, A, B, 0, None), code)
    refused(L.odi_cuda_kv_move(c, A, B, 1, None, None), code)
    refused(L.odi_cuda_attention_tree(A, 256, c, B, None, A, 1, 2, 1.0, A, 1 << 20, None), code)
    assert L.odi_cuda_kv_read(None, 0, 1, A, B, 0, None) == INVALID


def test_append_refusals():
    L, c = ob.lib(), ctypes.byref(cache())

    def call(qkv=A, ld=768, out=B, ldq=256, st=A, T=1, H=2, theta=1e4, qn=None, kn=None, depth=None):
        return L.odi_cuda_qk_rope_append(qkv, ld, qn, kn, 1e-6, out, ldq, c, st, depth, T, H, theta, None)

    for kw in (dict(qkv=None), dict(out=None), dict(st=None), dict(T=0), dict(T=-1), dict(H=0), dict(ld=767),
               dict(ldq=255), dict(theta=0.0), dict(theta=float("nan")), dict(T=1 << 30), dict(qkv=A + 2), dict(out=B + 1),
               dict(st=A + 2), dict(qn=A + 1), dict(kn=A + 2), dict(depth=A + 3),
               # q rows over qkv's: another stride, another column, a row further, the last row's end
               dict(out=A, T=2), dict(out=A + 4, ldq=768, T=2), dict(out=A + 768 * 4, ldq=768, T=2),
               dict(out=A + (768 + 767) * 4, ldq=768, T=2)):
        refused(call(**kw))



def test_read_and_move_refusals():
    L, c = ob.lib(), ctypes.byref(cache())
    for a in ((-1, 1, A, B, 0), (0, -1, A, B, 0), (60, 5, A, B, 0), (64, 1, A, B, 0), (2147483647, 2147483647, A, B, 0),
              (0, 1, None, None, 0), (0, 1, A + 4, B, 0)):
        refused(L.odi_cuda_kv_read(c, *a, None))
    refused(L.odi_cuda_kv_read(c, 0, 1, A, B, 2, None), DTYPE)
    assert L.odi_cuda_kv_read(c, 64, 0, None, None, 0, None) == 0  # nothing to read
    for a in ((A, B, -1), (A, B, draft.KV_MOVE_MAX + 1), (None, B, 1), (A, None, 1), (A + 2, B, 1), (A, B + 1, 1)):
        refused(L.odi_cuda_kv_move(c, *a, None, None))
    refused(L.odi_cuda_kv_move(c, A, B, 1, A + 2, None))
    assert L.odi_cuda_kv_move(c, None, None, 0, None, None) == 0


def test_attention_refusals():
    L, c = ob.lib(), ctypes.byref(cache())
    need = L.odi_cuda_attention_tree_scratch_bytes(4, 6, 2, 128, 64)
    assert need > 0

    def call(q=A, ld=768, out=B, st=A, T=4, H=6, scale=1.0, scr=A, n=need, mask=None):
        return L.odi_cuda_attention_tree(q, ld, c, out, mask, st, T, H, scale, scr, n, None)

    for kw in (dict(q=None), dict(out=None), dict(st=None), dict(scr=None), dict(T=0), dict(T=draft.TREE_MAX + 1),
               dict(H=5), dict(H=0), dict(H=2048, ld=1 << 20), dict(ld=767), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(n=need - 1), dict(scr=A + 4), dict(q=A + 2), dict(mask=A + 1), dict(st=A + 2)):
        refused(call(**kw))
    for off, ld, T, clash in ((768, 768, 1, False), (767, 768, 1, True), (-768, 768, 1, False), (768, 768, 2, True),
                              (1536, 768, 2, False), (768, 1536, 1, False), (768, 2304, 2, False), (768, 2303, 2, True)):
        refused(call(out=A + 4 * off, ld=ld, T=T, n=0), word="overlap" if clash else "scratch")
    for a in ((0, 6, 2, 128, 64), (257, 6, 2, 128, 64), (4, 5, 2, 128, 64), (4, 6, 2, 80, 64), (4, 6, 2, 128, 0)):
        assert L.odi_cuda_attention_tree_scratch_bytes(*a) == 0


def test_logits_refusals():
    L = ob.lib()

    def call(x=A, ld=100, out=B, ldo=100, tok=A, rows=2, V=100, scr=A, n=32, **o):
        f = dict(repeat_penalty=1.0, frequency_penalty=0.0, presence_penalty=0.0, history=0, history_ld=0, history_len=0,
                 history_max=0, bias_ids=0, bias=0, bias_count=0, mask=0, mask_ld=0)
        assert set(o) <= set(f)
        opts = draft._LOGITS_OPTS.pack(*{**f, **o}.values())
        return L.odi_cuda_logits_adjust(x, ld, out, ldo, tok, rows, V, opts, scr, n, None)

    for kw in (dict(x=None), dict(out=None, tok=None), dict(rows=-1), dict(rows=70000), dict(V=0), dict(V=0x7fff0001, ld=1 << 31, ldo=1 << 31), dict(ld=99),
               dict(ldo=99), dict(x=A, out=A, ldo=101), dict(x=A + 2), dict(scr=None), dict(scr=A + 4), dict(n=31),
               dict(repeat_penalty=0.0), dict(repeat_penalty=float("nan")), dict(frequency_penalty=float("inf")),
               dict(presence_penalty=float("nan")), dict(history=A, history_ld=3, history_max=4),
               dict(history=A, history_max=65536), dict(bias_count=-1), dict(bias_count=65536), dict(bias_count=1),
               dict(bias_count=1, bias_ids=A), dict(mask=A, mask_ld=3), dict(history=A + 1, history_max=1), dict(mask=A + 2, mask_ld=4),
               dict(history_len=A + 2), dict(bias_count=1, bias_ids=A + 2, bias=A), dict(bias_count=1, bias_ids=A, bias=A + 3)):
        refused(call(**kw))
    # rows of 100: an output over the logits is refused, one beside them or in the
    # gaps of their stride is not (the missing scratch is, after it)
    for off, ldo, ld, rows, clash in ((0, 101, 100, 2, True), (1, 100, 100, 1, True), (99, 100, 100, 1, True),
                                      (100, 100, 100, 1, False), (100, 100, 100, 2, True), (200, 100, 100, 2, False),
                                      (100, 200, 200, 5, False), (101, 200, 200, 5, True), (99, 200, 200, 5, True),
                                      (-100, 200, 200, 5, False), (-99, 200, 200, 5, True), (150, 250, 250, 9, False),
                                      (100, 400, 200, 3, False), (100, 350, 200, 3, True), (0, 100, 100, 2, False)):
        refused(call(ld=ld, out=A + 4 * off, ldo=ldo, rows=rows, scr=None), word="overlap" if clash else "scratch")
    assert L.odi_cuda_logits_scratch_bytes(0) == 0 and L.odi_cuda_logits_scratch_bytes(3) == 48


def test_tensors_that_do_not_fit_are_refused():
    z = torch.zeros
    with pytest.raises(ValueError):
        draft.kv_cache_bytes("q4", 2, 128, 64)
    with pytest.raises(ValueError):
        draft.KVCache(z(1), z(1), "q4", 2, 128, 64)
    with pytest.raises(ValueError):  # not on a CUDA device
        draft.KVCache(z(2, 64, 128, dtype=torch.float16), z(2, 64, 128, dtype=torch.float16), "f16", 2, 128, 64)
    with pytest.raises(TypeError):
        draft.KVCache(z(2, 64, 128), z(2, 64, 128), "f16", 2, 128, 64)
    with pytest.raises(ValueError):
        draft.logits_adjust(z(2, 5), z(2, 5))
    with pytest.raises(ValueError):
        draft._state_ptr(z(4, dtype=torch.int32), 0)
