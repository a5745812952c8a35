"""What the drafted-token calls hand to the library, and what DraftVerifier
keeps between calls.  No GPU: tensors that say they are on cuda:0, and library
calls that are recorded, not made."""
import pytest
import torch

from odiengine_b200 import draft


class OnGpu:
    """A CPU tensor that passes for one of cuda:0 (its memory is never followed)."""

    is_cuda = True

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return 0


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(draft, "_call", lambda dev, stream, fn, *args: made.append((fn.__name__, args)))
    return made


def z(*shape, dtype=torch.float32):
    return OnGpu(torch.zeros(shape, dtype=dtype))


def logits_opts(calls, **kw):
    """The options that logits_adjust packs for 4 rows of 64."""
    draft.logits_adjust(z(4, 64), z(4, 64), **kw)
    name, args = calls[-1]
    assert name == "odi_cuda_logits_adjust"
    keys = ("repeat", "frequency", "presence", "history", "history_ld", "history_len", "history_max", "bias_ids", "bias",
            "bias_count", "mask", "mask_ld")
    return dict(zip(keys, draft._LOGITS_OPTS.unpack(args[7])))


@pytest.mark.parametrize("what,width", [("history", 5), ("mask", 2)])
def test_rows_that_overlap_are_not_one_row(calls, what, width):
    """A stride of 0 means one row for all rows of logits; a sliding window's
    rows (stride 1) are rows of their own, and refused."""
    i32 = torch.int32
    full = torch.zeros((4, width), dtype=i32)
    assert logits_opts(calls, **{what: OnGpu(full)})[what + "_ld"] == width
    assert logits_opts(calls, **{what: OnGpu(torch.zeros((4, width + 3), dtype=i32)[:, :width])})[what + "_ld"] == width + 3
    for one in (full[:1], full[:1].expand(4, width)):
        assert logits_opts(calls, **{what: OnGpu(one)})[what + "_ld"] == 0
    n = len(calls)
    for view in (torch.zeros(width + 3, dtype=i32).unfold(0, width, 1), torch.zeros(4 * width, dtype=i32).as_strided((4, width), (width - 1, 1))):
        assert view.shape == (4, width)
        with pytest.raises(ValueError, match="overlap"):
            logits_opts(calls, **{what: OnGpu(view)})
    with pytest.raises(ValueError):
        logits_opts(calls, **{what: OnGpu(full[:3])})
    assert len(calls) == n


# ---- caches ----------------------------------------------------------------------------------------------------

def aligned(n, dtype):
    """n values from a 16-byte boundary on."""
    t = torch.zeros(n + 16, dtype=dtype)
    return t[(-t.data_ptr() % 16) // t.element_size():][:n]


def test_cache_halves_that_do_not_fit_are_refused():
    """K and V in one memory, and an fp16 tensor of another cache's shape (its
    heads would be read from other places than it has them)."""
    f16, n = torch.float16, 2 * 8 * 64
    buf = aligned(3 * n, f16)
    k, v = buf[:n].view(2, 8, 64), buf[n:2 * n].view(2, 8, 64)
    c = draft.KVCache(OnGpu(k), OnGpu(v), "f16", 2, 64, 8)
    assert (c._struct.k, c._struct.v) == (k.data_ptr(), v.data_ptr())
    draft.KVCache(OnGpu(buf[:n]), OnGpu(buf[n:]), "f16", 2, 64, 8)  # flat, and longer than it has to be
    for other in (k, buf[n - 8:2 * n - 8].view(2, 8, 64)):
        with pytest.raises(ValueError, match="share"):
            draft.KVCache(OnGpu(k), OnGpu(other), "f16", 2, 64, 8)
    with pytest.raises(ValueError, match="wanted"):
        draft.KVCache(OnGpu(buf[:n].view(2, 8, 64)), OnGpu(buf[n:2 * n].view(8, 2, 64)), "f16", 2, 64, 8)
    with pytest.raises(ValueError, match="wanted"):
        draft.KVCache(OnGpu(buf[:n].view(2, 8, 64)), OnGpu(v), "f16", 2, 64, 4)
    need = draft.kv_cache_bytes("i8", 2, 64, 8)
    u8 = aligned(2 * need, torch.uint8)
    draft.KVCache(OnGpu(u8[:need]), OnGpu(u8[need:]), "i8", 2, 64, 8)
    with pytest.raises(ValueError, match="share"):
        draft.KVCache(OnGpu(u8[:need]), OnGpu(u8[16:need + 16]), "i8", 2, 64, 8)


def test_read_refuses_outputs_over_each_other_or_the_cache():
    """Addresses of nothing: no call below reaches a launch."""
    import ctypes

    import odiengine_b200 as ob

    L, K, V = ob.lib(), 0x100000, 0x200000
    c = ctypes.byref(draft._KvCacheStruct(K, V, draft.KV_F16, 2, 64, 100))  # 25,600 bytes each
    size, out = 2 * 10 * 64 * 2, 0x300000                                   # 10 positions as fp16
    for k, v, dt in ((out, out, 0), (out, out + size - 16, 0), (out + size, out + 16, 0), (out, out + size, 1),
                     (K, None, 0), (None, K + 25600 - 16, 0), (V - size + 16, out, 0), (out, V, 0)):
        assert L.odi_cuda_kv_read(c, 0, 10, k, v, dt, None) == 2
        assert "overlap" in L.odi_cuda_last_error().decode()
    rows = draft._KvCacheStruct(K, V, draft.KV_I8, 2, 64, 100)              # the scales are the cache's too
    assert L.odi_cuda_kv_read(ctypes.byref(rows), 0, 10, K + 12800, out, 0, None) == 2


# ---- sequences -------------------------------------------------------------------------------------------------

@pytest.fixture
def verifier(monkeypatch):
    """A DraftVerifier without a device: its forward pass does nothing."""
    import contextlib
    import types

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(draft.DraftVerifier, "_ordered", lambda self: contextlib.nullcontext(), raising=False)
    monkeypatch.setattr(draft.DraftVerifier, "_forward", lambda self, *a: None)
    monkeypatch.setattr(draft.DraftVerifier, "_check", lambda self: None)
    v = object.__new__(draft.DraftVerifier)
    v.cfg = types.SimpleNamespace(vocab=100, ctx=64)
    v.device, v.max_nodes, v.history = torch.device("cpu"), 4, 0
    v.pos, v.pending, v.tokens = 0, None, []
    return v


@pytest.mark.parametrize("where", ["_forward", "_check"])
def test_a_prompt_that_failed_leaves_no_sequence(verifier, monkeypatch, where):
    """start that raises midway leaves nothing that verify could go on from,
    the sequence before it neither."""
    verifier.start([1, 2, 3])
    assert verifier.pending == 3 and verifier.pos == 2

    def fail(self, *a):
        raise RuntimeError("a launch failed")

    with monkeypatch.context() as m:
        m.setattr(draft.DraftVerifier, where, fail)
        with pytest.raises(RuntimeError, match="a launch failed"):
            verifier.start([4, 5, 6, 7, 8, 9])
    with pytest.raises(RuntimeError, match="start a sequence"):
        verifier.verify()
    verifier.start([7, 8])
    assert verifier.pending == 8 and verifier.tokens == [7, 8]


def test_verify_takes_what_adjusts_the_logits_only(verifier):
    """Another stream, other outputs, or a history beside the verifier's own
    would be ordered or counted wrongly: refused before anything runs."""
    verifier.start([1, 2, 3])
    for bad in (dict(stream=None), dict(out=None), dict(tokens=None), dict(scratch=None), dict(penalty=1.1)):
        with pytest.raises(TypeError, match=next(iter(bad))):
            verifier.verify(**bad)
    verifier.history = 8
    for bad in (dict(history=z(1, 3, dtype=torch.int32)), dict(history_lens=z(1, dtype=torch.int32))):
        with pytest.raises(TypeError, match="history"):
            verifier.verify(**bad)
    assert verifier.pending == 3 and verifier.pos == 2


# ---- arguments left out ----------------------------------------------------------------------------------------

def test_what_is_missing_is_named(calls):
    """A list without its partner, or a state or scratch left out, is a
    TypeError or ValueError that names it, and no call."""
    import types

    c = types.SimpleNamespace(index=0, kv_heads=2, head_dim=64, ctx=8, device="cpu", _ref=0)
    q, out = z(1, 256), z(1, 256)
    st, scr, i32 = z(4, dtype=torch.int32), z(1024, dtype=torch.uint8), torch.int32
    with pytest.raises(TypeError, match="state"):
        draft.attention_tree(q, c, out, heads=4, scale=0.1, scratch=scr)
    with pytest.raises(TypeError, match="scratch"):
        draft.attention_tree(q, c, out, st, heads=4, scale=0.1, scratch=None)
    with pytest.raises(TypeError, match="state"):
        draft.qk_rope_append(z(1, 512), c, None, q, heads=4, theta=1e4)
    x = z(4, 64)
    with pytest.raises(TypeError, match="bias"):
        draft.logits_adjust(x, x, bias_ids=z(3, dtype=i32))
    with pytest.raises(ValueError, match="bias_ids"):
        draft.logits_adjust(x, x, bias=z(3))
    with pytest.raises(ValueError, match="history"):
        draft.logits_adjust(x, x, history_lens=z(4, dtype=i32))
    assert not calls
    draft.attention_tree(q, c, out, st, heads=4, scale=0.1, scratch=scr)
    draft.logits_adjust(x, x, bias_ids=z(3, dtype=i32), bias=z(3))
    assert len(calls) == 2
