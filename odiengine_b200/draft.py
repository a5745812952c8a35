"""Verifying drafted tokens: the operators of a step that checks T drafted
tokens (a chain or a tree) of one sequence in one pass, on device tensors.

    qk_rope_append   per-head q/k norm + rotation, k and v rows into the cache
    attention_tree   every node over the cache and its ancestors
    logits_adjust    penalties, biases, grammar mask, greedy token of each node
    kv_move          the accepted path's cache rows into place
    kv_read          cache rows out as fp16 / fp32

over a :class:`KVCache` of fp16 rows (the layout of the decode step) or of
int8 rows with one scale each (half the bytes).  Calls are asynchronous on
`stream` (default: the tensors' device's current stream); errors are
:class:`odiengine_b200.OdiCudaError`, or ValueError / TypeError for tensors
that do not fit.  The position is device resident (`state`, the decode
step's odi_cuda_decode_state as int32[4]), so calls can be captured in a CUDA
graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import check, lib

KV_F16, KV_I8 = 0, 1                      # ODI_CUDA_KV_*
KV_DTYPES = {"f16": KV_F16, "i8": KV_I8}
TREE_MAX = 256                            # ODI_CUDA_TREE_MAX
KV_MOVE_MAX = 256                         # ODI_CUDA_KV_MOVE_MAX


class _KvCacheStruct(ctypes.Structure):
    """odi_cuda_kv_cache (include/odi_cuda.h)."""

    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("dtype", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("ctx", ctypes.c_int)]


class _LogitsOpts(ctypes.Structure):
    """odi_cuda_logits_opts (include/odi_cuda.h)."""

    _fields_ = [("repeat_penalty", ctypes.c_float), ("frequency_penalty", ctypes.c_float),
                ("presence_penalty", ctypes.c_float), ("history", ctypes.c_void_p), ("history_ld", ctypes.c_int64),
                ("history_len", ctypes.c_void_p), ("history_max", ctypes.c_int), ("bias_ids", ctypes.c_void_p),
                ("bias", ctypes.c_void_p), ("bias_count", ctypes.c_int), ("mask", ctypes.c_void_p),
                ("mask_ld", ctypes.c_int64)]


def _need(t, dtype, what: str, dev=None):
    if t.dtype != dtype:
        raise TypeError(f"{what}: {dtype} wanted, got {t.dtype}")
    if not t.is_cuda or (dev is not None and t.device != dev):
        raise ValueError(f"{what}: must be on {dev or 'a CUDA device'}, is on {t.device}")


def _flat(t, dtype, what: str, dev, numel: int = None):
    _need(t, dtype, what, dev)
    if not t.is_contiguous() or (numel is not None and t.numel() != numel):
        raise ValueError(f"{what}: must be contiguous with {numel} values, got {tuple(t.shape)}")


def _rows2(t, dtype, what: str, dev, width: int) -> int:
    """A 2-D tensor of rows of unit stride: its row stride in values."""
    _need(t, dtype, what, dev)
    if t.dim() != 2 or t.shape[1] != width or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{what}: rows of {width} adjacent values wanted, got {tuple(t.shape)} strides {t.stride()}")
    return t.stride(0) if t.shape[0] > 1 else max(width, t.stride(0))


def _call(dev, stream, fn, *args) -> None:
    """One library call on `dev`, which need not be the current device."""
    if torch.cuda.current_device() == dev.index:
        check(fn(*args, (stream or torch.cuda.current_stream(dev)).cuda_stream))
    else:
        with torch.cuda.device(dev):
            check(fn(*args, (stream or torch.cuda.current_stream(dev)).cuda_stream))


class KVCache:
    """One layer's K and V.  `k`, `v`: fp16 [kv_heads, ctx, head_dim] ("f16",
    what DecodeModel keeps per layer), or uint8 of :func:`kv_cache_bytes`
    bytes ("i8": int8 codes, then one fp32 scale per row)."""

    def __init__(self, k, v, dtype: str, kv_heads: int, head_dim: int, ctx: int):
        if dtype not in KV_DTYPES:
            raise ValueError(f"cache dtype {dtype!r}: one of {sorted(KV_DTYPES)}")
        need = kv_cache_bytes(dtype, kv_heads, head_dim, ctx)
        for t, n in ((k, "k"), (v, "v")):
            _need(t, torch.float16 if dtype == "f16" else torch.uint8, f"cache {n}", k.device)
            if not t.is_contiguous() or t.numel() * t.element_size() < need:
                raise ValueError(f"cache {n}: {need} contiguous bytes wanted")
            if t.data_ptr() % 16:
                raise ValueError(f"cache {n}: must be 16-byte aligned")
        self.k, self.v, self.dtype = k, v, dtype
        self.kv_heads, self.head_dim, self.ctx = kv_heads, head_dim, ctx
        self.device = k.device
        self._struct = _KvCacheStruct(k.data_ptr(), v.data_ptr(), KV_DTYPES[dtype], kv_heads, head_dim, ctx)
        self._ref = ctypes.addressof(self._struct)

    @classmethod
    def new(cls, dtype: str, kv_heads: int, head_dim: int, ctx: int, device="cuda") -> "KVCache":
        """An empty (zero) cache."""
        n = kv_cache_bytes(dtype, kv_heads, head_dim, ctx)
        if dtype == "f16":
            k, v = (torch.zeros((kv_heads, ctx, head_dim), dtype=torch.float16, device=device) for _ in range(2))
        else:
            k, v = (torch.zeros(n, dtype=torch.uint8, device=device) for _ in range(2))
        return cls(k, v, dtype, kv_heads, head_dim, ctx)

    @property
    def nbytes(self) -> int:
        return 2 * kv_cache_bytes(self.dtype, self.kv_heads, self.head_dim, self.ctx)


def kv_cache_bytes(dtype: str, kv_heads: int, head_dim: int, ctx: int) -> int:
    """Bytes of K (and again of V)."""
    n = lib().odi_cuda_kv_cache_bytes(KV_DTYPES.get(dtype, -1), kv_heads, head_dim, ctx)
    if not n:
        raise ValueError(f"no cache of dtype {dtype!r}, kv_heads {kv_heads}, head_dim {head_dim}, ctx {ctx}")
    return n


def _state_ptr(state, dev) -> int:
    if state.dtype != torch.int32 or state.numel() != 4 or state.device != dev or not state.is_contiguous():
        raise ValueError(f"state: int32[4] (odi_cuda_decode_state) on {dev} wanted")
    return state.data_ptr()


def qk_rope_append(qkv, cache: KVCache, state, q_out=None, *, heads: int, theta: float, q_norm=None, k_norm=None,
                   eps: float = 1e-6, depth=None, stream=None):
    """Rows of qkv [T, (heads + 2 kv_heads) * head_dim] fp32: q and k normed
    per head (q_norm / k_norm: head_dim weights, or None), rotated at position
    state.pos + depth[t] (depth int32 [T]; None: t), k and v stored at slot
    state.pos + t.  Returns the rotated q in q_out [T, heads * head_dim]."""
    dev, hd = cache.device, cache.head_dim
    ld = _rows2(qkv, torch.float32, "qkv", dev, (heads + 2 * cache.kv_heads) * hd)
    T = qkv.shape[0]
    if q_out is None:
        q_out = torch.empty((T, heads * hd), dtype=torch.float32, device=dev)
    ld_q = _rows2(q_out, torch.float32, "q_out", dev, heads * hd)
    if q_out.shape[0] != T:
        raise ValueError("q_out: one row per row of qkv wanted")
    for t, n in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _flat(t, torch.float32, n, dev, hd)
    if depth is not None:
        _flat(depth, torch.int32, "depth", dev, T)
    _call(dev, stream, lib().odi_cuda_qk_rope_append, qkv.data_ptr(), ld, q_norm.data_ptr() if q_norm is not None else None,
          k_norm.data_ptr() if k_norm is not None else None, eps, q_out.data_ptr(), ld_q, cache._ref,
          _state_ptr(state, dev), depth.data_ptr() if depth is not None else None, T, heads, theta)
    return q_out


def kv_read(cache: KVCache, start: int, count: int, k_out=None, v_out=None, stream=None):
    """Positions start .. start + count - 1 as [kv_heads, count, head_dim],
    fp16 or fp32 by the outputs' type (default: new fp16 tensors)."""
    dev = cache.device
    if k_out is None and v_out is None:
        k_out, v_out = (torch.empty((cache.kv_heads, count, cache.head_dim), dtype=torch.float16, device=dev)
                        for _ in range(2))
    ref = k_out if k_out is not None else v_out
    if ref.dtype not in (torch.float16, torch.float32):
        raise TypeError(f"kv_read: outputs are fp16 or fp32, not {ref.dtype}")
    for t in (k_out, v_out):
        if t is not None:
            _flat(t, ref.dtype, "kv_read output", dev, cache.kv_heads * count * cache.head_dim)
    _call(dev, stream, lib().odi_cuda_kv_read, cache._ref, start, count, k_out.data_ptr() if k_out is not None else None,
          v_out.data_ptr() if v_out is not None else None, 0 if ref.dtype == torch.float16 else 1)
    return k_out, v_out


def kv_move(cache: KVCache, src, dst, state=None, stream=None) -> None:
    """Cache rows src[i] -> dst[i] (int32, at most KV_MOVE_MAX) as if all were
    read before any is written; relative to state.pos, or absolute."""
    dev, n = cache.device, src.numel()
    _flat(src, torch.int32, "src", dev, n)
    _flat(dst, torch.int32, "dst", dev, n)
    _call(dev, stream, lib().odi_cuda_kv_move, cache._ref, src.data_ptr(), dst.data_ptr(), n,
          _state_ptr(state, dev) if state is not None else None)


def attention_tree_scratch(cache: KVCache, tokens: int, heads: int):
    """Zeroed scratch for attention_tree calls of this shape on one stream
    (any layer; a smaller `tokens` fits too if its own size does)."""
    n = lib().odi_cuda_attention_tree_scratch_bytes(tokens, heads, cache.kv_heads, cache.head_dim, cache.ctx)
    if not n:
        raise ValueError(f"attention_tree: no such shape (tokens {tokens}, heads {heads}, kv_heads {cache.kv_heads})")
    return torch.zeros(n, dtype=torch.uint8, device=cache.device)


def attention_tree(q, cache: KVCache, out=None, state=None, *, heads: int, scale: float, scratch, mask=None,
                   stream=None):
    """Node t's rotated queries q[t] (fp32 [T, heads * head_dim]) over the
    slots below state.pos and the tree slots of its mask row (int32 / uint32
    [T, ceil(T / 32)], bit j: node t sees node j; None: j <= t)."""
    dev, hd = cache.device, cache.head_dim
    ld = _rows2(q, torch.float32, "q", dev, heads * hd)
    T = q.shape[0]
    if out is None:
        out = torch.empty((T, heads * hd), dtype=torch.float32, device=dev)
    _flat(out, torch.float32, "out", dev, T * heads * hd)
    if mask is not None and (mask.dtype not in (torch.int32, torch.uint32) or mask.device != dev or not mask.is_contiguous()
                             or mask.shape != (T, (T + 31) // 32)):
        raise ValueError(f"mask: int32 words {(T, (T + 31) // 32)} on {dev} wanted")
    _need(scratch, torch.uint8, "scratch", dev)
    _call(dev, stream, lib().odi_cuda_attention_tree, q.data_ptr(), ld, cache._ref, out.data_ptr(),
          mask.data_ptr() if mask is not None else None, _state_ptr(state, dev), T, heads, scale, scratch.data_ptr(),
          scratch.numel())
    return out


def logits_scratch(rows: int, device="cuda"):
    """Zeroed scratch for logits_adjust calls of up to `rows` rows on one stream."""
    return torch.zeros(max(16, lib().odi_cuda_logits_scratch_bytes(rows)), dtype=torch.uint8, device=device)


def logits_adjust(logits, out=None, tokens=None, *, scratch=None, history=None, history_lens=None,
                  repeat_penalty: float = 1.0, frequency_penalty: float = 0.0, presence_penalty: float = 0.0,
                  bias_ids=None, bias=None, mask=None, stream=None):
    """Rows of logits [rows, V] adjusted into `out` (may be `logits`; None:
    not stored) and their greedy tokens (int32 [rows]; None: not wanted).
    history int32 [rows, H] or [1, H] with history_lens int32 [rows];
    bias_ids / bias [n] for all rows; mask int32 words [rows or 1, ceil(V / 32)]."""
    dev = logits.device
    rows, V = logits.shape
    ld = _rows2(logits, torch.float32, "logits", dev, V)
    ld_out = 0
    if out is not None:
        ld_out = _rows2(out, torch.float32, "out", dev, V)
        if out.shape[0] != rows:
            raise ValueError("out: one row per row of logits wanted")
    if tokens is not None:
        _flat(tokens, torch.int32, "tokens", dev, rows)
        if scratch is None:
            raise ValueError("logits_adjust: tokens need a scratch (logits_scratch)")
        _need(scratch, torch.uint8, "scratch", dev)
    o = _LogitsOpts(repeat_penalty, frequency_penalty, presence_penalty)
    if history is not None:
        o.history_ld = _rows2(history, torch.int32, "history", dev, history.shape[-1])
        if history.shape[0] not in (1, rows):
            raise ValueError("history: one row, or one per row of logits")
        if history.shape[0] == 1:
            o.history_ld = 0
        o.history, o.history_max = history.data_ptr(), history.shape[1]
        if history_lens is not None:
            _flat(history_lens, torch.int32, "history_lens", dev, rows)
            o.history_len = history_lens.data_ptr()
    if bias_ids is not None and bias_ids.numel():
        n = bias_ids.numel()
        _flat(bias_ids, torch.int32, "bias_ids", dev, n)
        _flat(bias, torch.float32, "bias", dev, n)
        o.bias_ids, o.bias, o.bias_count = bias_ids.data_ptr(), bias.data_ptr(), n
    if mask is not None:
        if mask.dtype not in (torch.int32, torch.uint32):
            raise TypeError("mask: int32 words wanted")
        o.mask_ld = _rows2(mask, mask.dtype, "mask", dev, (V + 31) // 32)
        if mask.shape[0] not in (1, rows):
            raise ValueError("mask: one row, or one per row of logits")
        if mask.shape[0] == 1:
            o.mask_ld = 0
        o.mask = mask.data_ptr()
    _call(dev, stream, lib().odi_cuda_logits_adjust, logits.data_ptr(), ld, out.data_ptr() if out is not None else None,
          ld_out, tokens.data_ptr() if tokens is not None else None, rows, V, ctypes.addressof(o),
          scratch.data_ptr() if scratch is not None else None, scratch.numel() if scratch is not None else 0)
    return out, tokens
