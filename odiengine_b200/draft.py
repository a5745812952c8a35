"""Verifying drafted tokens: the operators of a step that checks T drafted
tokens (a chain or a tree) of one sequence in one pass, on device tensors.

    qk_rope_append   per-head q/k norm + rotation, k and v rows into the cache
    attention_tree   every node over the cache and its ancestors
    logits_adjust    penalties, biases, grammar mask, greedy token of each node
    kv_move          the accepted path's cache rows into place
    kv_read          cache rows out as fp16 / fp32

over a :class:`KVCache` of fp16 rows (the layout of the decode step) or of
int8 rows with one scale each (half the bytes).  :class:`DraftVerifier` is the
step made of them and of the library's products, for the models of
odiengine_b200.decode.  Calls are asynchronous on
`stream` (default: the tensors' device's current stream), where outputs that
a call makes are allocated too; tensors of another stream that are handed in
are the caller's to order and to keep (Tensor.record_stream).  Errors are
:class:`odiengine_b200.OdiCudaError`, or ValueError / TypeError for tensors
that do not fit.  The position is device resident (`state`, the decode
step's odi_cuda_decode_state as int32[4]), so calls can be captured in a CUDA
graph.
"""
from __future__ import annotations

import contextlib
import ctypes
import struct

import torch

from . import FLAG_PDL, MatmulOpts, check, lib, new_workspace, workspace_bytes

KV_F16, KV_I8 = 0, 1                      # ODI_CUDA_KV_*
KV_DTYPES = {"f16": KV_F16, "i8": KV_I8}
TREE_MAX = 256                            # ODI_CUDA_TREE_MAX
KV_MOVE_MAX = 256                         # ODI_CUDA_KV_MOVE_MAX


class _KvCacheStruct(ctypes.Structure):
    """odi_cuda_kv_cache (include/odi_cuda.h)."""

    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("dtype", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("ctx", ctypes.c_int)]


# odi_cuda_logits_opts (include/odi_cuda.h) in native layout: packed bytes take
# 1 us less of the host than a ctypes structure (a call of one row: 10.1 -> 9.1 us).
_LOGITS_OPTS = struct.Struct("@fffPqPiPPiPq")  # a null pointer is 0


# The current stream's handle and the current device by index, without building
# torch's Stream object (2.2 us of a call that launches in 3).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _refuse(t, dtype, what: str, dev: int, shape) -> None:
    if t.dtype is not dtype:
        raise TypeError(f"{what}: {dtype} wanted, got {t.dtype}")
    if t.get_device() != dev or dev < 0:
        raise ValueError(f"{what}: must be on {'a CUDA device' if dev < 0 else f'cuda:{dev}'}, is on {t.device}")
    raise ValueError(f"{what}: {shape} wanted, got {tuple(t.shape)} strides {t.stride()}")


# Devices are compared by index, get_device() being the cheaper of the two and
# -1 for a tensor that is on no GPU.
def _flat(t, dtype, what: str, dev: int, numel: int) -> int:
    """The address of a contiguous tensor of numel values."""
    if t is None:
        raise TypeError(f"{what}: a tensor of {dtype} wanted, got None")
    if t.dtype is not dtype or t.get_device() != dev or dev < 0 or t.numel() != numel or not t.is_contiguous():
        _refuse(t, dtype, what, dev, f"{numel} contiguous values")
    return t.data_ptr()


def _rows2(t, dtype, what: str, dev: int, rows, width: int) -> int:
    """The stride in values of a 2-D tensor of `rows` rows (None: any) of
    `width` adjacent values."""
    if t.dtype is dtype and t.get_device() == dev >= 0 and t.dim() == 2:
        n, w = t.shape
        if w == width and (rows is None or n == rows):
            ld, one = t.stride()
            if one == 1 or w == 1:
                return ld if n > 1 and ld >= w else max(ld, w) if n <= 1 else 0
    _refuse(t, dtype, what, dev, f"{'rows' if rows is None else rows} of {width} adjacent values")


def _per_row(t, dtype, what: str, dev: int, rows: int, width: int) -> int:
    """The stride between the rows of a list for each of `rows` rows, or 0 for
    one list that all share: t has one row, or is one row expanded."""
    n = t.shape[0]
    if n != rows and n != 1:
        raise ValueError(f"{what}: one row, or one per row of logits")
    ld = _rows2(t, dtype, what, dev, n, width)
    # rows that overlap otherwise (a sliding window's view) are rows of their own
    if not ld and n > 1 and t.stride(0):
        raise ValueError(f"{what}: rows of {width} values that start {t.stride(0)} apart overlap; pass a contiguous copy")
    return ld if n == rows else 0


def _call(dev: int, stream, fn, *args) -> None:
    """One library call on device `dev`, which need not be the current one."""
    s = _raw_stream(dev) if stream is None else stream.cuda_stream
    if _current_device() == dev:
        rc = fn(*args, s)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, s)
    if rc:
        check(rc)


def _new(shape, dtype, cache, stream):
    """An output that a call makes: allocated on the stream that writes it, so
    that its memory is neither still in use elsewhere nor handed out again."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=cache.device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=cache.device)


class KVCache:
    """One layer's K and V.  `k`, `v`: fp16 [kv_heads, ctx, head_dim] ("f16",
    what DecodeModel keeps per layer), or uint8 of :func:`kv_cache_bytes`
    bytes ("i8": int8 codes, then one fp32 scale per row)."""

    def __init__(self, k, v, dtype: str, kv_heads: int, head_dim: int, ctx: int):
        if dtype not in KV_DTYPES:
            raise ValueError(f"cache dtype {dtype!r}: one of {sorted(KV_DTYPES)}")
        need = kv_cache_bytes(dtype, kv_heads, head_dim, ctx)
        want = torch.float16 if dtype == "f16" else torch.uint8
        for t, n in ((k, "k"), (v, "v")):
            if t.dtype is not want or t.device != k.device or not t.is_cuda or not t.is_contiguous() \
                    or t.numel() * t.element_size() < need:
                _refuse(t, want, f"cache {n}", k.get_device(), f"{need} contiguous bytes")
            if t.data_ptr() % 16:
                raise ValueError(f"cache {n}: must be 16-byte aligned")
            if dtype == "f16" and t.dim() == 3 and tuple(t.shape) != (kv_heads, ctx, head_dim):
                raise ValueError(f"cache {n}: [{kv_heads}, {ctx}, {head_dim}] wanted, got {tuple(t.shape)}")
        if abs(k.data_ptr() - v.data_ptr()) < need:
            raise ValueError("cache: k and v share memory")
        self.k, self.v, self.dtype = k, v, dtype
        self.kv_heads, self.head_dim, self.ctx = kv_heads, head_dim, ctx
        self.device, self.index = k.device, k.get_device()
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
    return _flat(state, torch.int32, "state (odi_cuda_decode_state)", dev, 4)


def qk_rope_append(qkv, cache: KVCache, state, q_out=None, *, heads: int, theta: float, q_norm=None, k_norm=None,
                   eps: float = 1e-6, depth=None, stream=None):
    """Rows of qkv [T, (heads + 2 kv_heads) * head_dim] fp32: q and k normed
    per head (q_norm / k_norm: head_dim weights, or None), rotated at position
    state.pos + depth[t] (depth int32 [T]; None: t), k and v stored at slot
    state.pos + t.  Returns the rotated q in q_out [T, heads * head_dim]."""
    dev, hd, f32 = cache.index, cache.head_dim, torch.float32
    ld = _rows2(qkv, f32, "qkv", dev, None, (heads + 2 * cache.kv_heads) * hd)
    T = qkv.shape[0]
    if q_out is None:
        q_out = _new((T, heads * hd), f32, cache, stream)
    ld_q = _rows2(q_out, f32, "q_out", dev, T, heads * hd)
    _call(dev, stream, lib().odi_cuda_qk_rope_append, qkv.data_ptr(), ld,
          None if q_norm is None else _flat(q_norm, f32, "q_norm", dev, hd),
          None if k_norm is None else _flat(k_norm, f32, "k_norm", dev, hd), eps, q_out.data_ptr(), ld_q, cache._ref,
          _state_ptr(state, dev), None if depth is None else _flat(depth, torch.int32, "depth", dev, T), T, heads, theta)
    return q_out


def kv_read(cache: KVCache, start: int, count: int, k_out=None, v_out=None, stream=None):
    """Positions start .. start + count - 1 as [kv_heads, count, head_dim],
    fp16 or fp32 by the outputs' type (default: new fp16 tensors)."""
    dev = cache.index
    if k_out is None and v_out is None:
        k_out, v_out = (_new((cache.kv_heads, max(count, 0), cache.head_dim), torch.float16, cache, stream) for _ in range(2))
    t = (v_out if k_out is None else k_out).dtype
    if t is not torch.float16 and t is not torch.float32:
        raise TypeError(f"kv_read: outputs are fp16 or fp32, not {t}")
    n = cache.kv_heads * max(count, 0) * cache.head_dim
    _call(dev, stream, lib().odi_cuda_kv_read, cache._ref, start, count,
          None if k_out is None else _flat(k_out, t, "k_out", dev, n),
          None if v_out is None else _flat(v_out, t, "v_out", dev, n), 0 if t is torch.float16 else 1)
    return k_out, v_out


def kv_move(cache: KVCache, src, dst, state=None, stream=None) -> None:
    """Cache rows src[i] -> dst[i] (int32, at most KV_MOVE_MAX) as if all were
    read before any is written; relative to state.pos, or absolute."""
    dev, n = cache.index, src.numel()
    _call(dev, stream, lib().odi_cuda_kv_move, cache._ref, _flat(src, torch.int32, "src", dev, n),
          _flat(dst, torch.int32, "dst", dev, n), n, None if state is None else _state_ptr(state, dev))


def attention_tree_scratch(cache: KVCache, tokens: int, heads: int):
    """Zeroed scratch for attention_tree calls on one stream: of any layer, any
    number of tokens and any heads of this head_dim."""
    n = lib().odi_cuda_attention_tree_scratch_bytes(tokens, heads, cache.kv_heads, cache.head_dim, cache.ctx)
    if not n:
        raise ValueError(f"attention_tree: no such shape (tokens {tokens}, heads {heads}, kv_heads {cache.kv_heads})")
    return torch.zeros(n, dtype=torch.uint8, device=cache.device)


def attention_tree(q, cache: KVCache, out=None, state=None, *, heads: int, scale: float, scratch, mask=None,
                   stream=None):
    """Node t's rotated queries q[t] (fp32 [T, heads * head_dim]) over the
    slots below state.pos and the tree slots of its mask row (int32 / uint32
    [T, ceil(T / 32)], bit j: node t sees node j; None: j <= t)."""
    dev, w, f32 = cache.index, heads * cache.head_dim, torch.float32
    ld = _rows2(q, f32, "q", dev, None, w)
    T = q.shape[0]
    st, n = _state_ptr(state, dev), 0 if scratch is None else scratch.numel()
    if out is None:
        out = _new((T, w), f32, cache, stream)
    if mask is not None:
        t = mask.dtype
        if t is not torch.int32 and t is not torch.uint32:
            raise TypeError("mask: int32 words wanted")
        mask = _flat(mask, t, "mask", dev, T * ((T + 31) // 32))
    _call(dev, stream, lib().odi_cuda_attention_tree, q.data_ptr(), ld, cache._ref, _flat(out, f32, "out", dev, T * w),
          mask, st, T, heads, scale, _flat(scratch, torch.uint8, "scratch", dev, n), n)
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
    bias_ids / bias [n] for all rows; mask int32 words [rows or 1, ceil(V / 32)].
    One row, also one expanded to all rows, serves them all; rows that overlap
    otherwise are refused."""
    dev, f32, i32 = logits.get_device(), torch.float32, torch.int32
    rows, V = logits.shape
    ld = _rows2(logits, f32, "logits", dev, rows, V)
    h = hl = ids = bv = mk = h_ld = H = nb = mk_ld = 0
    if history is not None:
        H = history.shape[1]
        h, h_ld = history.data_ptr(), _per_row(history, i32, "history", dev, rows, H)
        if history_lens is not None:
            hl = _flat(history_lens, i32, "history_lens", dev, rows)
    elif history_lens is not None:
        raise ValueError("logits_adjust: history_lens without a history")
    if bias_ids is not None:
        nb = bias_ids.numel()
        ids, bv = _flat(bias_ids, i32, "bias_ids", dev, nb), _flat(bias, f32, "bias", dev, nb)
    elif bias is not None:
        raise ValueError("logits_adjust: bias without bias_ids")
    if mask is not None:
        t = mask.dtype
        if t is not i32 and t is not torch.uint32:
            raise TypeError("mask: int32 words wanted")
        mk, mk_ld = mask.data_ptr(), _per_row(mask, t, "mask", dev, rows, (V + 31) // 32)
    o = _LOGITS_OPTS.pack(repeat_penalty, frequency_penalty, presence_penalty, h, h_ld, hl, H, ids, bv, nb, mk, mk_ld)
    if tokens is not None and scratch is None:
        raise ValueError("logits_adjust: tokens need a scratch (logits_scratch)")
    n = 0 if scratch is None else scratch.numel()
    _call(dev, stream, lib().odi_cuda_logits_adjust, logits.data_ptr(), ld, None if out is None else out.data_ptr(),
          0 if out is None else _rows2(out, f32, "out", dev, rows, V),
          None if tokens is None else _flat(tokens, i32, "tokens", dev, rows), rows, V, o,
          None if scratch is None else _flat(scratch, torch.uint8, "scratch", dev, n), n)
    return out, tokens


# what verify hands on to logits_adjust
_VERIFY_ADJUST = {"repeat_penalty", "frequency_penalty", "presence_penalty", "bias_ids", "bias", "mask"}


class DraftVerifier:
    """Greedy decoding of one sequence that checks drafted tokens, a tree of
    them per step: the model of decode.DecodeModel (its fused step, for T
    tokens at once) over a cache of fp16 or int8 rows.

        v = DraftVerifier(cfg, seeded_model(cfg, interleave_gate_up=False), cache="i8")
        v.start(prompt)
        new = v.verify(drafted_tokens, parents)   # 1 .. 1 + len(drafted) tokens

    The weights keep gate|up in [gate | up] order (the SwiGLU prologue reads
    it).  q_norms / k_norms: per-layer head_dim weights of models that norm q
    and k per head.  history: how many of the last tokens (the node's own
    ancestors included) the penalties of verify count.  Calls run on the current
    stream, which may differ from call to call; one at a time."""

    def __init__(self, cfg, weights, *, cache: str = "f16", max_nodes: int = 64, history: int = 0, q_norms=None,
                 k_norms=None, norm_eps: float = 1e-6, device=None):
        if weights.gu_interleaved:
            raise ValueError("DraftVerifier needs gate|up weights in [gate | up] order (interleave_gate_up=False)")
        if not 1 <= max_nodes <= TREE_MAX:
            raise ValueError(f"max_nodes: 1 to {TREE_MAX}")
        self.cfg, self.w = cfg, weights
        dev = torch.device("cuda" if device is None else device)
        self.device = dev = torch.device("cuda", torch.cuda.current_device()) if dev.index is None else dev
        self.max_nodes, self.history = max_nodes, history
        self.q_norms, self.k_norms, self.norm_eps = q_norms, k_norms, norm_eps
        self.caches = [KVCache.new(cache, cfg.kv_heads, cfg.head_dim, cfg.ctx, dev) for _ in range(cfg.layers)]
        T, f32 = max_nodes, torch.float32
        self.x = torch.empty((T, cfg.hidden), dtype=f32, device=dev)
        self.qkv = torch.empty((T, cfg.qkv_rows), dtype=f32, device=dev)
        self.q = torch.empty((T, cfg.heads * cfg.head_dim), dtype=f32, device=dev)
        self.attn = torch.empty_like(self.q)
        self.gu = torch.empty((T, 2 * cfg.ffn), dtype=f32, device=dev)
        self.logits = torch.empty((T, cfg.vocab), dtype=f32, device=dev)
        self.greedy = torch.empty(T, dtype=torch.int32, device=dev)
        # an odi_cuda_decode_state per node: its token, and the slot of node 0
        self.states = torch.zeros((T, 4), dtype=torch.int32, device=dev)
        self.scratch = attention_tree_scratch(self.caches[0], T, cfg.heads)
        self.logits_ws = logits_scratch(T, dev)
        # one workspace for all products (the steps' calls are on one stream), and
        # not the weights' own: other models and verifiers may run on those
        products = [dw for lw in weights.layers for dw in (lw.wqkv, lw.wo, lw.wgu, lw.wdown)] + [weights.output]
        self.products_ws = new_workspace(max(workspace_bytes(dw.dtype, T, dw.N, dw.K, cfg.act_mode) for dw in products), dev)
        self.pos, self.pending, self.tokens = 0, None, []
        # the last call's work, for a next call on another stream (the fills above,
        # rows on their way into place)
        self._last = torch.cuda.Event()
        self._last.record(torch.cuda.current_stream(dev))

    @contextlib.contextmanager
    def _ordered(self):
        """On the verifier's device, with the current stream after the last call's work."""
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream()
            stream.wait_event(self._last)
            try:
                yield
            finally:
                self._last.record(stream)

    # ---- the forward pass of T nodes --------------------------------------
    def _product(self, dw, x, y, T, norm=None, swiglu=False, accumulate=False):
        o = MatmulOpts(None if norm is None else norm.data_ptr(), self.cfg.eps, int(swiglu), int(accumulate), None, 0, None)
        ws = self.products_ws
        check(lib().odi_cuda_matmul_fused(dw.dtype, dw.data_ptr, x.data_ptr(), y.data_ptr(), T, dw.N, dw.K,
                                          self.cfg.act_mode, ws.data_ptr(), ws.numel(), FLAG_PDL, ctypes.byref(o),
                                          _raw_stream(self.device.index)))

    def _forward(self, tokens, depth, mask, logits: bool) -> None:
        """Nodes at slots pos .. pos + T - 1; logits rows 0 .. T - 1."""
        cfg, T = self.cfg, len(tokens)
        host = torch.tensor([[t, self.pos, 0, 0] for t in tokens], dtype=torch.int32)
        self.states[:T].copy_(host)
        state, stream = self.states[0], _raw_stream(self.device.index)
        for t in range(T):
            check(lib().odi_cuda_embed(self.w.token_embd.data_ptr(), cfg.vocab, cfg.hidden, self.states.data_ptr() + 16 * t,
                                       self.x.data_ptr() + 4 * cfg.hidden * t, None, None, None, stream))
        for i, lw in enumerate(self.w.layers):
            self._product(lw.wqkv, self.x, self.qkv, T, norm=lw.attn_norm)
            qk_rope_append(self.qkv[:T], self.caches[i], state, self.q[:T], heads=cfg.heads, theta=cfg.theta,
                           q_norm=self.q_norms[i] if self.q_norms else None,
                           k_norm=self.k_norms[i] if self.k_norms else None, eps=self.norm_eps, depth=depth)
            attention_tree(self.q[:T], self.caches[i], self.attn[:T], state, heads=cfg.heads,
                           scale=cfg.head_dim ** -0.5, scratch=self.scratch, mask=mask)
            self._product(lw.wo, self.attn, self.x, T, accumulate=True)
            self._product(lw.wgu, self.x, self.gu, T, norm=lw.ffn_norm)
            self._product(lw.wdown, self.gu, self.x, T, swiglu=True, accumulate=True)
        if logits:
            self._product(self.w.output, self.x, self.logits, T, norm=self.w.out_norm)

    def status(self) -> int:
        """OR of the device error words (0: no bounded wait gave up)."""
        words = [ws[:4].view(torch.int32) for ws in (self.scratch, self.products_ws)]
        v = 0
        for x in torch.cat(words).cpu().tolist():
            v |= x
        return v

    def _check(self) -> None:
        st = self.status()
        if st:
            raise RuntimeError(f"draft verification: a bounded device wait gave up (error word {st:#x})")

    # ---- sequences ---------------------------------------------------------
    def start(self, prompt) -> None:
        """A new sequence: all but the prompt's last token into the cache,
        max_nodes at a time; the last one is what verify starts from."""
        if not prompt or any(not 0 <= t < self.cfg.vocab for t in prompt):
            raise ValueError("start: a prompt of tokens of the vocabulary wanted")
        if len(prompt) > self.cfg.ctx:
            raise ValueError("prompt longer than the context")
        # no sequence until the prompt has run
        self.pos, self.pending, self.tokens = 0, None, list(prompt)
        with self._ordered():
            for i in range(0, len(prompt) - 1, self.max_nodes):
                chunk = prompt[i:min(i + self.max_nodes, len(prompt) - 1)]
                self._forward(chunk, None, None, False)
                self.pos += len(chunk)
            self._check()
        self.pending = prompt[-1]

    def verify(self, drafted=(), parents=None, **adjust) -> list:
        """Checks drafted tokens: node 0 is the pending token, drafted[i] is
        node i + 1 with parent node parents[i] <= i (None: a chain).  Returns
        the greedy tokens along the accepted path: one, plus one for every
        drafted token on it.  The last returned token is pending (not in the
        cache).  adjust: logits_adjust's penalties, biases and mask (mask rows
        per node, or one); without a history of the verifier's own also its
        history and history_lens."""
        other = set(adjust) - _VERIFY_ADJUST - (set() if self.history else {"history", "history_lens"})
        if other:
            raise TypeError(f"verify: no argument {', '.join(sorted(other))}" +
                            (" (the verifier counts its own history)" if self.history else ""))
        T = 1 + len(drafted)
        parents = list(range(T - 1)) if parents is None else list(parents)
        if self.pending is None:
            raise RuntimeError("verify: start a sequence first")
        if T > self.max_nodes or len(parents) != T - 1 or any(not 0 <= p <= i for i, p in enumerate(parents)):
            raise ValueError(f"verify: at most {self.max_nodes - 1} drafted tokens, each after its parent")
        if any(not 0 <= t < self.cfg.vocab for t in drafted):
            raise ValueError("verify: drafted token outside the vocabulary")
        if not self.history and adjust.get("history") is None and (
                adjust.get("repeat_penalty", 1.0), adjust.get("frequency_penalty", 0.0), adjust.get("presence_penalty", 0.0)) != (1.0, 0.0, 0.0):
            raise ValueError("verify: penalties count a history (DraftVerifier(history=...))")
        if self.pos + T > self.cfg.ctx:
            raise ValueError("verification would run past the context")
        nodes = [self.pending, *drafted]
        up = [-1, *parents]
        depth, sees, path = [], [], []
        for i, p in enumerate(up):
            depth.append(0 if p < 0 else depth[p] + 1)
            sees.append((0 if p < 0 else sees[p]) | (1 << i))
            path.append([i] if p < 0 else path[p] + [i])
        dev = self.device
        with self._ordered():
            W = (T + 31) // 32
            words = [[(s >> (32 * w)) & 0xFFFFFFFF for w in range(W)] for s in sees]
            mask = torch.tensor([[x - (1 << 32) if x >> 31 else x for x in r] for r in words], dtype=torch.int32).to(dev)
            self._forward(nodes, torch.tensor(depth, dtype=torch.int32).to(dev), mask, True)
            if self.history:
                rows = [(self.tokens + [nodes[j] for j in path[i][1:]])[-self.history:] for i in range(T)]
                H = max(len(r) for r in rows)
                adjust = {**adjust, "history": torch.tensor([r + [-1] * (H - len(r)) for r in rows], dtype=torch.int32).to(dev)}
            logits_adjust(self.logits[:T], self.logits[:T], self.greedy[:T], scratch=self.logits_ws, **adjust)
            greedy = self.greedy[:T].tolist()
            self._check()
            at, kept, out = 0, [0], [greedy[0]]
            while True:
                nxt = next((i for i in range(at + 1, T) if up[i] == at and nodes[i] == greedy[at]), None)
                if nxt is None:
                    break
                at = nxt
                kept.append(at)
                out.append(greedy[at])
            if out[-1] < 0:
                raise RuntimeError("verify: the mask allows no token")
            if kept != list(range(len(kept))):  # a branch: its rows to the slots after the root's
                src = torch.tensor(kept, dtype=torch.int32).to(dev)
                dst = torch.arange(len(kept), dtype=torch.int32).to(dev)
                for c in self.caches:
                    kv_move(c, src, dst, state=self.states[0])
        self.pos += len(kept)
        self.pending = out[-1]
        self.tokens += out
        return out
