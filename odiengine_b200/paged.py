"""Several requests over a paged KV cache: the operators of a step in which
every request brings new tokens (one, a chain of drafts, a chunk of its
prompt), on device tensors.

    paged_step              pages handed out, the step's rows and slots
    qk_rope_append_paged    per-head q/k norm + rotation, k and v rows into pages
    attention_paged         every new token over its request's pages
    verify_sampled          drafts against the target's probabilities

over :class:`PagedCache` (a layer's pages, fp16 or bf16), :class:`PageTables`
(who holds which page, one for all layers) and :class:`PagedBatch` (a step's
rows).  :class:`PagedDecoder` is the step made of them and of the library's
products, for the models of odiengine_b200.decode.  Calls are asynchronous on
`stream` (default: the tensors' device's current stream), where outputs that a
call makes are allocated too; tensors of another stream that are handed in are
the caller's to order and to keep (Tensor.record_stream).  Errors are
:class:`odiengine_b200.OdiCudaError`, or ValueError / TypeError for tensors
that do not fit.  Lengths and rows stay on the device, so calls can be captured
in a CUDA graph.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import FLAG_PDL, MatmulOpts, check, lib, new_workspace, workspace_bytes
from .draft import _call, _flat, _raw_stream, _refuse, _rows2, logits_adjust, logits_scratch

PAGED_DTYPES = {torch.float16: 0, torch.bfloat16: 1}  # ODI_CUDA_PAGED_*
PAGE_SIZES = (16, 32, 64, 128)
OUT_CACHE, OUT_F32 = 0, 1                             # ODI_CUDA_PAGED_OUT_*
# a step's status (ODI_CUDA_PAGED_*)
NO_PAGES, TOO_LONG, BAD_NEW, TOO_MANY_ROWS, BAD_KEEP, BAD_LENGTH = 1, 2, 4, 8, 16, 32


class _CacheStruct(ctypes.Structure):
    """odi_cuda_paged_cache (include/odi_cuda.h)."""

    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("dtype", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("page_size", ctypes.c_int), ("num_pages", ctypes.c_int)]


class _TablesStruct(ctypes.Structure):
    """odi_cuda_page_tables (include/odi_cuda.h)."""

    _fields_ = [("table", ctypes.c_void_p), ("lens", ctypes.c_void_p), ("free_pages", ctypes.c_void_p),
                ("free_count", ctypes.c_void_p), ("requests", ctypes.c_int), ("max_pages", ctypes.c_int),
                ("page_size", ctypes.c_int), ("num_pages", ctypes.c_int)]


class _BatchStruct(ctypes.Structure):
    """odi_cuda_paged_batch (include/odi_cuda.h)."""

    _fields_ = [("starts", ctypes.c_void_p), ("lens", ctypes.c_void_p), ("positions", ctypes.c_void_p),
                ("slots", ctypes.c_void_p), ("work", ctypes.c_void_p), ("requests", ctypes.c_int),
                ("max_rows", ctypes.c_int), ("max_new", ctypes.c_int), ("heads", ctypes.c_int),
                ("kv_heads", ctypes.c_int), ("page_size", ctypes.c_int)]


def _new(shape, dtype, device, stream):
    """An output that a call makes, allocated on the stream that writes it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _apart(what: str, handle, dev: int) -> None:
    raise ValueError(f"{what}: must be on cuda:{dev}, is on cuda:{handle.index}")


class PagedCache:
    """One layer's K and V: fp16 or bf16 [num_pages, kv_heads, page_size, head_dim]."""

    def __init__(self, k, v):
        if k.dtype not in PAGED_DTYPES:
            raise TypeError(f"cache k: fp16 or bf16 wanted, got {k.dtype}")
        if k.dim() != 4:
            raise ValueError(f"cache k: [num_pages, kv_heads, page_size, head_dim] wanted, got {tuple(k.shape)}")
        for t, n in ((k, "k"), (v, "v")):
            if t.dtype is not k.dtype or t.device != k.device or not t.is_cuda or not t.is_contiguous() or t.shape != k.shape:
                _refuse(t, k.dtype, f"cache {n}", k.get_device(), f"contiguous {tuple(k.shape)}")
            if t.data_ptr() % 16:
                raise ValueError(f"cache {n}: must be 16-byte aligned")
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        if self.page_size not in PAGE_SIZES or self.head_dim not in (64, 128):
            raise ValueError(f"cache: page_size of {PAGE_SIZES} and head_dim 64 or 128 wanted, got {tuple(k.shape)}")
        if abs(k.data_ptr() - v.data_ptr()) < k.numel() * 2:
            raise ValueError("cache: k and v share memory")
        self.k, self.v, self.dtype = k, v, k.dtype
        self.device, self.index = k.device, k.get_device()
        self._struct = _CacheStruct(k.data_ptr(), v.data_ptr(), PAGED_DTYPES[k.dtype], self.kv_heads, self.head_dim,
                                    self.page_size, self.num_pages)
        self._ref = ctypes.addressof(self._struct)

    @classmethod
    def new(cls, dtype, num_pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> "PagedCache":
        """Empty (zero) pages."""
        return cls(*(torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(2)))

    @property
    def nbytes(self) -> int:
        return 2 * self.k.numel() * 2


class PageTables:
    """Who holds which page.  int32 tensors: table [requests, max_pages], lens
    [requests], free [num_pages] (a stack of free pages) and free_count [1]."""

    def __init__(self, table, lens, free, free_count, page_size: int):
        i32, dev = torch.int32, table.get_device()
        if table.dim() != 2:
            raise ValueError(f"table: [requests, max_pages] wanted, got {tuple(table.shape)}")
        self.requests, self.max_pages = table.shape
        self.num_pages, self.page_size = free.numel(), page_size
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size: one of {PAGE_SIZES}")
        self._struct = _TablesStruct(
            _flat(table, i32, "table", dev, self.requests * self.max_pages), _flat(lens, i32, "lens", dev, self.requests),
            _flat(free, i32, "free", dev, self.num_pages), _flat(free_count, i32, "free_count", dev, 1), self.requests,
            self.max_pages, page_size, self.num_pages)
        self.table, self.lens, self.free, self.free_count = table, lens, free, free_count
        self.device, self.index = table.device, dev
        self._ref = ctypes.addressof(self._struct)

    @classmethod
    def new(cls, requests: int, max_pages: int, num_pages: int, page_size: int, device="cuda") -> "PageTables":
        """Tables of requests that hold nothing, every page free (page 0 is taken first)."""
        i32 = torch.int32
        return cls(torch.full((requests, max_pages), -1, dtype=i32, device=device), torch.zeros(requests, dtype=i32, device=device),
                   torch.arange(num_pages - 1, -1, -1, dtype=i32, device=device),
                   torch.full((1,), num_pages, dtype=i32, device=device), page_size)


class PagedBatch:
    """A step's rows, written by paged_step: starts [requests + 1], lens
    [requests], positions and slots [max_rows] (int32).  max_new: new tokens of
    one request at most; it says which attention kernel suits, so a batch of
    single tokens and one of prompts' chunks are best kept apart."""

    def __init__(self, tables: PageTables, *, max_rows: int, max_new: int, heads: int, kv_heads: int):
        n = lib().odi_cuda_paged_work_bytes(tables.requests, max_rows, max_new, heads, kv_heads)
        if not n:
            raise ValueError(f"no batch of {tables.requests} requests, max_rows {max_rows}, max_new {max_new}, heads {heads}, "
                             f"kv_heads {kv_heads}")
        new = lambda k: torch.zeros(k, dtype=torch.int32, device=tables.device)  # noqa: E731
        self.starts, self.lens = new(tables.requests + 1), new(tables.requests)
        self.positions, self.slots, self.work = new(max_rows), new(max_rows), new(n // 4)
        self.requests, self.max_rows, self.max_new, self.heads, self.kv_heads = tables.requests, max_rows, max_new, heads, kv_heads
        self.page_size, self.device, self.index = tables.page_size, tables.device, tables.index
        self._struct = _BatchStruct(self.starts.data_ptr(), self.lens.data_ptr(), self.positions.data_ptr(),
                                    self.slots.data_ptr(), self.work.data_ptr(), self.requests, max_rows, max_new, heads,
                                    kv_heads, self.page_size)
        self._ref = ctypes.addressof(self._struct)

    def status(self, stream=None) -> int:
        """The last step's status bits (NO_PAGES, ...).  `stream`: the step's, or one
        that comes after it (default: the current one); the call waits for it."""
        with contextlib.nullcontext() if stream is None else torch.cuda.stream(stream):
            return int(self.work[0].item())


def paged_step(tables: PageTables, batch: PagedBatch, new, keep=None, prefix=None, stream=None) -> None:
    """Request b keeps keep[b] of its positions (None: all) and takes new[b]
    more (int32 [requests]); prefix[b] positions see one another both ways.
    Tables and batch are brought up to date.  Pages are handed out in the
    requests' order: one that finds too few is refused (batch.status()), and with
    it those after it that need any."""
    dev, B = tables.index, tables.requests
    if batch.index != dev:
        _apart("batch", batch, dev)
    i32 = torch.int32
    _call(dev, stream, lib().odi_cuda_paged_step, tables._ref, batch._ref,
          None if keep is None else _flat(keep, i32, "keep", dev, B), _flat(new, i32, "new", dev, B),
          None if prefix is None else _flat(prefix, i32, "prefix", dev, B))


def qk_rope_append_paged(qkv, cache: PagedCache, batch: PagedBatch, q_out=None, *, heads: int, theta: float, q_norm=None,
                         k_norm=None, eps: float = 1e-6, stream=None):
    """The batch's rows of qkv [T, (heads + 2 kv_heads) * head_dim] fp32: q and
    k normed per head (q_norm / k_norm: head_dim weights, or None) and rotated
    at their positions, k and v stored at their slots.  Returns the rotated q
    in q_out [T, heads * head_dim] of the cache's type."""
    dev, hd, f32 = cache.index, cache.head_dim, torch.float32
    if batch.index != dev:
        _apart("batch", batch, dev)
    ld = _rows2(qkv, f32, "qkv", dev, None, (heads + 2 * cache.kv_heads) * hd)
    T = qkv.shape[0]
    if q_out is None:
        q_out = _new((T, heads * hd), cache.dtype, cache.device, stream)
    ld_q = _rows2(q_out, cache.dtype, "q_out", dev, T, heads * hd)
    _call(dev, stream, lib().odi_cuda_qk_rope_append_paged, qkv.data_ptr(), ld,
          None if q_norm is None else _flat(q_norm, f32, "q_norm", dev, hd),
          None if k_norm is None else _flat(k_norm, f32, "k_norm", dev, hd), eps, q_out.data_ptr(), ld_q, cache._ref,
          batch._ref, T, heads, theta)
    return q_out


def attention_paged_scratch(cache: PagedCache, batch: PagedBatch):
    """Zeroed scratch for attention_paged calls on one stream: of any layer, and
    of any batch that needs no more."""
    n = lib().odi_cuda_attention_paged_scratch_bytes(batch.requests, batch.max_rows, batch.max_new, batch.heads, batch.kv_heads,
                                                     cache.head_dim)
    return torch.zeros(n, dtype=torch.uint8, device=cache.device)


def attention_paged(q, cache: PagedCache, tables: PageTables, batch: PagedBatch, out=None, *, scale: float, softcap: float = 0.0,
                    slopes=None, scratch, stream=None):
    """The batch's rows of q (rotated, of the cache's type, [T, heads *
    head_dim]) over their requests' positions: those up to a row's own, and its
    request's prefix.  softcap: scores are capped by softcap * tanh(s /
    softcap); slopes fp32 [heads]: scores lose slope * distance.  out: of the
    cache's type (the default), with softmax weights of that type, or fp32, with
    weights of twice its bits; rows behind the batch's last are left."""
    dev, w = cache.index, batch.heads * cache.head_dim
    if tables.index != dev:
        _apart("tables", tables, dev)
    if batch.index != dev:
        _apart("batch", batch, dev)
    ld = _rows2(q, cache.dtype, "q", dev, None, w)
    T = q.shape[0]
    if out is None:
        out = _new((T, w), cache.dtype, cache.device, stream)
    o32 = out.dtype is torch.float32
    ld_o = _rows2(out, torch.float32 if o32 else cache.dtype, "out", dev, T, w)
    n = 0 if scratch is None else scratch.numel()
    _call(dev, stream, lib().odi_cuda_attention_paged, q.data_ptr(), ld, cache._ref, tables._ref, batch._ref, out.data_ptr(),
          ld_o, OUT_F32 if o32 else OUT_CACHE, T, scale, softcap,
          None if slopes is None else _flat(slopes, torch.float32, "slopes", dev, batch.heads),
          _flat(scratch, torch.uint8, "scratch", dev, n), n)
    return out


def verify_scratch(rows: int, requests: int, vocab: int, device="cuda"):
    """Zeroed scratch for verify_sampled calls of up to these sizes on one stream."""
    n = lib().odi_cuda_verify_scratch_bytes(rows, requests, vocab)
    if not n:
        raise ValueError(f"verify_sampled: no such sizes (rows {rows}, requests {requests}, vocabulary {vocab})")
    return torch.zeros(n, dtype=torch.uint8, device=device)


def verify_sampled(logits, tokens, starts, u_accept, u_next, accepted=None, next=None, *, temperature: float = 1.0,
                   draft_probs=None, scratch, stream=None):
    """Drafts against p = softmax(logits / temperature).  logits fp32 [rows, V],
    rows starts[b] .. starts[b + 1] - 1 (int32 [requests + 1]) being request
    b's; tokens int32 [rows]: each row's token, so row r judges the draft
    tokens[r + 1].  It is kept iff u_accept[r] * q < p, with q row r of
    draft_probs fp32 [rows, V] (None: 1).  Returns accepted and next (int32
    [requests]): drafts kept, and the token after them, drawn with u_next."""
    dev, f32, i32 = logits.get_device(), torch.float32, torch.int32
    if logits.dim() != 2 or starts.numel() < 2:
        raise ValueError(f"verify_sampled: logits [rows, V] and starts [requests + 1] wanted, got {tuple(logits.shape)} and {tuple(starts.shape)}")
    R, V = logits.shape
    B = starts.numel() - 1
    ld = _rows2(logits, f32, "logits", dev, R, V)
    if accepted is None:
        accepted = _new((B,), i32, logits.device, stream)
    if next is None:
        next = _new((B,), i32, logits.device, stream)
    n = 0 if scratch is None else scratch.numel()
    _call(dev, stream, lib().odi_cuda_verify_sampled, logits.data_ptr(), ld, _flat(tokens, i32, "tokens", dev, R),
          _flat(starts, i32, "starts", dev, B + 1), R, B, V, temperature,
          None if draft_probs is None else draft_probs.data_ptr(),
          0 if draft_probs is None else _rows2(draft_probs, f32, "draft_probs", dev, R, V),
          _flat(u_accept, f32, "u_accept", dev, R), _flat(u_next, f32, "u_next", dev, B), _flat(accepted, i32, "accepted", dev, B),
          _flat(next, i32, "next", dev, B), _flat(scratch, torch.uint8, "scratch", dev, n), n)
    return accepted, next


class PagedDecoder:
    """Decoding of several sequences at once, over one paged cache: the model of
    decode.DecodeModel for every request's new tokens in one pass.

        d = PagedDecoder(cfg, seeded_model(cfg, interleave_gate_up=False), requests=8, num_pages=512)
        a, b = d.add([1, 2, 3]), d.add(prompt)
        while d.left(b): d.step()          # prompts go in `chunk` tokens at a time
        new = d.step({a: [5, 9]})          # drafted tokens after a's pending one
        d.finish(a)                        # its pages are free again

    step returns, for every request whose prompt is in the cache, the tokens
    that follow: those drafts that the target keeps, and one more.  With a
    temperature they are sampled (drafts are verified by verify_sampled, random
    numbers from `generator` or a generator of its own); without one greedy.  The
    weights keep gate|up in [gate | up] order.  softcap, slopes: as
    attention_paged has them, for scores of q and k that are rotated as always.  Calls
    run on the current stream, which may differ from call to call; one at a time."""

    def __init__(self, cfg, weights, *, requests: int, num_pages: int, page_size: int = 16, dtype=torch.float16,
                 max_drafts: int = 7, chunk: int = 256, temperature=None, generator=None, softcap: float = 0.0, slopes=None,
                 device=None):
        if weights.gu_interleaved:
            raise ValueError("PagedDecoder needs gate|up weights in [gate | up] order (interleave_gate_up=False)")
        if max_drafts < 0 or chunk < 1 or requests < 1:
            raise ValueError("PagedDecoder: max_drafts 0 or more, chunk and requests 1 or more")
        if temperature is not None and not 1e-6 <= temperature <= 1e6:
            raise ValueError("temperature: 1e-6 to 1e6, or None for greedy decoding")
        self.cfg, self.w, self.temperature = cfg, weights, temperature
        dev = torch.device("cuda" if device is None else device)
        self.device = dev = torch.device("cuda", torch.cuda.current_device()) if dev.index is None else dev
        if weights.token_embd.get_device() != dev.index:
            raise ValueError(f"weights: must be on {dev}, are on {weights.token_embd.device}")
        self.requests, self.max_drafts, self.chunk = requests, max_drafts, chunk
        self.softcap, self.slopes = softcap, slopes
        self.page_size, self.num_pages = page_size, num_pages
        with torch.cuda.device(dev):
            self.caches = [PagedCache.new(dtype, num_pages, cfg.kv_heads, page_size, cfg.head_dim, dev) for _ in range(cfg.layers)]
            self.tables = PageTables.new(requests, -(-cfg.ctx // page_size), num_pages, page_size, dev)
            decode_rows = requests * (1 + max_drafts)
            self.rows = T = max(decode_rows, chunk)
            # single tokens, drafts and chunks apart: the batch's max_new chooses attention's kernel
            batch = lambda rows, new: PagedBatch(self.tables, max_rows=rows, max_new=new, heads=cfg.heads, kv_heads=cfg.kv_heads)  # noqa: E731
            self._single, self._drafts, self._chunks = batch(requests, 1), batch(decode_rows, 1 + max_drafts), batch(T, chunk)
            self.attention_ws = max((attention_paged_scratch(self.caches[0], b) for b in (self._single, self._drafts, self._chunks)),
                                    key=lambda ws: ws.numel())
            f32, w = torch.float32, cfg.heads * cfg.head_dim
            new = lambda *s, dt=f32: torch.empty(s, dtype=dt, device=dev)  # noqa: E731
            self.x, self.qkv, self.q = new(T, cfg.hidden), new(T, cfg.qkv_rows), new(T, w, dt=dtype)
            self.attn, self.gu = new(T, w), new(T, 2 * cfg.ffn)
            self.logits = new(decode_rows, cfg.vocab)
            self.states = torch.zeros((T, 4), dtype=torch.int32, device=dev)
            self.verify_ws = verify_scratch(decode_rows, requests, cfg.vocab, dev)
            self.greedy_ws, self.greedy = logits_scratch(decode_rows, dev), new(decode_rows, dt=torch.int32)
            self.generator = torch.Generator(device=dev) if generator is None else generator
            products = [m for lw in weights.layers for m in (lw.wqkv, lw.wo, lw.wgu, lw.wdown)] + [weights.output]
            self.products_ws = new_workspace(max(workspace_bytes(m.dtype, T, m.N, m.K, cfg.act_mode) for m in products), dev)
            self._last = torch.cuda.Event()
            self._last.record(torch.cuda.current_stream(dev))
        # per request: tokens to go into the cache (a prompt's rest, then the pending
        # token), and how many positions it holds; None: free
        self._todo, self._len = [None] * requests, [0] * requests

    @contextlib.contextmanager
    def _ordered(self):
        """On the decoder's device, with the current stream after the last call's work."""
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream()
            stream.wait_event(self._last)
            try:
                yield
            finally:
                self._last.record(stream)

    def _product(self, dw, x, y, T, norm=None, swiglu=False, accumulate=False):
        o = MatmulOpts(None if norm is None else norm.data_ptr(), self.cfg.eps, int(swiglu), int(accumulate), None, 0, None)
        ws = self.products_ws
        check(lib().odi_cuda_matmul_fused(dw.dtype, dw.data_ptr, x.data_ptr(), y.data_ptr(), T, dw.N, dw.K, self.cfg.act_mode,
                                          ws.data_ptr(), ws.numel(), FLAG_PDL, ctypes.byref(o), _raw_stream(self.device.index)))

    def _forward(self, batch: PagedBatch, tokens: dict, logits: bool) -> None:
        """The new tokens of some requests, {request: tokens}, in the requests' order."""
        cfg, rows = self.cfg, [t for b in range(self.requests) for t in tokens.get(b, ())]
        T, stream = len(rows), _raw_stream(self.device.index)
        host = torch.tensor([self._len, [len(tokens.get(b, ())) for b in range(self.requests)]], dtype=torch.int32)
        keep, fresh = host.to(self.device)
        paged_step(self.tables, batch, fresh, keep=keep)
        self.states[:T].copy_(torch.tensor([[t, 0, 0, 0] for t in rows], dtype=torch.int32))
        for r in range(T):
            check(lib().odi_cuda_embed(self.w.token_embd.data_ptr(), cfg.vocab, cfg.hidden, self.states.data_ptr() + 16 * r,
                                       self.x.data_ptr() + 4 * cfg.hidden * r, None, None, None, stream))
        for cache, lw in zip(self.caches, self.w.layers):
            self._product(lw.wqkv, self.x, self.qkv, T, norm=lw.attn_norm)
            qk_rope_append_paged(self.qkv[:T], cache, batch, self.q[:T], heads=cfg.heads, theta=cfg.theta)
            attention_paged(self.q[:T], cache, self.tables, batch, self.attn[:T], scale=cfg.head_dim ** -0.5,
                            softcap=self.softcap, slopes=self.slopes, scratch=self.attention_ws)
            self._product(lw.wo, self.attn, self.x, T, accumulate=True)
            self._product(lw.wgu, self.x, self.gu, T, norm=lw.ffn_norm)
            self._product(lw.wdown, self.gu, self.x, T, swiglu=True, accumulate=True)
        if logits:
            self._product(self.w.output, self.x, self.logits, T, norm=self.w.out_norm)

    def status(self) -> int:
        """OR of the device error words (0: no bounded wait gave up, every page was one)."""
        words = [ws[:4].view(torch.int32) for ws in (self.attention_ws, self.products_ws)]
        v = 0
        for x in torch.cat(words).cpu().tolist():
            v |= x
        return v

    def _check(self, batch: PagedBatch) -> None:
        st, refused = self.status(), batch.status()
        if st or refused:
            raise RuntimeError(f"paged decoding: a device wait gave up or a page was none (error word {st:#x}), or a request "
                               f"was refused (status {refused})")

    def _pages(self, n: int) -> int:
        return -(-n // self.page_size)

    @property
    def free_pages(self) -> int:
        """Pages that no request's positions need."""
        return self.num_pages - sum(self._pages(n) for n in self._len)

    # ---- requests ------------------------------------------------------------
    def add(self, prompt) -> int:
        """A new request; its prompt goes into the cache with the next steps."""
        prompt = list(prompt)
        if not prompt or any(not 0 <= t < self.cfg.vocab for t in prompt):
            raise ValueError("add: a prompt of tokens of the vocabulary wanted")
        if len(prompt) > self.cfg.ctx:
            raise ValueError("add: prompt longer than the context")
        b = next((b for b in range(self.requests) if self._todo[b] is None), None)
        if b is None:
            raise RuntimeError(f"add: all {self.requests} requests are in use")
        self._todo[b], self._len[b] = prompt, 0
        return b

    def left(self, request: int) -> int:
        """Prompt tokens that are not in the cache yet, but for the last."""
        return len(self._tokens(request)) - 1

    def finish(self, request: int) -> None:
        """The request is over: its pages go back with the next step."""
        self._tokens(request)
        self._todo[request], self._len[request] = None, 0

    def _tokens(self, b) -> list:
        if not 0 <= b < self.requests or self._todo[b] is None:
            raise ValueError(f"no request {b}")
        return self._todo[b]

    def step(self, drafts=None) -> dict:
        """One step of every request: a chunk of those whose prompt is not in the
        cache; the pending token, and drafts[request] after it, of the others.
        Returns {request: new tokens} of the latter; the last of them is pending."""
        drafts = dict(drafts or {})
        for b, d in drafts.items():
            if self.left(b):
                raise ValueError(f"step: request {b} has prompt left")
            if len(d) > self.max_drafts or any(not 0 <= t < self.cfg.vocab for t in d):
                raise ValueError(f"step: at most {self.max_drafts} drafted tokens of the vocabulary")
        live = [b for b in range(self.requests) if self._todo[b] is not None]
        room, chunks = self.chunk, {}
        for b in live:
            n = min(room, len(self._todo[b]) - 1)
            if n > 0:
                chunks[b] = self._todo[b][:n]
                room -= n
        decode = {b: [self._todo[b][0], *drafts.get(b, ())] for b in live if len(self._todo[b]) == 1}
        need = {b: self._len[b] + len(t) for b, t in (*chunks.items(), *decode.items())}
        if any(n > self.cfg.ctx for n in need.values()):
            raise ValueError("step: a request would run past the context")
        if sum(self._pages(need.get(b, self._len[b])) for b in range(self.requests)) > self.num_pages:
            raise RuntimeError("step: not enough free pages")
        out = {}
        with self._ordered():
            if chunks:
                self._forward(self._chunks, chunks, False)
                self._check(self._chunks)
                for b, t in chunks.items():
                    self._len[b] += len(t)
                    self._todo[b] = self._todo[b][len(t):]
            if decode:
                batch = self._single if all(len(t) == 1 for t in decode.values()) else self._drafts
                self._forward(batch, decode, True)
                accepted, nxt = self._choose(batch, decode)
                self._check(batch)
                if any(nxt[b] < 0 for b in decode):
                    raise RuntimeError("step: logits without a finite value")
                for b, t in decode.items():
                    out[b] = [*t[1:1 + accepted[b]], nxt[b]]
                    self._len[b] += 1 + accepted[b]
                    self._todo[b] = [nxt[b]]
        return out

    def _choose(self, batch: PagedBatch, decode: dict):
        """Drafts kept and the next token of each request, by the last pass's logits."""
        T = sum(len(t) for t in decode.values())
        if self.temperature is None:
            _, g = logits_adjust(self.logits[:T], None, self.greedy[:T], scratch=self.greedy_ws)
            greedy, accepted, nxt, r = g.tolist(), [0] * self.requests, [-1] * self.requests, 0
            for b in range(self.requests):
                t = decode.get(b, [])
                while accepted[b] + 1 < len(t) and t[accepted[b] + 1] == greedy[r + accepted[b]]:
                    accepted[b] += 1
                if t:
                    nxt[b] = greedy[r + accepted[b]]
                r += len(t)
            return accepted, nxt
        u = torch.rand(T + self.requests, device=self.device, generator=self.generator)
        self.u_accept, self.u_next = u[:T], u[T:]
        tokens = self.states[:T, 0].contiguous()
        accepted, nxt = verify_sampled(self.logits[:T], tokens, batch.starts, self.u_accept, self.u_next,
                                       temperature=self.temperature, scratch=self.verify_ws)
        return accepted.tolist(), nxt.tolist()
