"""Serving many requests over a paged KV cache: the decoder layer's cache operators (mimo_moe.layer's KVCache,
rope_store and attention hold one sequence) for a batch of requests of different lengths, with every length on the
device, so a step of any mix of decoding requests and prompt chunks needs no host synchronisation and a captured
decode step advances by itself when it is replayed.

    table  = PageTable(max_requests, max_len, num_pages, page_size)        # block tables, lengths, free pages
    caches = [PagedKVCache(layer.attn.cfg, num_pages, page_size) for layer in layers]
    step   = table.step(new_lens, tokens)       # pages, row offsets, positions, slots of this step's token rows
    q      = rope_store_paged(qkv, cfg, cache, step)
    o      = attention_paged(q, cache, cfg, step, sinks)
    table.release(done)                         # finished requests give their pages back

A step's token rows are its requests' new tokens, one request after another; rows behind the last one are padding.
`PagedDecoderStack` runs whole decoder layers this way.  The kernels are this library's (include/mimo_moe_paged.h);
there is no CPU path."""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import check, lib
from .layer import AttentionConfig, DecoderStack, bf16_value
from .ops import _need_cuda, _ptr, read_status

PAGE_SIZES = (16, 32, 64, 128)
MAX_REQUESTS = 4096


def _launch(dev: torch.device, where: str, fn, *args) -> None:
    """fn(*args, current stream of dev), on dev."""
    i = dev.index
    if i != torch._C._cuda_getDevice():
        with torch.cuda.device(i):
            return _launch(dev, where, fn, *args)
    rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))   # current_stream(dev).cuda_stream without the object
    if rc:
        check(rc, where)


def _int32(t: torch.Tensor, name: str, shape, dev=None) -> torch.Tensor:
    if t.dtype is torch.int32 and t.shape == shape and t.is_contiguous() and (t.is_cuda if dev is None
                                                                              else t.device == dev):
        return t
    _need_cuda(t, name)
    if dev is not None and t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {dev}")
    raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def _bf16(t: torch.Tensor, name: str, shape, dev) -> torch.Tensor:
    """An activation input: any float type and layout, cast and made contiguous (no-ops for the layers' own)."""
    if t.shape != shape or t.device != dev:
        _need_cuda(t, name)
        raise ValueError(f"{name} must have shape {tuple(shape)} on {dev}, got {tuple(t.shape)} on {t.device}")
    return t if t.dtype is torch.bfloat16 and t.is_contiguous() else t.to(torch.bfloat16).contiguous()


def _buffer(t: torch.Tensor, name: str, shape, dev) -> torch.Tensor:
    """A tensor the kernels write: taken as it is."""
    if t.shape != shape or t.device != dev or t.dtype is not torch.bfloat16 or not t.is_cuda or not t.is_contiguous():
        _need_cuda(t, name)
        raise ValueError(f"{name} must be a contiguous bf16 tensor of shape {tuple(shape)} on {dev}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t


def _check_status(status: torch.Tensor, where: str) -> None:
    try:
        read_status(status, where, "no free pages left, a length or a row count that does not fit, or a page or slot "
                                   "outside the pool")
    finally:
        status.zero_()


def _page_size(page_size: int) -> int:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    return int(page_size)


class PageStep:
    """The row layout of one step of R requests (what page_plan writes; a program with a page allocator of its own
    fills it itself, with a slot of its own for every row): block_table int32 [R, width], cu_q int32 [R + 1], seq_lens
    int32 [R] (lengths with the step's tokens), positions and slots int32 [tokens].  n_free int32 [1] and status int32
    [1] are page_plan's."""

    def __init__(self, *, block_table: torch.Tensor, page_size: int, cu_q: torch.Tensor, seq_lens: torch.Tensor,
                 positions: torch.Tensor, slots: torch.Tensor, n_free: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None):
        _need_cuda(block_table, "block_table")
        if block_table.dim() != 2:
            raise ValueError("block_table must be a matrix: a row of page numbers for each request")
        R, dev = block_table.shape[0], block_table.device
        if not 1 <= R <= MAX_REQUESTS:
            raise ValueError(f"a step has 1 to {MAX_REQUESTS} requests, got {R}")
        if positions.dim() != 1:
            raise ValueError("positions must be a vector: one position for each token row")
        T = positions.shape[0]
        self.page_size = _page_size(page_size)
        self.block_table = _int32(block_table, "block_table", block_table.shape)
        self.cu_q = _int32(cu_q, "cu_q", (R + 1,), dev)
        self.seq_lens = _int32(seq_lens, "seq_lens", (R,), dev)
        self.positions = _int32(positions, "positions", (T,), dev)
        self.slots = _int32(slots, "slots", (T,), dev)
        self.n_free = None if n_free is None else _int32(n_free, "n_free", (1,), dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev) if status is None else _int32(status, "status",
                                                                                                 (1,), dev)
        self.requests, self.width, self.tokens, self.device = R, block_table.shape[1], T, dev
        self.version = 0      # how often its lengths were planned anew: an attention plan goes with one of them
        self.rows = _Rows()   # scratch of the layers that work on this step, one after another

    @classmethod
    def empty(cls, requests: int, tokens: int, block_table: torch.Tensor, page_size: int,
              status: Optional[torch.Tensor] = None) -> "PageStep":
        """Buffers for page_plan(..., out=)."""
        _need_cuda(block_table, "block_table")
        if tokens < 0:
            raise ValueError(f"a step has no {tokens} token rows")
        dev = block_table.device
        return cls(block_table=block_table, page_size=page_size,
                   cu_q=torch.zeros(requests + 1, dtype=torch.int32, device=dev),
                   seq_lens=torch.zeros(requests, dtype=torch.int32, device=dev),
                   positions=torch.full((tokens,), -1, dtype=torch.int32, device=dev),
                   slots=torch.full((tokens,), -1, dtype=torch.int32, device=dev),
                   n_free=torch.zeros(1, dtype=torch.int32, device=dev), status=status)

    def last_rows(self) -> torch.Tensor:
        """The row of each request's last new token, int32 [R] (the rows whose hidden state goes to the lm_head); a
        request without new tokens has the row before its own, -1 for the first."""
        return self.cu_q[1:] - 1

    def check(self, where: str = "paged step") -> None:
        """Synchronise on the status word: ValueError for pages that ran out and lengths or pages that do not fit,
        MimoError for an expired wait.  Clears it."""
        _check_status(self.status, where)


def page_plan(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
              n_free: torch.Tensor, page_size: int, tokens: int, out: Optional[PageStep] = None) -> PageStep:
    """Plan a step in which request r brings new_lens[r] tokens to the lens[r] it holds: takes the pages it needs from
    the end of free_pages[:n_free], writes them into block_table (in place) and returns the step's row layout.  lens
    and n_free stay as they are; the step's seq_lens and n_free are the new ones.  When the pages do not suffice, or a
    length does not fit, the step is one without new tokens and its status says so (PageStep.check)."""
    if out is None:
        out = PageStep.empty(block_table.shape[0], tokens, block_table, page_size)
    elif out.block_table is not block_table or out.tokens != tokens or out.page_size != page_size \
            or out.n_free is None:
        raise ValueError("page_plan: out is a step of other rows, pages or another block table")
    R, dev = out.requests, out.device
    if free_pages.dim() != 1:
        raise ValueError("free_pages must be a vector")
    _int32(lens, "lens", (R,), dev)
    _int32(new_lens, "new_lens", (R,), dev)
    _int32(free_pages, "free_pages", free_pages.shape, dev)
    _int32(n_free, "n_free", (1,), dev)
    _launch(dev, "page_plan", lib().mimo_moe_page_plan, lens.data_ptr(), new_lens.data_ptr(), R, block_table.data_ptr(),
            out.width, free_pages.data_ptr(), n_free.data_ptr(), free_pages.shape[0], out.page_size, tokens,
            out.cu_q.data_ptr(), out.seq_lens.data_ptr(), out.n_free.data_ptr(), out.positions.data_ptr(),
            out.slots.data_ptr(), out.status.data_ptr())
    out.version += 1
    return out


def page_release(done: torch.Tensor, lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 n_free: torch.Tensor, page_size: int, status: Optional[torch.Tensor] = None) -> None:
    """Return the pages of the requests with done[r] (bool or uint8 [R]) to the free list; their lens become 0 and
    their table entries -1.  All in place."""
    _need_cuda(done, "done")
    dev, R = block_table.device, block_table.shape[0]
    if done.dtype not in (torch.bool, torch.uint8) or tuple(done.shape) != (R,) or not done.is_contiguous() \
            or done.device != dev:
        raise ValueError(f"done must be a contiguous bool tensor of {R} requests on {dev}")
    if free_pages.dim() != 1:
        raise ValueError("free_pages must be a vector")
    _int32(block_table, "block_table", block_table.shape)
    _int32(lens, "lens", (R,), dev)
    _int32(free_pages, "free_pages", free_pages.shape, dev)
    _int32(n_free, "n_free", (1,), dev)
    _launch(dev, "page_release", lib().mimo_moe_page_release, done.data_ptr(), R, lens.data_ptr(),
            block_table.data_ptr(), block_table.shape[1], free_pages.data_ptr(), n_free.data_ptr(), free_pages.shape[0],
            _page_size(page_size), _ptr(status))


class _Rows:
    """Buffers with a row for each token of a step, grown as steps of more rows come.  A buffer that was outgrown is
    kept: a captured graph may hold its address."""

    def __init__(self):
        self._bufs, self._outgrown = {}, []

    def get(self, key, rows: int, make) -> torch.Tensor:
        """The first `rows` rows of the buffer `key`; make(n) makes one of n rows."""
        buf = self._bufs.get(key)
        if buf is None or buf.shape[0] < rows:
            if buf is not None:
                self._outgrown.append(buf)
            buf = self._bufs[key] = make(max(rows, 2 * buf.shape[0] if buf is not None else rows))
        return buf[:rows]


class PageTable:
    """Block tables, lengths and free pages of up to max_requests requests of at most max_len tokens, over pools of
    num_pages pages.  Row r of every tensor is request r; a free row has length 0."""

    def __init__(self, max_requests: int, max_len: int, num_pages: int, page_size: int = 64, device=None):
        dev = torch.device(device or "cuda")
        self.page_size = _page_size(page_size)
        if not 1 <= max_requests <= MAX_REQUESTS or max_len < 1 or num_pages < 1 \
                or num_pages * page_size > 2**31 - 1 or max_len > 2**31 - 1 - page_size:
            raise ValueError(f"page table: {max_requests} requests of {max_len} tokens over {num_pages} pages of "
                             f"{page_size}")
        self.num_pages = int(num_pages)
        width = -(-max_len // self.page_size)
        self.block_table = torch.full((max_requests, width), -1, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=dev)  # page 0 is taken first
        self._state = torch.zeros(max_requests + 1, dtype=torch.int32, device=dev)
        self._state[max_requests:] = num_pages
        self.lens, self.n_free = self._state[:max_requests], self._state[max_requests:]
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.requests, self.device = int(max_requests), self.block_table.device
        self._cu_q = torch.zeros(max_requests + 1, dtype=torch.int32, device=dev)
        self._after = torch.zeros(max_requests + 1, dtype=torch.int32, device=dev)   # the step's lengths and free pages
        self._rows = _Rows()
        self._step: Optional[PageStep] = None   # the one planned last

    def step(self, new_lens: torch.Tensor, tokens: int) -> PageStep:
        """Plan a step (page_plan) and take its lengths and free pages over.  The step's buffers are the table's: the
        next step writes them again."""
        if tokens < 0:
            raise ValueError(f"a step has no {tokens} token rows")
        R = self.requests

        def rows(n):
            return torch.empty(n, dtype=torch.int32, device=self.device)

        out = PageStep(block_table=self.block_table, page_size=self.page_size, cu_q=self._cu_q,
                       seq_lens=self._after[:R], positions=self._rows.get("positions", tokens, rows),
                       slots=self._rows.get("slots", tokens, rows), n_free=self._after[R:], status=self.status)
        out.rows = self._rows
        page_plan(self.lens, new_lens, self.block_table, self.free_pages, self.n_free, self.page_size, tokens, out=out)
        if self._step is not None:
            self._step.version += 1   # its buffers are the new step's
        self._step = out
        self._state.copy_(self._after)
        return out

    def last_rows(self) -> torch.Tensor:
        """PageStep.last_rows of the step planned last."""
        return self._cu_q[1:] - 1

    def release(self, done: torch.Tensor) -> None:
        """Give back the pages of the requests with done[r]."""
        page_release(done, self.lens, self.block_table, self.free_pages, self.n_free, self.page_size, self.status)


class PagedKVCache:
    """Paged KV cache of one attention layer: k [num_pages, n_kv, page_size, head_dim], v [num_pages, n_kv, page_size,
    v_head_dim] bf16 (new and zeroed, or the tensors given).  `step` is the PageStep the layer's next call works on,
    `plan` that step's attention plan for the layer's kind (None: made at the call)."""

    paged = True

    def __init__(self, cfg: AttentionConfig, num_pages: int, page_size: int = 64, device=None,
                 k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None):
        self.cfg, self.num_pages, self.page_size = cfg, int(num_pages), _page_size(page_size)
        ks = (self.num_pages, cfg.n_kv_heads, self.page_size, cfg.head_dim)
        vs = (self.num_pages, cfg.n_kv_heads, self.page_size, cfg.v_head_dim)
        if (k is None) != (v is None):
            raise ValueError("PagedKVCache: give both k and v, or neither")
        if k is None:
            dev = torch.device(device or "cuda")
            k = torch.zeros(ks, dtype=torch.bfloat16, device=dev)
            v = torch.zeros(vs, dtype=torch.bfloat16, device=dev)
        self.k, self.v = _buffer(k, "k", ks, k.device), _buffer(v, "v", vs, k.device)
        self.device = k.device
        self.step: Optional[PageStep] = None
        self.plan: Optional["AttentionPlan"] = None

    def attend(self, qkv: torch.Tensor, sinks: Optional[torch.Tensor]) -> torch.Tensor:
        """The layer's cache half (RoPE + append, attention) for the projection rows of `step`'s tokens.  The result is
        the step's scratch, which the next layer's call writes again; its padding rows are zero."""
        step, cfg = self.step, self.cfg
        if step is None:
            raise ValueError("PagedKVCache: no step set (cache.step = table.step(new_lens, tokens))")
        _fits(self, cfg, step, "PagedKVCache")   # before the scratch is made on this cache's device

        def rows(n):
            return torch.zeros(n, cfg.n_heads, cfg.v_head_dim, dtype=torch.bfloat16, device=self.device)

        out = step.rows.get(("attention", cfg.n_heads, cfg.v_head_dim), step.tokens, rows)
        q = rope_store_paged(qkv, cfg, self, step, clear=out)
        return attention_paged(q, self, cfg, step, sinks, plan=self.plan, out=out)


def _fits(cache: PagedKVCache, cfg: AttentionConfig, step: PageStep, where: str) -> None:
    if (cache.page_size, cache.device) != (step.page_size, step.device):
        raise ValueError(f"{where}: the cache has pages of {cache.page_size} on {cache.device}, the step pages of "
                         f"{step.page_size} on {step.device}")
    own = cache.cfg
    if own is not cfg and (own.n_kv_heads, own.head_dim, own.v_head_dim) != (cfg.n_kv_heads, cfg.head_dim,
                                                                             cfg.v_head_dim):
        raise ValueError(f"{where}: the cache was made for another attention config")


def rope_store_paged(qkv: torch.Tensor, cfg: AttentionConfig, cache: PagedKVCache, step: PageStep,
                     q_out: Optional[torch.Tensor] = None, clear: Optional[torch.Tensor] = None) -> torch.Tensor:
    """mimo_moe.layer.rope_store for a step's token rows: RoPE on q and k at each row's position, v * the value scale,
    k and v to each row's cache slot.  Returns q bf16 [tokens, n_heads, head_dim]; padding rows are not written.  clear:
    the attention's `out` (bf16 [tokens, n_heads, v_head_dim]), whose padding rows (those without a slot) become zero."""
    _fits(cache, cfg, step, "rope_store_paged")
    T, dev = step.tokens, step.device
    qkv = _bf16(qkv, "qkv", (T, cfg.qkv_width), dev)
    shape = (T, cfg.n_heads, cfg.head_dim)
    q = torch.empty(shape, dtype=torch.bfloat16, device=dev) if q_out is None else _buffer(q_out, "q_out", shape, dev)
    entry, more = lib().mimo_moe_paged_rope_store, ()
    if clear is not None:
        _buffer(clear, "clear", (T, cfg.n_heads, cfg.v_head_dim), dev)
        entry, more = lib().mimo_moe_paged_rope_store_clear, (clear.data_ptr(), cfg.n_heads * cfg.v_head_dim)
    if T == 0:
        return q
    vs = 0.0 if cfg.v_scale is None else bf16_value(cfg.v_scale)
    _launch(dev, "rope_store_paged", entry, qkv.data_ptr(), T, cfg.n_heads, cfg.n_kv_heads,
            cfg.head_dim, cfg.v_head_dim, cfg.rotary_dim, cfg.rope_theta, vs, step.positions.data_ptr(),
            step.slots.data_ptr(), cache.num_pages, cache.page_size, q.data_ptr(), cache.k.data_ptr(),
            cache.v.data_ptr(), *more, step.status.data_ptr())
    return q


def _kind(cfg: AttentionConfig):
    """What layers of one attention plan have in common."""
    return cfg.n_heads, cfg.n_kv_heads, cfg.window, cfg.keep_first


class AttentionPlan:
    """How attention_paged deals a step's work to the SMs, made from the step's lengths: one for all layers with the
    same heads, window and keep_first (attention_plan).  It holds until the step's lengths change: attention_paged refuses
    it after another page_plan into the step or a later step of the same table, until update().  (A program that writes
    cu_q or seq_lens itself, or replays a graph that does, calls update() itself.)"""

    def __init__(self, step: PageStep, cfg: AttentionConfig):
        if cfg.keep_first and not cfg.window:
            raise ValueError("attention_plan: keep_first needs a window (without one every earlier token is visible)")
        if cfg.n_heads < 1 or cfg.n_kv_heads < 1 or cfg.n_heads % cfg.n_kv_heads or cfg.n_heads // cfg.n_kv_heads > 128:
            raise ValueError(f"attention_plan: {cfg.n_heads} heads over {cfg.n_kv_heads} kv heads")
        self.step, self.kind, self.version = step, _kind(cfg), step.version
        self.buffer, self._ws = None, {}
        if step.tokens == 0:
            return
        with torch.cuda.device(step.device):
            nb = lib().mimo_moe_paged_attention_plan_bytes(step.tokens, step.requests, cfg.n_heads, cfg.n_kv_heads)
            self.buffer = torch.empty(nb, dtype=torch.uint8, device=step.device)
        self.update()

    def workspace_bytes(self, v_head_dim: int) -> int:
        nb = self._ws.get(v_head_dim)
        if nb is None:
            with torch.cuda.device(self.step.device):
                nb = self._ws[v_head_dim] = lib().mimo_moe_paged_attention_workspace_bytes(
                    self.step.tokens, self.step.requests, self.kind[0], self.kind[1], v_head_dim)
        return nb

    def update(self) -> None:
        """Make the plan again from the step's present lengths, in the same buffer."""
        step, (nq, nkv, window, keep) = self.step, self.kind
        if self.buffer is not None:
            _launch(step.device, "attention_plan", lib().mimo_moe_paged_attention_plan, step.cu_q.data_ptr(),
                    step.seq_lens.data_ptr(), step.requests, step.tokens, nq, nkv, window, keep, step.width,
                    step.page_size, self.buffer.data_ptr(), self.buffer.numel(), step.status.data_ptr())
        self.version = step.version


def attention_plan(step: PageStep, cfg: AttentionConfig) -> AttentionPlan:
    """The plan of a step for the layers of cfg's kind, for attention_paged(..., plan=)."""
    return AttentionPlan(step, cfg)


def attention_paged(q: torch.Tensor, cache: PagedKVCache, cfg: AttentionConfig, step: PageStep,
                    sinks: Optional[torch.Tensor] = None, plan: Optional[AttentionPlan] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """mimo_moe.layer.attention for a step's token rows over the paged cache: causal; with cfg.window a sliding window,
    in which each request's first cfg.keep_first tokens stay visible; sinks float32 [n_heads].  plan: the step's
    attention_plan for this kind of layer (made for this call when None).  Cache slots that no query of the step sees
    may hold anything; v at a position that one query sees must be finite for the request's earlier queries too, and
    below 2^40 in magnitude.
    Returns bf16 [tokens, n_heads, v_head_dim]; padding rows of a given `out` are not written, those of a new one are
    zero."""
    _fits(cache, cfg, step, "attention_paged")
    T, dev = step.tokens, step.device
    q = _bf16(q, "q", (T, cfg.n_heads, cfg.head_dim), dev)
    shape = (T, cfg.n_heads, cfg.v_head_dim)
    o = torch.zeros(shape, dtype=torch.bfloat16, device=dev) if out is None else _buffer(out, "out", shape, dev)
    if sinks is not None:
        if tuple(sinks.shape) != (cfg.n_heads,):
            raise ValueError(f"attention_paged: {cfg.n_heads} heads need as many sinks, got {tuple(sinks.shape)}")
        sinks = sinks.to(device=dev, dtype=torch.float32).contiguous()
    if plan is None:
        plan = AttentionPlan(step, cfg)
    elif plan.step is not step or plan.kind != _kind(cfg):
        raise ValueError("attention_paged: the plan was made for another step or kind of layer")
    elif plan.version != step.version:
        raise ValueError("attention_paged: the step's lengths were planned anew since its attention plan was made "
                         "(plan.update() makes it again)")
    if T == 0:
        return o
    nb = plan.workspace_bytes(cfg.v_head_dim)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)   # the call's own: two streams or graphs never share it
    _launch(dev, "attention_paged", lib().mimo_moe_paged_attention, q.data_ptr(), cache.k.data_ptr(),
            cache.v.data_ptr(), _ptr(sinks), step.block_table.data_ptr(), step.width, step.requests, T, cfg.n_heads,
            cfg.n_kv_heads, cfg.head_dim, cfg.v_head_dim, cfg.scale, cfg.window, cfg.keep_first, cache.num_pages,
            cache.page_size, plan.buffer.data_ptr(), plan.buffer.numel(), o.data_ptr(), ws.data_ptr(), nb,
            step.status.data_ptr())
    return o


class PagedDecoderStack(DecoderStack):
    """DecoderStack for many requests: one PageTable and a PagedKVCache per layer.  __call__(x bf16 [tokens, hidden],
    new_lens int32 [max_requests]) plans the step, runs the layers and returns the rows' hidden states (a buffer of the
    stack's, which the next call writes again); the lengths advance on the device, so a decode step captured once as a
    CUDA graph serves the tokens that follow as well.  `release(done)` frees finished requests' rows; `check()` raises
    when a step could not be planned (it then ran without new tokens).  Padding rows of x need only be finite.  One table
    serves all layers, so sliding-window layers hold every token of a request too, not a window of them."""

    def __init__(self, layers, max_requests: int, max_len: int, num_pages: int, page_size: int = 64):
        if not layers:
            raise ValueError("empty stack")
        self.layers = list(layers)
        dev = self.layers[0].attn.w_o.device
        self.hidden = self.layers[0].attn.w_o.shape[0]
        self.table = PageTable(max_requests, max_len, num_pages, page_size, dev)
        self.caches = [PagedKVCache(l.attn.cfg, num_pages, page_size, dev) for l in self.layers]

    def at(self, pos: int) -> "PagedDecoderStack":
        raise ValueError("a paged stack has a position for every request: table.lens")

    @property
    def offset(self) -> torch.Tensor:
        return self.table.lens

    def release(self, done: torch.Tensor) -> None:
        self.table.release(done)

    def check(self) -> None:
        """Synchronise on the status word of the table's steps (PageStep.check)."""
        _check_status(self.table.status, "paged stack")

    def _result(self, h: torch.Tensor) -> torch.Tensor:
        return self.table._rows.get(("result", h.shape[1]), h.shape[0],
                                    lambda n: torch.empty(n, h.shape[1], dtype=h.dtype, device=h.device))

    def __call__(self, x: torch.Tensor, new_lens: torch.Tensor) -> torch.Tensor:
        _need_cuda(x, "x")
        if x.dim() != 2 or x.shape[1] != self.hidden or x.device != self.table.device:
            raise ValueError(f"paged stack: x must have shape [tokens, {self.hidden}] on {self.table.device}, got "
                             f"{tuple(x.shape)} on {x.device}")
        step = self.table.step(new_lens, x.shape[0])
        if step.tokens == 0:
            return x.to(torch.bfloat16)
        plans = {}
        for c in self.caches:   # one attention plan for each kind of layer
            kind = _kind(c.cfg)
            if kind not in plans:
                plans[kind] = attention_plan(step, c.cfg)
            c.step, c.plan = step, plans[kind]
        return super().__call__(x)


__all__ = ["AttentionPlan", "PageStep", "PageTable", "PagedDecoderStack", "PagedKVCache", "attention_paged",
           "attention_plan", "page_plan", "page_release", "rope_store_paged"]
