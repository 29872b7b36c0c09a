"""A paged key-value cache and the attention that reads it.

``PagedCache`` holds a pool of pages and the requests' tables into it, all on
the device: the layout of a page is the reference's FlashInfer engine's
(m8than/yapd ``chatterbox_flash/engines/flashinfer.py:110-115``, blocks of
``(2, page_size, kv_heads, head_dim)``), the slots are the engines' request rows
(``server/engine.py:332``).  One tick of an autoregressive engine
(``server/engine_ar.py:382-422``) is::

    cache.reserve(1)                            # room for the token of every slot
    for layer in range(layers):
        q, k, v = project(layer, hidden)        # (B, heads, D), (B, kv_heads, D) twice
        hidden = finish(layer, cache.attend(layer, q, k, v))
    token = sample_rows(head(hidden))

A block-diffusion engine reserves its 16 positions once and calls ``attend``
with ``causal=False`` at every step (``server/engine.py:512-515``): the block's
keys and values are stored again each time and every position sees the block.

Everything runs the kernels of ``libyapd_select.so`` on the current CUDA stream
and synchronises nothing.  Lists of slots, pages and token counts are device
tensors; what only the device can see wrong in them (a full pool, a slot listed
twice) leaves the slot alone and sets bits of ``cache.status()``.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _native as N

_DTYPES = {torch.float32: N.YAPD_DTYPE_F32, torch.bfloat16: N.YAPD_DTYPE_BF16, torch.float16: N.YAPD_DTYPE_F16}

_MOST = 2 ** 63 - 1  # larger numbers would be cut off on their way to the library


class PagedCache:
    """Pages ``kv`` ``(layers, pages, 2, page_size, kv_heads, head_dim)`` in
    float32, bfloat16 or float16, with the tables of ``slots`` requests.

    ``page_table`` ``(slots, max_pages)`` int32 (-1: no page), ``kv_len``
    ``(slots,)`` int64 and ``refs`` ``(pages,)`` int32 are the caller's tensors,
    updated in place; ``PagedCache.empty`` makes them.  A slot whose length is
    negative or more than its table holds is empty to ``attend`` and left alone by
    the page operations, but for ``free``.  Each page's block has to
    be contiguous; the first two strides of ``kv`` are free.  ``head_dim`` is 32,
    64, 96 or 128.  The cache's calls share a workspace: they are ordered on one
    stream, or by events where a program uses several.  Threads may share a
    cache: a call's arguments and launches are one step to the others.
    """

    def __init__(self, kv: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor, refs: torch.Tensor):
        if not kv.is_cuda:
            raise ValueError("PagedCache runs on CUDA tensors only (no CPU fallback)")
        if kv.dtype not in _DTYPES:
            raise TypeError(f"kv must be float32, bfloat16 or float16, got {kv.dtype}")
        if kv.dim() != 6 or kv.shape[2] != 2:
            raise ValueError("kv must be (layers, pages, 2, page_size, kv_heads, head_dim)")
        if kv.shape[5] not in (32, 64, 96, 128):
            raise ValueError(f"head_dim must be 32, 64, 96 or 128, got {kv.shape[5]}")
        if kv.numel() == 0 or not kv[0, 0].is_contiguous():
            raise ValueError("each page of kv must be contiguous, and there must be one")
        layers, pages = kv.shape[:2]
        dev = kv.device
        slots = kv_len.shape[0] if kv_len.dim() == 1 else 0
        if slots < 1 or page_table.dim() != 2 or page_table.shape[0] != slots:
            raise ValueError("kv_len must be (slots,) and page_table (slots, max_pages)")
        for name, t, dtype, shape in (("page_table", page_table, torch.int32, tuple(page_table.shape)),
                                      ("kv_len", kv_len, torch.int64, (slots,)), ("refs", refs, torch.int32, (pages,))):
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous() or t.device != dev:
                raise ValueError(f"{name} must be a contiguous {dtype} {shape} tensor on {dev}")
        self.kv, self.page_table, self.kv_len, self.refs = kv, page_table, kv_len, refs
        self.slots, self.device = slots, dev
        self._vec = 16 // kv.element_size()
        self._layers, self._heads, self._dim, self._dtype, self._index = layers, kv.shape[4], kv.shape[5], kv.dtype, \
            kv.get_device()
        c = N.Cache()
        c.layers, c.pages, _, c.page_size, c.kv_heads, c.head_dim = kv.shape
        c.dtype, c.slots, c.max_pages = _DTYPES[kv.dtype], slots, page_table.shape[1]
        c.kv = kv.data_ptr()
        c.stride_layer, c.stride_page = kv.stride(0), kv.stride(1)
        c.page_table, c.kv_len, c.refs = page_table.data_ptr(), kv_len.data_ptr(), refs.data_ptr()
        self._lib = N.lib()
        need = self._lib.yapd_cache_workspace_size(C.byref(c))
        if need == 0:
            raise ValueError("page_size, kv_heads or max_pages * page_size is out of range")
        self._workspace = torch.zeros(need, dtype=torch.uint8, device=dev)
        c.workspace, c.workspace_bytes = self._workspace.data_ptr(), need
        # the argument structures are kept from call to call, and a call's kernels share the workspace
        self._lock = threading.Lock()
        self._pages = N.PagesArgs()
        self._cache = self._pages.cache = c
        self._scale, self._plans = self._dim ** -0.5, {}

    @classmethod
    def empty(cls, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, slots: int,
              max_pages: int, dtype=torch.bfloat16, device="cuda") -> "PagedCache":
        """A pool of free pages and empty slots, each with room for ``max_pages`` pages."""
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        return cls(torch.empty(layers, pages, 2, page_size, kv_heads, head_dim, dtype=dtype, device=dev),
                   torch.full((slots, max_pages), -1, dtype=torch.int32, device=dev),
                   torch.zeros(slots, dtype=torch.int64, device=dev),
                   torch.zeros(pages, dtype=torch.int32, device=dev))

    # ------------------------------------------------------------- attention

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor | None = None, v: torch.Tensor | None = None, *,
               slots: torch.Tensor | None = None, causal: bool = True, window: int = 0, sinks: int = 0,
               scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False,
               wait_limit_ns: int = 0):
        """Attention of each request's last tokens over its pages in ``layer``.

        ``q`` is ``(B, heads, D)`` for one new token per request or ``(B, T,
        heads, D)`` for its last ``T <= 32``, with ``heads`` a multiple of
        ``kv_heads``; row ``b`` is slot ``slots[b]`` (int32), or slot ``b``.
        ``k`` and ``v`` (``q``'s shape with ``kv_heads``) are stored in the
        tokens' pages by the same call (of rows with the same slot the first one's);
        without them the pages are only read.
        The tokens are part of ``kv_len`` already (``reserve``).  ``out``, if given,
        overlaps none of the inputs.

        Query ``i``, at position ``p = kv_len - T + i``, sees the tokens of its
        request, up to ``p`` if ``causal``, and with ``window > 0`` only those
        after ``p - window`` and the first ``sinks``.  ``scale`` is ``D ** -0.5``
        if not given.  A query that sees nothing gets zeros (and an ``lse`` of
        -inf).  Returns the output in ``q``'s shape and type, with
        ``return_lse`` also the ``(B, T, heads)`` or ``(B, heads)`` float32
        logarithms of the softmax's sums.  ``wait_limit_ns`` bounds each wait for
        a copy, as in ``select_step``.
        """
        key = (q.shape, q.stride(), q.dtype)
        if k is not None and v is not None:
            key += (k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype)
        elif k is not v:
            raise ValueError("k and v come together")
        plan = self._plans.get(key)
        if plan is None:
            plan = self._plan(key)
        a, B, copies, shape, o, out_like, lse_like = plan
        if q.get_device() != self._index or (k is not None and (k.get_device() != self._index or
                                                                v.get_device() != self._index)):
            raise TypeError(f"q, k and v must be on {self.device}")
        if not 0 <= layer < self._layers:
            raise ValueError(f"layer {layer} of {self._layers}")
        if not 0 <= sinks <= _MOST or not -_MOST <= window <= _MOST:
            raise ValueError("sinks must not be negative, and sinks and window fit 64 bits")
        if slots is not None:
            self._check_list("slots", slots, B)
        elif B > self.slots:
            raise ValueError(f"{B} requests, but {self.slots} slots")
        at = q.data_ptr()
        if copies or at % 16 or (k is not None and (k.data_ptr() % 16 or v.data_ptr() % 16)):
            # rows that the kernels cannot read: contiguous copies
            q = q.clone(memory_format=torch.contiguous_format)
            if k is not None:
                k, v = (t.clone(memory_format=torch.contiguous_format) for t in (k, v))
            return self.attend(layer, q, k, v, slots=slots, causal=causal, window=window, sinks=sinks, scale=scale,
                               out=out, return_lse=return_lse, wait_limit_ns=wait_limit_ns)
        if out is None:
            out = torch.empty_like(out_like)
        else:
            o = out.stride()
            if out.shape != shape or out.dtype != self._dtype or out.get_device() != self._index or \
                    out.data_ptr() % 16 or self._unreadable(o):
                raise ValueError(f"out must be a {tuple(shape)} {self._dtype} tensor on {self.device} whose rows are aligned")
        lse = torch.empty_like(lse_like) if return_lse else None
        with self._lock:
            a.q = at
            if k is not None:
                a.k, a.v = k.data_ptr(), v.data_ptr()
            a.slots = None if slots is None else slots.data_ptr()
            a.out = out.data_ptr()
            a.out_stride_req, a.out_stride_pos, a.out_stride_head = (o[0], 0, o[1]) if len(o) == 3 else o[:3]
            a.lse = lse.data_ptr() if return_lse else None
            a.layer, a.scale = layer, self._scale if scale is None else scale
            a.causal, a.window, a.sinks, a.wait_limit_ns = 1 if causal else 0, window, sinks, wait_limit_ns
            self._call(self._lib.yapd_attend, a)
        return (out, lse) if return_lse else out

    def _unreadable(self, strides) -> bool:
        """Whether the kernels cannot read rows with these strides."""
        return strides[-1] != 1 or any(s % self._vec for s in strides[:-1])

    def _plan(self, key):
        """The checks of an attention call's shapes, strides and types, and its
        arguments as far as they follow from them: kept, for the layers of a
        tick and the ticks of a batch are alike."""
        shape, stride, dtype = key[:3]
        if len(shape) not in (3, 4) or shape[-1] != self._dim or shape[-2] % self._heads or shape[-2] == 0:
            raise ValueError(f"q must be (B, [T,] heads, {self._dim}) with heads a multiple of {self._heads}, "
                             f"got {tuple(shape)}")
        B, T, H, D = shape if len(shape) == 4 else (shape[0], 1, *shape[1:])
        if not 1 <= T <= N.YAPD_MAX_NEW_TOKENS:
            raise ValueError(f"1 to {N.YAPD_MAX_NEW_TOKENS} new tokens, got {T}")
        if dtype != self._dtype:
            raise TypeError(f"q must be {self._dtype}, got {dtype}")
        a = N.AttendArgs()
        a.cache = self._cache
        a.B, a.new_tokens, a.heads = B, T, H
        three = lambda st: (st[0], 0, st[1]) if len(st) == 3 else st[:3]  # noqa: E731
        a.q_stride_req, a.q_stride_pos, a.q_stride_head = three(stride)
        copies = self._unreadable(stride)
        if len(key) > 3:
            want = (*shape[:-2], self._heads, D)
            if tuple(key[3]) != want or tuple(key[6]) != want:
                raise ValueError(f"k and v must be {want}, got {tuple(key[3])} and {tuple(key[6])}")
            if key[5] != self._dtype or key[8] != self._dtype:
                raise TypeError(f"k and v must be {self._dtype}")
            a.k_stride_req, a.k_stride_pos, a.k_stride_head = three(key[4])
            a.v_stride_req, a.v_stride_pos, a.v_stride_head = three(key[7])
            copies = copies or self._unreadable(key[4]) or self._unreadable(key[7])
        if len(self._plans) >= 64:
            self._plans.clear()
        # one element seen in the outputs' shapes: torch.empty_like costs half of torch.empty
        like = lambda dtype, shape: torch.empty(1, dtype=dtype, device=self.device).expand(shape)  # noqa: E731
        out_like, lse_like = like(self._dtype, shape), like(torch.float32, shape[:-1])
        self._plans[key] = plan = (a, B, copies, shape, torch.empty_like(out_like).stride(), out_like, lse_like)
        return plan

    # ----------------------------------------------------------------- pages

    def reserve(self, tokens, slots: torch.Tensor | None = None) -> torch.Tensor:
        """Room for ``tokens`` more (an int, or int64 ``(n,)``) in each slot of
        the list, in its order; ``kv_len`` grows.  A partly filled last page that
        other slots hold too is copied first.  Returns ``(n,)`` bool: the first
        slot that the pool has no room for, and all after it, are refused."""
        n, at = self._listed(slots)
        same, each = self._tokens(tokens, n)
        granted = torch.empty(n, dtype=torch.bool, device=self.device)
        p = self._pages
        with self._lock:
            p.n, p.slots, p.tokens, p.tokens_each, p.granted = n, at, same, each, granted.data_ptr()
            self._call(self._lib.yapd_pages_reserve, p)
        return granted

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """The empty slots ``dst`` become copies of ``src`` and share their pages
        (both int32 ``(n,)``; no slot is in both)."""
        n, at = self._listed(dst)
        self._check_list("src", src, n)
        p = self._pages
        with self._lock:
            p.n, p.slots, p.src = n, at, src.data_ptr()
            self._call(self._lib.yapd_pages_fork, p)

    def truncate(self, tokens, slots: torch.Tensor | None = None) -> None:
        """Takes the last ``tokens`` (an int, or int64 ``(n,)``) from each slot."""
        n, at = self._listed(slots)
        self._truncate(n, at, *self._tokens(tokens, n))

    def free(self, slots: torch.Tensor | None = None) -> None:
        """Empties the slots; pages that no other slot holds become free."""
        self._truncate(*self._listed(slots), -1, None)

    def trim(self, window: int, sinks: int = 0, slots: torch.Tensor | None = None) -> None:
        """Gives up the pages that attention with this ``window`` and ``sinks``
        no longer sees, from the slots' next token on."""
        if not 1 <= window <= _MOST or not 0 <= sinks <= _MOST:
            raise ValueError("window must be positive and sinks not negative, and both fit 64 bits")
        n, at = self._listed(slots)
        p = self._pages
        with self._lock:
            p.n, p.slots, p.window, p.sinks = n, at, window, sinks
            self._call(self._lib.yapd_pages_trim, p)

    def compact(self) -> torch.Tensor:
        """Moves the live pages to the pool's lowest numbers, in all layers and
        tables.  Returns their number, a ``(1,)`` int32 device tensor."""
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        p = self._pages
        with self._lock:
            p.n, p.live = 0, live.data_ptr()
            self._call(self._lib.yapd_pages_compact, p)
        return live

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copies pages ``src`` to ``dst`` (int32 ``(n,)``) in all layers; no page
        is both read and written, or written twice."""
        if dst.dim() != 1 or dst.shape[0] > self.kv.shape[1]:
            raise ValueError("dst must be (n,) with n at most the number of pages")
        self._check_list("dst", dst, dst.shape[0])
        self._check_list("src", src, dst.shape[0])
        p = self._pages
        with self._lock:
            p.n, p.src, p.dst = dst.shape[0], src.data_ptr(), dst.data_ptr()
            self._call(self._lib.yapd_pages_copy, p)

    # ---------------------------------------------------------------- status

    def status(self) -> int:
        """The status word (``YAPD_STATUS_*`` bits; synchronises the stream)."""
        word = C.c_uint32(0)
        N.check(self._lib.yapd_read_status(C.c_void_p(self._workspace.data_ptr()), self._stream(), C.byref(word)))
        return word.value

    def clear_status(self) -> None:
        N.check(self._lib.yapd_clear_status(C.c_void_p(self._workspace.data_ptr()), self._stream()))

    # --------------------------------------------------------------- private

    def _stream(self) -> int:
        return torch._C._cuda_getCurrentRawStream(self._index)

    def _call(self, entry, args) -> None:
        if torch.cuda.current_device() == self._index:
            rc = entry(args, self._stream())
        else:
            with torch.cuda.device(self.device):
                rc = entry(args, self._stream())
        if rc:
            N.check(rc)

    def _truncate(self, n, at, same, each) -> None:
        p = self._pages
        with self._lock:
            p.n, p.slots, p.tokens, p.tokens_each = n, at, same, each
            self._call(self._lib.yapd_pages_truncate, p)

    def _check_list(self, name: str, t: torch.Tensor, n: int) -> None:
        if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or t.get_device() != self._index or \
                (n > 1 and t.stride(0) != 1):
            raise ValueError(f"{name} must be a contiguous int32 ({n},) tensor on {self.device}")

    def _listed(self, slots: torch.Tensor | None):
        """Length and address of a list of slots (none: all of them)."""
        if slots is None:
            return self.slots, None
        if slots.dim() != 1 or slots.shape[0] > self.slots:
            raise ValueError(f"slots must be (n,) with n <= {self.slots}")
        self._check_list("slots", slots, slots.shape[0])
        return slots.shape[0], slots.data_ptr()

    def _tokens(self, tokens, n: int):
        """A number for all of the list, or the address of one for each."""
        if isinstance(tokens, torch.Tensor):
            if tokens.dtype != torch.int64 or tuple(tokens.shape) != (n,) or tokens.device != self.device or \
                    not tokens.is_contiguous():
                raise ValueError(f"tokens must be an int or a contiguous int64 ({n},) tensor on {self.device}")
            return 0, tokens.data_ptr()
        tokens = int(tokens)
        if not 0 <= tokens <= _MOST:
            raise ValueError(f"tokens must not be negative, and fit 64 bits, got {tokens}")
        return tokens, None
