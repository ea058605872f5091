"""Serving: a paged key-value cache, the attention of one new token over it, and its eviction.

Additional operators with no counterpart in the reference, which trains only: they serve what the
training path has trained, with the same mask (window, sink tokens, learned sink logits) and
grouped heads.  Keys and values lie in pages of one pool, ``[n_pages, Hkv, page_size, D]``; slot
``j`` of sequence ``b`` is row ``j % page_size`` of page ``page_table[b, j // page_size]``, and
``seq_lens[b]`` slots are in use.  One step of a layer:

    cache.advance()                                         # every sequence gets one token
    q = cache.append(k, v, q=q, positions=pos, rotary=rot)  # rotate q and k, write k and v
    o = cache.decode(q, window_size=128, sink_size=4, sinks=logits)

With ``weights`` and ``positions`` the cache also tracks how much attention each slot has had
(``decode(..., weights_out=cache.weights)``), and ``evict`` cuts sequences down to a budget by it.
All calls are asynchronous on the current stream and can be captured into a CUDA graph; none is
differentiable.  The compute is the C-ABI library's ``swa_paged_append`` / ``swa_paged_decode`` / ``swa_paged_evict``.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from .flash_attention_gpt_oss import _DTYPES, _KERNEL_HEAD_DIMS
from .rotary import Rotary, _empty

_WHOLE = 2**31 - 1


def _rows_ok(t: torch.Tensor) -> bool:
    """Rows of 16-byte aligned, contiguous values."""
    *outer, inner = t.stride()
    bits = t.data_ptr() // 2
    for s in outer:
        bits |= s
    return inner == 1 and bits % 8 == 0


def _packed(t: torch.Tensor) -> _lib.SwaPackedTensor:
    return _lib.SwaPackedTensor(None, *t.stride()[:2])


def _form(t: Optional[torch.Tensor]):
    """All of a tensor but its address and device."""
    return None if t is None else (t.shape, t.stride(), t.dtype)


class PagedKVCache:
    """The cache of one attention layer.

    ``k_pages``, ``v_pages``: ``[n_pages, Hkv, page_size, D]``, fp16 or bf16, D 16, 32, 64 or 128,
    page_size a multiple of 16, the last dimension contiguous, the others with any strides of
    whole 16 bytes.  ``page_table``: int32 ``[B, max_pages]``, ``seq_lens``: int32 ``[B]``; entries
    behind a sequence's last page are not read.  For eviction also ``weights`` (fp32) and
    ``positions`` (int32), ``[B, Hkv, max_pages * page_size]``: the attention that each slot has
    had and the number of its token; and ``seen`` (int32 ``[B]``): tokens so far, which evictions
    leave as it is.  Without ``seen``, ``seq_lens`` counts the tokens: that holds until the first
    eviction shortens it, so such a cache is evicted once and refuses a second time.  Caches that
    are evicted do not share ``seq_lens``: the first one's eviction would cut the others unselected.

    The tensors are the caller's: their values may change between calls (also under a captured
    graph), the cache itself holds only their addresses.  A page number outside the pool or a
    length beyond the table is not followed: that sequence's output is NaN, its rows of
    ``weights_out`` stay, an eviction leaves it as it is, an append writes only tokens whose own
    page is in range, and :meth:`check` raises."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, weights: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, seen: Optional[torch.Tensor] = None):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
            raise ValueError("k_pages and v_pages must both be [n_pages, Hkv, page_size, D]")
        if k_pages.dtype not in _DTYPES or v_pages.dtype != k_pages.dtype:
            raise TypeError(f"pages must share one dtype in (float16, bfloat16); got {k_pages.dtype}, "
                            f"{v_pages.dtype}")
        n, hkv, page, d = k_pages.shape
        if d not in _KERNEL_HEAD_DIMS:
            raise ValueError(f"a cache's head dimension must be one of {_KERNEL_HEAD_DIMS}; got {d}")
        if page <= 0 or page % 16:
            raise ValueError(f"page_size must be a multiple of 16; got {page}")
        if hkv <= 0:
            raise ValueError("a cache needs a KV head")
        if page_table.dim() != 2 or seq_lens.dim() != 1 or page_table.shape[0] != seq_lens.shape[0]:
            raise ValueError("page_table must be [B, max_pages] and seq_lens [B]")
        b, m = page_table.shape
        if m * page > _WHOLE - 1024:
            raise ValueError("a sequence can hold at most 2^31 - 1025 slots")
        for name, t, dtype in (("page_table", page_table, torch.int32), ("seq_lens", seq_lens, torch.int32),
                               ("weights", weights, torch.float32), ("positions", positions, torch.int32),
                               ("seen", seen, torch.int32)):
            if t is not None and t.dtype != dtype:
                raise TypeError(f"{name} must be {dtype}; got {t.dtype}")
        if not k_pages.is_cuda or any(t is not None and t.device != k_pages.device for t in
                                      (v_pages, page_table, seq_lens, weights, positions, seen)):
            raise ValueError("a cache's tensors must be on the same CUDA device")
        if not (_rows_ok(k_pages) and _rows_ok(v_pages)):
            raise ValueError("rows of pages must be contiguous and 16-byte aligned, strides multiples of 8")
        for name, t in (("weights", weights), ("positions", positions)):
            if t is not None and (t.shape != (b, hkv, m * page) or (t.numel() and t.stride(-1) != 1)):
                raise ValueError(f"{name} must be [{b}, {hkv}, {m * page}] with the last dimension contiguous")
        if m > 1 and page_table.stride(1) != 1:
            raise ValueError("rows of page_table must be contiguous")
        for name, t in (("seq_lens", seq_lens), ("seen", seen)):
            if t is not None and (t.shape != (b,) or (b > 1 and t.stride(0) != 1)):
                raise ValueError(f"{name} must be [{b}], contiguous")
        if b and seen is not None and seen.data_ptr() == seq_lens.data_ptr():
            raise ValueError("seen must not be seq_lens itself, which evictions shorten")
        self._t = (k_pages, v_pages, page_table, seq_lens, weights, positions, seen)
        self._dev, self._dtype = k_pages.device, k_pages.dtype
        self._b, self._hkv, self._d, self._cap = b, hkv, d, m * page
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        st = lambda t: (0, 0) if t is None else t.stride()[:2]  # noqa: E731
        self._c = _lib.SwaPagedKV(ptr(k_pages), ptr(v_pages), *k_pages.stride()[:3], *v_pages.stride()[:3],
                                  ptr(page_table), page_table.stride(0), ptr(seq_lens), ptr(seen), ptr(weights),
                                  ptr(positions), *st(weights), *st(positions), n, page, m, b, hkv, d,
                                  _DTYPES[k_pages.dtype])
        self._calls = _lib.Calls()
        self._cut = False  # evicted before

    @classmethod
    def allocate(cls, batch: int, n_kv_heads: int, head_dim: int, max_len: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", track: bool = False) -> "PagedKVCache":
        """An empty cache in which every sequence has pages of its own for ``max_len`` slots;
        ``track`` adds weights, positions and seen for eviction."""
        dev = torch.device(device)
        m = -(-max_len // page_size)
        pages = torch.zeros((2, max(1, batch * m), n_kv_heads, page_size, head_dim), dtype=dtype, device=dev)
        table = torch.arange(batch * m, dtype=torch.int32, device=dev).view(batch, m)
        lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        if not track:
            return cls(pages[0], pages[1], table, lens)
        shape = (batch, n_kv_heads, m * page_size)
        return cls(pages[0], pages[1], table, lens, weights=torch.zeros(shape, device=dev),
                   positions=torch.zeros(shape, dtype=torch.int32, device=dev), seen=torch.zeros_like(lens))

    k_pages = property(lambda self: self._t[0])
    v_pages = property(lambda self: self._t[1])
    page_table = property(lambda self: self._t[2])
    seq_lens = property(lambda self: self._t[3])
    weights = property(lambda self: self._t[4])
    positions = property(lambda self: self._t[5])
    seen = property(lambda self: self._t[6])

    def advance(self, n=1):
        """Count ``n`` new tokens of every sequence (a number, or int32 ``[B]``) before their append."""
        self.seq_lens.add_(n)
        if self.seen is not None:
            self.seen.add_(n)

    def check(self):
        """Wait for the current stream, and raise if a call met a page number or a length out of range.

        The flag is the device's, not the cache's: it tells of any cache's calls since the last check
        (or ``swa_check_device``), which clears it, on other streams as far as they have got."""
        with torch.cuda.device(self._dev):
            _lib.check(_lib.lib().swa_check_device(torch.cuda.current_stream().cuda_stream), "PagedKVCache")

    def _tokens(self, name, t, heads=None):
        if t.dim() != 3 or t.shape[-1] != self._d or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {self._d}]; "
                             f"got {tuple(t.shape)}")
        if t.dtype != self._dtype:
            raise TypeError(f"{name} must be {self._dtype} like the pages; got {t.dtype}")

    def _here(self, *tensors):
        for t in tensors:
            if t is not None and t.device != self._dev:
                raise ValueError("all tensors of a call must be on the device of the pages")

    def append(self, k: torch.Tensor, v: torch.Tensor, cu_new: Optional[torch.Tensor] = None,
               q: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
               rotary: Optional[Rotary] = None) -> Optional[torch.Tensor]:
        """Write new tokens, ``k``, ``v`` ``[T, Hkv, D]``, behind their sequences.

        ``seq_lens`` (and ``seen``) already count them (:meth:`advance`).  ``cu_new``: int32
        ``[B + 1]`` CUDA offsets of each sequence's tokens; omitted, every sequence has T / B.  A token
        before the first offset or behind the last is no sequence's: it is written to no page, and
        :meth:`check` raises.
        With ``rotary`` and ``positions`` (``[T]``, or ``[axes, T]``), k is rotated on the way, and
        so is ``q`` ``[T, Hq, D]``, which is returned."""
        k = k if k.stride(-1) == 1 else k.contiguous()
        v = v if v.stride(-1) == 1 else v.contiguous()
        if q is not None and q.stride(-1) != 1:
            q = q.contiguous()
        key = ("append", rotary, _form(k), _form(v), _form(q), _form(positions), _form(cu_new))
        block = self._calls.get(key)
        if block is None:
            block = self._calls.put(key, self._append_block(k, v, cu_new, q, positions, rotary))
        self._here(k, v, cu_new, q, positions)
        args = _lib.SwaPagedAppendArgs.from_buffer_copy(block)
        args.k.ptr, args.v.ptr = k.data_ptr(), v.data_ptr()
        if cu_new is not None:
            args.cu_new = cu_new.data_ptr()
        out = None
        if rotary is not None:
            rotary._on(self._dev, positions)
            args.r.positions = positions.data_ptr()
            if q is not None:
                out = _empty(q)
                args.q.ptr, args.q_out.ptr = q.data_ptr(), out.data_ptr()
        _lib.call("swa_paged_append", args, self._dev)
        return out

    def _append_block(self, k, v, cu_new, q, positions, rotary) -> _lib.SwaPagedAppendArgs:
        """The argument block of an append of this form, without addresses."""
        self._tokens("k", k, self._hkv)
        self._tokens("v", v, self._hkv)
        t = k.shape[0]
        if v.shape[0] != t:
            raise ValueError("k and v must have the same tokens")
        if (rotary is None) != (positions is None) or (q is not None and rotary is None):
            raise ValueError("rotary and positions go together, and q is rotated with them")
        if cu_new is None:
            if t and (self._b == 0 or t % self._b):
                raise ValueError(f"{t} tokens cannot be dealt out evenly to {self._b} sequences: give cu_new")
        elif cu_new.dtype != torch.int32 or cu_new.shape != (self._b + 1,) or (self._b and cu_new.stride(0) != 1):
            raise ValueError(f"cu_new must be a contiguous int32 [{self._b + 1}] tensor")
        none = _lib.SwaPackedTensor(None, 0, 0)
        args = _lib.SwaPagedAppendArgs(self._c, None, t, 0, _packed(k), _packed(v), none, none, 0)
        if rotary is not None:
            if not isinstance(rotary, Rotary):
                raise TypeError("rotary must be a Rotary")
            if rotary.dim > self._d:
                raise ValueError(f"rotary turns {rotary.dim} values of a head of {self._d}")
            args.use_rotary, args.r = 1, rotary._bind(positions, None, t)
            if q is not None:
                self._tokens("q", q)
                if q.shape[0] != t:
                    raise ValueError("q and k must have the same tokens")
                args.n_q_heads, args.q = q.shape[1], _packed(q)
                args.q_out = _lib.SwaPackedTensor(None, q.shape[1] * self._d, self._d)
        return args

    def decode(self, q: torch.Tensor, window_size: Optional[int] = None, sink_size: int = 0,
               softmax_scale: Optional[float] = None, sinks: Optional[torch.Tensor] = None,
               weights_out: Optional[torch.Tensor] = None, decay: float = 1.0, return_lse: bool = False):
        """Attention of one new token per sequence, ``q`` ``[B, Hq, D]``, over its slots: ``o`` like q.

        The newest token (slot ``n - 1`` of ``n``) sees slot ``j`` iff ``n - 1 - j < window_size`` or
        ``j < sink_size`` (``window_size`` None: all); ``sinks``: learned sink logits ``[Hq]``.  A row
        that sees no key gives 0.  ``weights_out``: gets ``decay * cache.weights`` plus the softmax
        weights of this token, summed over the query heads of each KV head, in the slots in use
        (``cache.weights`` itself to accumulate in place; without cache.weights only the new ones).
        It takes a workspace of 32 bytes (more than 8 query heads a KV head: 64 for each 16 of them) a
        slot that the mask can reach and KV head.
        ``return_lse``: also the base-2 log-sum-exp ``[B, Hq]``."""
        # numbers as numbers: a tensor's value could change under its key
        if window_size is not None:
            window_size = int(window_size)
        if softmax_scale is not None:
            softmax_scale = float(softmax_scale)
        sink_size, decay = int(sink_size), float(decay)
        key = ("decode", q.shape, q.stride(), q.dtype, window_size, sink_size, softmax_scale, decay, _form(sinks),
               _form(weights_out))
        block = self._calls.get(key)
        if block is None or q.data_ptr() % 16:
            self._tokens("q", q)  # rows of another width may never be aligned
            if not _rows_ok(q):
                q = q.clone(memory_format=torch.contiguous_format)
                return self.decode(q, window_size, sink_size, softmax_scale, sinks, weights_out, decay, return_lse)
            block = self._calls.put(key, self._decode_block(q, window_size, sink_size, softmax_scale, sinks, weights_out, decay))
        dev = self._dev
        self._here(q, sinks, weights_out)
        block, ws_bytes, sinks_ok = block
        args = _lib.SwaPagedDecodeArgs.from_buffer_copy(block)
        o = _empty(q)
        args.q.ptr, args.o.ptr = q.data_ptr(), o.data_ptr()
        lse = None
        if return_lse:
            lse = torch.empty(q.shape[:2], device=dev, dtype=torch.float32)
            args.lse = lse.data_ptr()
        if sinks is not None:
            sinks = sinks if sinks_ok else sinks.detach().to(torch.float32).contiguous()
            args.sink_logits = sinks.data_ptr()
        if weights_out is not None:
            args.weights_out = weights_out.data_ptr()
        if ws_bytes:
            ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
            args.workspace, args.workspace_bytes = ws.data_ptr(), ws_bytes
        _lib.call("swa_paged_decode", args, dev)
        return (o, lse) if return_lse else o

    def _decode_block(self, q, window_size, sink_size, softmax_scale, sinks, weights_out, decay):
        """The argument block of an attention of this form (q's has been looked at), without addresses; the
        bytes of its workspace; whether the sink logits can be read as they are."""
        hq = q.shape[1]
        if q.shape[0] != self._b:
            raise ValueError(f"q must hold one token for each of {self._b} sequences; got {q.shape[0]}")
        if hq <= 0 or hq % self._hkv:
            raise ValueError("Number of query heads must be divisible by number of K/V heads")
        if sink_size < 0:
            raise ValueError("sink_size must not be negative")
        window = _WHOLE if window_size is None else max(-1, min(window_size, _WHOLE))
        scale = 1.0 / math.sqrt(self._d) if softmax_scale is None else softmax_scale
        args = _lib.SwaPagedDecodeArgs(self._c, hq, window, min(sink_size, _WHOLE), scale, _packed(q),
                                       _lib.SwaPackedTensor(None, hq * self._d, self._d))
        args.decay = decay
        if sinks is not None and (sinks.dim() != 1 or sinks.numel() != hq):
            raise ValueError(f"sinks must be [{hq}] logits")
        if weights_out is not None:
            if weights_out.shape != (self._b, self._hkv, self._cap) or weights_out.dtype != torch.float32 or \
                    (weights_out.numel() and weights_out.stride(-1) != 1):
                raise ValueError(f"weights_out must be an fp32 [{self._b}, {self._hkv}, {self._cap}] tensor "
                                 "with the last dimension contiguous")
            args.weights_out = 256  # it counts for the workspace
            args.wo_stride_b, args.wo_stride_h = weights_out.stride()[:2]
        return (args, _lib.lib().swa_paged_decode_workspace_size(ctypes.byref(args)),
                sinks is not None and sinks.dtype == torch.float32 and sinks.is_contiguous())

    def evict(self, keep: int, sink_size: int = 0, recent: int = 0, trigger: Optional[int] = None):
        """Cut sequences of more than ``max(trigger, keep)`` slots down to ``keep``.

        Each KV head keeps its tokens numbered below ``sink_size`` and its last ``recent`` ones, then
        those of the largest ``weights`` (ties: the lowest slot).  Kept slots below ``keep`` stay
        where they are, and the others, in order, fill the places that came free, so the order of
        slots is no longer that of tokens: attend with ``window_size=None`` afterwards.
        ``seq_lens`` becomes ``keep``.  Pages of a sequence that is cut must be its own.  More than one
        eviction, or a captured one, needs a cache with ``seen``.  Weights are what ``decode`` has
        added: those of a prompt are 0 after its append, which leaves its lowest slots."""
        keep, sink_size, recent = int(keep), int(sink_size), int(recent)
        trigger = keep if trigger is None else int(trigger)
        key = ("evict", keep, sink_size, recent, trigger)
        block = self._calls.get(key)
        if block is None:
            block = self._calls.put(key, self._evict_block(keep, sink_size, recent, trigger))
        block, ws_bytes = block
        if block is None:
            return
        args = _lib.SwaPagedEvictArgs.from_buffer_copy(block)
        if self._t[6] is None:
            with torch.cuda.device(self._dev):
                if self._cut or torch.cuda.is_current_stream_capturing():
                    raise ValueError("a cache without seen can be evicted once: seq_lens no longer counts its tokens")
                seen = self.seq_lens.clone()
            args.cache.seen = seen.data_ptr()
        ws = torch.empty(ws_bytes, device=self._dev, dtype=torch.uint8)
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws_bytes
        _lib.call("swa_paged_evict", args, self._dev)
        self._cut = True

    def _evict_block(self, keep, sink_size, recent, trigger):
        """The argument block of an eviction (None: no sequence can be that long) and the bytes of
        its workspace."""
        if self.weights is None or self.positions is None:
            raise ValueError("eviction needs a cache with weights and positions")
        if keep <= 0 or trigger < 0 or sink_size < 0 or recent < 0 or sink_size + recent > keep:
            raise ValueError("keep must be positive and hold sink_size + recent tokens")
        if keep >= self._cap or self._b == 0:
            return None, 0
        args = _lib.SwaPagedEvictArgs(self._c, keep, min(trigger, _WHOLE), sink_size, recent)
        return args, _lib.lib().swa_paged_evict_workspace_size(ctypes.byref(args))
