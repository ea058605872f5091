"""Rotary positions with several axes for q and k, forward and backward.

An additional operator with no counterpart in the reference, whose entry point takes q and k
already rotated (flash_attention_gpt_oss.py:437-438).  Frequency ``i`` of ``inv_freq`` turns one
pair of each head's values by ``positions[axis(i)] * inv_freq[i]``: the pair ``(i, n + i)``, or
``(2 i, 2 i + 1)`` when interleaved; values from ``2 n`` on stay as they are.  Text has one axis;
images and video have a position in time, height and width.  The compute is the C-ABI library's
``swa_rotary``.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _lib
from .flash_attention_gpt_oss import _DTYPES


class Rotary:
    """A model's rotation: its inverse frequencies and the axis that each one goes by.

    ``inv_freq``: ``[n]`` CUDA tensor, ``n <= 64`` (kept as fp32, copied).  ``sections``: how many
    consecutive frequencies each axis takes (``(n,)`` when omitted); or ``axes``: the axis of
    every frequency, in any order.  ``scale`` multiplies every rotated value (the length scaling
    of some rotary schemes)."""

    def __init__(self, inv_freq: torch.Tensor, sections: Optional[Sequence[int]] = None,
                 axes: Optional[Sequence[int]] = None, interleaved: bool = False,
                 scale: float = 1.0):
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1:
            raise ValueError("inv_freq must be a 1-D tensor")
        n = inv_freq.numel()
        if n > _lib.SWA_ROTARY_MAX_FREQS:
            raise ValueError(f"at most {_lib.SWA_ROTARY_MAX_FREQS} frequencies; got {n}")
        if not inv_freq.is_cuda:
            raise ValueError("inv_freq must be on a CUDA device")
        if axes is None:
            sections = (n,) if sections is None else tuple(int(x) for x in sections)
            if not sections or any(x < 0 for x in sections) or sum(sections) != n:
                raise ValueError(f"sections must be whole numbers that add up to {n}; got {sections}")
            axes = [a for a, x in enumerate(sections) for _ in range(x)]
            n_axes = len(sections)
        else:
            if sections is not None:
                raise ValueError("give sections or axes, not both")
            axes = [int(a) for a in axes]
            if len(axes) != n or any(a < 0 or a > 255 for a in axes):
                raise ValueError(f"axes must give {n} frequencies an axis each (0 .. 255)")
            n_axes = max(axes, default=0) + 1
        if n_axes > 256:
            raise ValueError("at most 256 axes")
        if not float(scale) == float(scale):
            raise ValueError("scale is NaN")
        self._inv_freq = inv_freq.detach().to(torch.float32, copy=True).contiguous()
        self._c = _lib.SwaRotary(self._inv_freq.data_ptr(), None, 0, 0, 0, 0, n_axes, n,
                                 int(bool(interleaved)), float(scale))
        self._c.axis[:n] = axes
        self._dev = self._inv_freq.device
        self._calls = _lib.Calls()

    inv_freq = property(lambda self: self._inv_freq)
    n_axes = property(lambda self: self._c.n_axes)
    dim = property(lambda self: 2 * self._c.n_freq, doc="values of a head that turn")
    interleaved = property(lambda self: bool(self._c.interleaved))
    scale = property(lambda self: self._c.scale)

    def _bind(self, positions: torch.Tensor, batch: Optional[int], length: int) -> _lib.SwaRotary:
        """The C block for positions of this form (their address is left out): ``[L]``, ``[B, L]``
        or ``[A, ..., L]``; ``batch`` None: packed tokens."""
        if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be an int32 or int64 tensor")
        shape, st = tuple(positions.shape), positions.stride()
        axis = self.n_axes > 1 or len(shape) == (2 if batch is None else 3)
        rest, rst = (shape[1:], st[1:]) if axis else (shape, st)
        ok = not axis or shape[:1] == (self.n_axes,)
        sb = 0
        if batch is not None and len(rest) == 2:
            ok, sb, rest, rst = ok and rest[0] == batch, rst[0], rest[1:], rst[1:]
        if not ok or rest != (length,):
            raise ValueError(f"positions {shape} do not fit {self.n_axes} axes and "
                             + (f"[{batch}, {length}] tokens" if batch is not None else f"{length} tokens"))
        c = _lib.SwaRotary.from_buffer_copy(self._c)
        c.pos_stride_axis = st[0] if axis else 0
        c.pos_stride_b, c.pos_stride_l = sb, rst[0]
        c.pos_is_64 = int(positions.dtype == torch.int64)
        return c

    def _on(self, dev: torch.device, positions: torch.Tensor):
        if positions.device != dev or self._dev != dev:
            raise ValueError("positions and inv_freq must be on the device of q")


def _as4(t: torch.Tensor) -> torch.Tensor:
    """[1, H, T, D] view of packed [T, H, D] tokens."""
    return t.transpose(0, 1).unsqueeze(0) if t.dim() == 3 else t


def _tensor(t: torch.Tensor) -> _lib.SwaTensor:
    return _lib.SwaTensor(None, *t.stride()[:3])


def _empty(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _validate(q, k, rotary):
    for name, t in (("q", q), ("k", k)):
        if t is None:
            continue
        if t.dim() not in (3, 4) or t.dim() != q.dim():
            raise ValueError("q and k must both be [B, H, L, D] or both be packed [T, H, D]")
        if t.dtype not in _DTYPES or t.dtype != q.dtype:
            raise TypeError(f"q and k must share one dtype in (float16, bfloat16); got {name}: {t.dtype}")
    if _as4(q).shape[1] == 0:
        raise ValueError("q has no heads")
    d = q.shape[-1]
    if d > 128 or d % 2 or d < rotary.dim:
        raise ValueError(f"head dimension {d} must be even, at most 128 and at least {rotary.dim}")
    if k is not None:
        a, b = (q.shape, k.shape) if q.dim() == 3 else (q.transpose(1, 2).shape, k.transpose(1, 2).shape)
        if a[:-2] != b[:-2] or a[-1] != b[-1]:
            raise ValueError("q and k must have the same tokens and head dimension")


def _block(q, k, positions, rotary, inverse) -> _lib.SwaRotaryArgs:
    """The argument block of a call of this form, without addresses."""
    _validate(q, k, rotary)
    packed = q.dim() == 3
    b, hq, l, d = _as4(q).shape
    none = _lib.SwaTensor(None, 0, 0, 0)
    dense = lambda t: _tensor(_as4(torch.empty(t.shape, device="meta")))  # noqa: E731
    return _lib.SwaRotaryArgs(b, hq, 0 if k is None else _as4(k).shape[1], l, d, _DTYPES[q.dtype], int(inverse),
                              rotary._bind(positions, None if packed else b, l), _tensor(_as4(q)),
                              none if k is None else _tensor(_as4(k)), dense(q), none if k is None else dense(k))


def rotate(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: Rotary,
           inverse: bool = False):
    """``(q', k')`` as new tensors (``k`` and ``k'`` may be None); ``inverse`` turns back, which
    is the gradient of the inputs from the gradient of the outputs.  No autograd."""
    if not isinstance(rotary, Rotary):
        raise TypeError("rotary must be a Rotary")
    if q.stride(-1) != 1:
        q = q.contiguous()
    if k is not None and k.stride(-1) != 1:
        k = k.contiguous()
    key = (q.shape, q.stride(), q.dtype, None if k is None else (k.shape, k.stride(), k.dtype), positions.shape,
           positions.stride(), positions.dtype, inverse)
    block = rotary._calls.get(key)
    if block is None:
        block = rotary._calls.put(key, _block(q, k, positions, rotary, inverse))
    dev = q.device
    if not q.is_cuda or (k is not None and k.device != dev):
        raise ValueError("q and k must be on the same CUDA device")
    rotary._on(dev, positions)
    args = _lib.SwaRotaryArgs.from_buffer_copy(block)
    qo = _empty(q)
    args.q.ptr, args.q_out.ptr, args.r.positions = q.data_ptr(), qo.data_ptr(), positions.data_ptr()
    ko = None
    if k is not None:
        ko = _empty(k)
        args.k.ptr, args.k_out.ptr = k.data_ptr(), ko.data_ptr()
    _lib.call("swa_rotary", args, dev)
    return qo, ko


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, rotary, inverse):
        ctx.save_for_backward(positions)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(positions)
        ctx.rotary, ctx.inverse, ctx.dtype = rotary, inverse, q.dtype
        return rotate(q, k, positions, rotary, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        # only the gradients that are asked for: a frozen q or k costs nothing
        need = ctx.needs_input_grad
        dq = dq.to(ctx.dtype) if need[0] else None
        dk = dk.to(ctx.dtype) if need[1] else None
        return *_turn_given(dq, dk, positions, ctx.rotary, not ctx.inverse), None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        (positions,) = ctx.saved_tensors
        return _turn_given(tq, tk, positions, ctx.rotary, ctx.inverse)


def _turn(q, k, positions, rotary, inverse):
    """Rotate, differentiably (in both modes) where a derivative is asked for."""
    if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))) or _dual(q, k):
        return _Rotate.apply(q, k, positions, rotary, inverse)
    return rotate(q, k, positions, rotary, inverse)


def _dual(q, k):
    """Whether one of them carries a tangent (no level open, no tangent: unpacking costs 0.5 us)."""
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (q, k))


def _turn_given(q, k, positions, rotary, inverse):
    """_turn of what is not None of q and k."""
    if q is not None:
        return _turn(q, k, positions, rotary, inverse)
    return None, None if k is None else _turn(k, None, positions, rotary, inverse)[0]


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 rotary: Rotary):
    """Rotate q and k (``k`` may be None) by their tokens' positions; differentiable in reverse and
    in forward mode.

    q ``[B, Hq, L, D]`` and k ``[B, Hkv, L, D]``, or packed ``[T, H, D]`` (fp16 or bf16, any
    strides); D even, at most 128.  ``positions`` (int32 or int64): ``[L]`` or ``[B, L]`` (packed:
    ``[T]``) for one axis, with a leading dimension of ``rotary.n_axes`` for several.  Angles
    are formed in 64 bits, so far positions lose nothing."""
    return _turn(q, k, positions, rotary, False)
