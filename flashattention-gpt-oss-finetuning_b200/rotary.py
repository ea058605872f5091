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

from . import _lib
from .flash_attention_gpt_oss import _DTYPES, _stream


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
        self.inv_freq = inv_freq.detach().to(torch.float32, copy=True).contiguous()
        self.n_axes = n_axes
        self.dim = 2 * n
        self.interleaved = bool(interleaved)
        self.scale = float(scale)
        self._c = _lib.SwaRotary(self.inv_freq.data_ptr(), None, 0, 0, 0, 0, n_axes, n,
                                 int(self.interleaved), self.scale)
        self._c.axis[:n] = axes

    def _bind(self, positions: torch.Tensor, dev: torch.device, batch: Optional[int], length: int) -> _lib.SwaRotary:
        """The C block for these positions: ``[L]``, ``[B, L]`` or ``[A, ..., L]``; ``batch`` None:
        packed tokens."""
        if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be an int32 or int64 tensor")
        if positions.device != dev or self.inv_freq.device != dev:
            raise ValueError("positions and inv_freq must be on the device of q")
        shape, st = tuple(positions.shape), positions.stride()
        axis = self.n_axes > 1 or len(shape) == (2 if batch is None else 3)
        want = ((self.n_axes,) if axis else ())
        rest, rst = (shape[1:], st[1:]) if axis else (shape, st)
        ok = bool(shape) and shape[:len(want)] == want
        if batch is not None and len(rest) == 2:
            ok, sb, rest, rst = ok and rest[0] == batch, rst[0], rest[1:], rst[1:]
        else:
            sb = 0
        if not ok or rest != (length,):
            raise ValueError(f"positions {shape} do not fit {self.n_axes} axes and "
                             + (f"[{batch}, {length}] tokens" if batch is not None else f"{length} tokens"))
        c = _lib.SwaRotary.from_buffer_copy(self._c)
        c.positions = positions.data_ptr()
        c.pos_stride_axis = st[0] if axis else 0
        c.pos_stride_b, c.pos_stride_l = sb, rst[0]
        c.pos_is_64 = int(positions.dtype == torch.int64)
        return c


def _as4(t: torch.Tensor) -> torch.Tensor:
    """[1, H, T, D] view of packed [T, H, D] tokens."""
    return t.transpose(0, 1).unsqueeze(0) if t.dim() == 3 else t


def _tensor(t: torch.Tensor) -> _lib.SwaTensor:
    s = t.stride()
    return _lib.SwaTensor(t.data_ptr(), s[0], s[1], s[2])


def _validate(q, k, rotary):
    if not isinstance(rotary, Rotary):
        raise TypeError("rotary must be a Rotary")
    for name, t in (("q", q), ("k", k)):
        if t is None:
            continue
        if t.dim() not in (3, 4) or t.dim() != q.dim():
            raise ValueError("q and k must both be [B, H, L, D] or both be packed [T, H, D]")
        if t.dtype not in _DTYPES or t.dtype != q.dtype:
            raise TypeError(f"q and k must share one dtype in (float16, bfloat16); got {name}: {t.dtype}")
        if not t.is_cuda or t.device != q.device:
            raise ValueError("q and k must be on the same CUDA device")
    d = q.shape[-1]
    if d > 128 or d % 2 or d < rotary.dim:
        raise ValueError(f"head dimension {d} must be even, at most 128 and at least {rotary.dim}")
    if k is not None:
        a, b = (q.shape, k.shape) if q.dim() == 3 else (q.transpose(1, 2).shape, k.transpose(1, 2).shape)
        if a[:-2] != b[:-2] or a[-1] != b[-1]:
            raise ValueError("q and k must have the same tokens and head dimension")


def rotate(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: Rotary,
           inverse: bool = False):
    """``(q', k')`` as new tensors (``k`` and ``k'`` may be None); ``inverse`` turns back, which
    is the gradient of the inputs from the gradient of the outputs.  No autograd."""
    _validate(q, k, rotary)
    packed = q.dim() == 3
    q4 = _as4(q if q.stride(-1) == 1 else q.contiguous())
    b, hq, l, d = q4.shape
    r = rotary._bind(positions, q.device, None if packed else b, l)
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    none = _lib.SwaTensor(None, 0, 0, 0)
    ko, kt, kot, hkv = None, none, none, 0
    if k is not None:
        k4 = _as4(k if k.stride(-1) == 1 else k.contiguous())
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
        kt, kot, hkv = _tensor(k4), _tensor(_as4(ko)), k4.shape[1]
    if hq:
        args = _lib.SwaRotaryArgs(b, hq, hkv, l, d, _DTYPES[q.dtype], int(inverse), r, _tensor(q4), kt,
                                  _tensor(_as4(qo)), kot)
        with _lib.on_device(q.device):
            _lib.check(_lib.lib().swa_rotary(ctypes.byref(args), _stream(q.device)), "swa_rotary")
    return qo, ko


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, rotary, inverse):
        ctx.save_for_backward(positions)
        ctx.rotary, ctx.inverse, ctx.dtype = rotary, inverse, q.dtype
        return rotate(q, k, positions, rotary, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        dq = dq.to(ctx.dtype)
        dk = None if dk is None else dk.to(ctx.dtype)
        dq, dk = _Rotate.apply(dq, dk, positions, ctx.rotary, not ctx.inverse)
        return dq, dk, None, None, None


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 rotary: Rotary):
    """Rotate q and k (``k`` may be None) by their tokens' positions; differentiable.

    q ``[B, Hq, L, D]`` and k ``[B, Hkv, L, D]``, or packed ``[T, H, D]`` (fp16 or bf16, any
    strides); D even, at most 128.  ``positions`` (int32 or int64): ``[L]`` or ``[B, L]`` (packed:
    ``[T]``) for one axis, with a leading dimension of ``rotary.n_axes`` for several.  Angles
    are formed in 64 bits, so far positions lose nothing."""
    return _Rotate.apply(q, k, positions, rotary, False)
