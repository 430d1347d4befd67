"""Rotary positions with several axes on the HIP kernel ``fovi_rotary``.

A token's position has one coordinate per axis: (row, column) of its sensor point, with the
number of its fixation in front when the tokens of several fixations are read together. Each axis
turns its own section of the pairs of a head, ``angle = position[axis] * freqs[pair]``.
``AxialRotary(head_dim)`` with the defaults gives the angles of the reference's sensor-point
positions (``fovi/arch/knnvit.py:420-464``: two axes, frequencies ``2 pi / 100 ** (j / n)``, pairs
``(j, j + head_dim / 2)``) from ``SamplingCoords.cartesian_rowcol``.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .. import _lib

__all__ = ["rotary", "AxialRotary"]

_PAIRINGS = {"half": _lib.PAIR_HALF, "adjacent": _lib.PAIR_ADJACENT}


def _launch(x, positions, freqs, ends, pairing, inverse):
    b, n, h, d = x.shape
    x0, x1, x2, x3 = x.stride()
    if x3 != 1:
        x = x.contiguous()
        x0, x1, x2, _ = x.stride()
    y = torch.empty_like(x)              # a dense layout of x is kept (heads before tokens, say)
    if b * n * h == 0:
        return y
    y0, y1, y2, y3 = y.stride()
    if y3 != 1:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        y0, y1, y2, _ = y.stride()
    a = _lib.RotaryArgs()
    a.x, a.dtype, a.pairing = x.data_ptr(), _lib.dtype_code(x.dtype), pairing
    a.batch, a.length, a.heads, a.head_dim = b, n, h, d
    a.x_stride[:] = (x0, x1, x2)
    a.positions, a.freqs = positions.data_ptr(), freqs.data_ptr()
    a.pos_stride[:] = positions.stride()[:2] if positions.dim() == 3 else (0, positions.stride(0))
    a.n_axes, a.inverse = len(ends), inverse
    a.section_end[:len(ends)] = ends
    a.y = y.data_ptr()
    a.y_stride[:] = (y0, y1, y2)
    _lib.check(_lib.load().fovi_rotary(a, _lib.stream_of(x)), "fovi_rotary")
    return y


class _RotaryFn(torch.autograd.Function):
    """``fovi_rotary``; its gradient is the rotation by the negative angles, itself differentiable."""

    @staticmethod
    def forward(ctx, x, positions, freqs, ends, pairing, inverse):
        ctx.save_for_backward(positions, freqs)
        ctx.ends, ctx.pairing, ctx.inverse = ends, pairing, inverse
        return _launch(x, positions, freqs, ends, pairing, inverse)

    @staticmethod
    def backward(ctx, dy):
        positions, freqs = ctx.saved_tensors
        call = _RotaryFn.apply if torch.is_grad_enabled() or _lib.forward_mode() else _launch
        return call(dy, positions, freqs, ctx.ends, ctx.pairing, 1 - ctx.inverse), None, None, None, None, None


def rotary(x, positions, freqs, sections, pairing="half"):
    """Turns the heads ``x [B, L, H, D]`` (fp32 or bf16) by their tokens' positions.

    ``positions [L, A]`` or ``[B, L, A]`` (taken in fp32), ``freqs [P]`` (fp32), ``sections`` the
    number of pairs of each of the A axes, in order (their sum is P, 2 P <= D; 1 to 4 axes).
    ``pairing``: 'half' pairs elements (j, j + P), 'adjacent' (2 j, 2 j + 1); elements from 2 P on
    stay as they are, and so does a token at position 0 (a class token, say). Differentiable in
    ``x``, any number of times; the layout of ``x`` is kept where it is dense.
    """
    _lib.require_device(x, positions, freqs)
    if x.dim() != 4 or x.shape[3] < 2:
        raise ValueError(f"rotary: expected [B, L, H, D] with D >= 2, got {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"rotary: unsupported dtype {x.dtype}")
    if pairing not in _PAIRINGS:
        raise ValueError(f"rotary: unknown pairing {pairing!r}")
    axes = len(sections)
    if not 1 <= axes <= _lib.ROTARY_MAX_AXES:
        raise ValueError(f"rotary: 1 to {_lib.ROTARY_MAX_AXES} axes, got {axes}")
    ends, n = [], 0
    for m in sections:
        if m < 0:
            raise ValueError(f"rotary: negative section in {tuple(sections)}")
        n += int(m)
        ends.append(n)
    if n < 1 or 2 * n > x.shape[3]:
        raise ValueError(f"rotary: {n} pairs do not fit heads of {x.shape[3]}")
    if freqs.shape != (n,):
        raise ValueError(f"rotary: freqs of shape {tuple(freqs.shape)} for {n} pairs")
    want = (x.shape[1], axes)
    if tuple(positions.shape) not in (want, (x.shape[0],) + want):
        raise ValueError(f"rotary: positions of shape {tuple(positions.shape)} for tokens {tuple(x.shape[:2])} and {axes} axes")
    if (positions.requires_grad or freqs.requires_grad) and torch.is_grad_enabled():
        raise ValueError("rotary: no gradient for positions or frequencies")
    if positions.device != x.device or freqs.device != x.device:
        raise ValueError("rotary: positions and freqs must be on the device of x")
    if positions.dtype != torch.float32:
        positions = positions.float()
    if positions.stride(-1) != 1:
        positions = positions.contiguous()
    if freqs.dtype != torch.float32 or not freqs.is_contiguous():
        freqs = freqs.float().contiguous()
    if (torch.is_grad_enabled() and x.requires_grad) or _lib.forward_mode():
        return _RotaryFn.apply(x, positions, freqs, ends, _PAIRINGS[pairing], 0)
    return _launch(x, positions, freqs, ends, _PAIRINGS[pairing], 0)


class AxialRotary(nn.Module):
    """``rotary`` with its frequencies: axis a of n pairs has ``scale / base ** (j / n)``, j = 0 .. n-1.

    ``sections`` defaults to two axes over the whole head; ``base`` and ``scale`` are one value or
    one per axis. The frequencies stay in fp32 when the module is converted to another type.
    """

    def __init__(self, head_dim, sections=None, base=100.0, scale=2 * math.pi, pairing="half", device="cuda"):
        super().__init__()
        if sections is None:
            if head_dim % 4:
                raise ValueError(f"AxialRotary: heads of {head_dim} do not split into two axes of pairs")
            sections = (head_dim // 4, head_dim // 4)
        axes = len(sections)
        base = tuple(base) if isinstance(base, (tuple, list)) else (base,) * axes
        scale = tuple(scale) if isinstance(scale, (tuple, list)) else (scale,) * axes
        if len(base) != axes or len(scale) != axes:
            raise ValueError(f"AxialRotary: {len(base)} bases and {len(scale)} scales for {axes} axes")
        if sum(sections) < 1 or 2 * sum(sections) > head_dim:
            raise ValueError(f"AxialRotary: sections {tuple(sections)} do not fit heads of {head_dim}")
        self.head_dim, self.sections, self.pairing = head_dim, tuple(int(n) for n in sections), pairing
        freqs = [scale[a] * float(base[a]) ** (-j / n) for a, n in enumerate(self.sections) for j in range(n)]
        self.register_buffer("freqs", torch.tensor(freqs, dtype=torch.float64, device="cpu").float().to(device),
                             persistent=False)

    def _apply(self, fn, recurse=True):
        freqs = self.freqs
        super()._apply(fn, recurse)
        if self.freqs.dtype != torch.float32:           # .bfloat16() and the like convert parameters; rounded
            self.freqs = freqs.to(self.freqs.device)    # frequencies would turn by other angles
        return self

    def forward(self, x, positions):
        if x.shape[-1] != self.head_dim:
            raise ValueError(f"AxialRotary: heads of {x.shape[-1]}, built for {self.head_dim}")
        return rotary(x, positions, self.freqs, self.sections, self.pairing)

    def extra_repr(self):
        return f"head_dim={self.head_dim}, sections={self.sections}, pairing={self.pairing!r}"
