"""The gated feed-forward block of token rows on the HIP kernels ``fovi_gated_mlp_fwd`` / ``fovi_gated_mlp_bwd``.

``y = (act(x w_gate^T) * (x w_up^T)) w_down^T``: both first projections, the activation and their product are one
kernel. The backward of bf16 calls with fewer than 768 channels keeps nothing but its inputs: it forms both
projections again beside the gradient that meets them. Others keep the projections in the inputs' type. Sums are fp32;
with bf16 inputs the product of the projections, and in the backward its two gradients (and the kept projections), are
rounded to bf16 (half a step, 2^-8 of each value at most) before the products that they enter. The weights'
gradients are summed in a fixed order: the same inputs give the same bits.

``GatedFeedForward`` is the block of a pre-norm model, with the residual's addition and RMS norm in front;
``GatedFeedForward.int8()`` is its form for serving, with products in 8 bits.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .. import _lib
from .int8 import GATES, Int8Rows, _matrix, gated_linear_int8, linear_int8, quantize_int8
from .norm import RMSNorm, rms_norm_int8

__all__ = ["gated_mlp", "GatedFeedForward", "Int8GatedFeedForward"]


def _args(x, w_gate, w_up, w_down, activation):
    """The arguments that both directions share, with the tensors that they point into."""
    x, rows, x_stride = _matrix(x)
    w_gate, _, gate_stride = _matrix(w_gate)
    w_up, _, up_stride = _matrix(w_up)
    w_down, _, down_stride = _matrix(w_down)
    a = _lib.GatedMlpArgs(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), _lib.dtype_code(x.dtype), activation,
                          rows, x.shape[-1], w_gate.shape[0], x_stride, gate_stride, up_stride, down_stride)
    return a, (x, w_gate, w_up, w_down)


def _workspace(a, nbytes, device):
    work = torch.empty(nbytes, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = work.data_ptr(), nbytes
    return work


def _forward(x, w_gate, w_up, w_down, activation, residual, keep_for_backward):
    a, keep = _args(x, w_gate, w_up, w_down, activation)
    lib = _lib.load()
    saved = None
    if keep_for_backward:
        n = lib.fovi_gated_mlp_saved_bytes(a.rows, a.dim, a.hidden, a.dtype)
        if n:
            saved = torch.empty(n, dtype=torch.uint8, device=x.device)
            a.saved = saved.data_ptr()
    if residual is not None:
        residual, _, a.residual_stride = _matrix(residual)
        a.residual = residual.data_ptr()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a.y, a.y_stride = y.data_ptr(), a.dim
    work = _workspace(a, lib.fovi_gated_mlp_fwd_workspace_bytes(a), x.device)
    _lib.launch(lib.fovi_gated_mlp_fwd, (a,), x, "fovi_gated_mlp_fwd")
    del work, keep
    return y, saved


def _backward(ctx, saved, dy):
    x, w_gate, w_up, w_down, kept = saved
    need_x, need_gate, need_up, need_down = ctx.needs_input_grad[:4]
    a, keep = _args(x, w_gate, w_up, w_down, ctx.activation)
    lib = _lib.load()
    dres = dy if ctx.needs_input_grad[5] else None
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    dyr, _, a.dy_stride = _matrix(dy)
    a.dy = dyr.data_ptr()
    if kept is not None:
        a.saved = kept.data_ptr()
    dx = dgate = dup = ddown = None

    def like(t):
        return torch.empty(t.shape, dtype=t.dtype, device=t.device)

    if need_x:
        dx = like(x)
        a.dx = dx.data_ptr()
    if need_gate or need_up:
        dgate, dup = like(w_gate), like(w_up)
        a.dw_gate, a.dw_up = dgate.data_ptr(), dup.data_ptr()
    if need_down:
        ddown = like(w_down)
        a.dw_down = ddown.data_ptr()
    if need_x or need_gate or need_up or need_down:
        work = _workspace(a, lib.fovi_gated_mlp_bwd_workspace_bytes(a), x.device)
        _lib.launch(lib.fovi_gated_mlp_bwd, (a,), x, "fovi_gated_mlp_bwd")
        del work
    del keep
    return dx, dgate if need_gate else None, dup if need_up else None, ddown, None, dres


class _GatedMlpFn(torch.autograd.Function):
    """Forward ``fovi_gated_mlp_fwd``; backward ``fovi_gated_mlp_bwd``."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation, residual):
        y, kept = _forward(x, w_gate, w_up, w_down, activation, residual, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, kept)
        ctx.activation = activation
        return y

    @staticmethod
    def backward(ctx, dy):
        return _lib.differentiated_once(_backward, ctx, dy)


def _autocast_bf16():
    return torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16


def gated_mlp(x, w_gate, w_up, w_down, activation="silu", residual=None):
    """``(act(x w_gate^T) * (x w_up^T)) w_down^T + residual`` of ``x [..., C]``, in its type (fp32 or bf16).

    ``w_gate, w_up [F, C]`` and ``w_down [C, F]`` are of ``x``'s type (under bf16 autocast fp32 inputs are taken in bf16);
    ``activation`` 'silu' or 'gelu' (the exact one); ``residual`` of ``x``'s shape and type, or None. Rows of any stride and
    alignment are read where they are. Differentiable once in everything.
    """
    tensors = (x, w_gate, w_up, w_down) if residual is None else (x, w_gate, w_up, w_down, residual)
    _lib.require_device(*tensors)
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"gated_mlp: expected [..., C] with C >= 1, got {tuple(shape)}")
    c, weights = shape[-1], w_gate.shape
    if len(weights) != 2 or weights[0] < 1 or weights[1] != c or w_up.shape != weights or w_down.shape != (c, weights[0]):
        raise ValueError(f"gated_mlp: weights {tuple(weights)}, {tuple(w_up.shape)} and {tuple(w_down.shape)} for {c} channels")
    if activation not in GATES:
        raise ValueError(f"gated_mlp: unknown activation {activation!r}")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"gated_mlp: residual of shape {tuple(residual.shape)} for rows {tuple(shape)}")
    if _autocast_bf16():
        tensors = tuple(t.to(torch.bfloat16) for t in tensors)
        x, w_gate, w_up, w_down = tensors[:4]
        residual = None if residual is None else tensors[4]
    dtype, device, grad = x.dtype, x.device, False
    for t in tensors:
        if t.dtype is not dtype or dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"gated_mlp: unsupported dtypes {', '.join(str(t.dtype) for t in tensors)}")
        if t.device != device:
            raise ValueError("gated_mlp: all tensors must be on one device")
        grad = grad or t.requires_grad
    if x.numel() == 0:
        y = (x @ w_gate.t() * (x @ w_up.t())) @ w_down.t()         # zero gradients for the weights
        return y if residual is None else y + residual
    if (grad and torch.is_grad_enabled()) or _lib.forward_mode():
        return _GatedMlpFn.apply(x, w_gate, w_up, w_down, GATES[activation], residual)
    return _forward(x, w_gate, w_up, w_down, GATES[activation], residual, False)[0]


class GatedFeedForward(nn.Module):
    """``total + gated_mlp(rms_norm(total))`` with ``total = x + residual``: the feed-forward half of a pre-norm block.

    ``x`` is what the half in front adds to its ``residual`` (without one, ``total`` is ``x``). ``hidden`` defaults to 8/3 of
    ``dim``, rounded up to a multiple of 64. Weights are fp32; under bf16 autocast the products are in bf16.
    """

    def __init__(self, dim, hidden=None, activation="silu", eps=1e-6, device="cuda"):
        super().__init__()
        if activation not in GATES:
            raise ValueError(f"GatedFeedForward: unknown activation {activation!r}")
        hidden = -(-8 * dim // (3 * 64)) * 64 if hidden is None else hidden
        self.dim, self.hidden, self.activation = dim, hidden, activation
        self.norm = RMSNorm(dim, eps=eps, device=device)
        self.w_gate = nn.Parameter(torch.empty(hidden, dim, device=device))
        self.w_up = nn.Parameter(torch.empty(hidden, dim, device=device))
        self.w_down = nn.Parameter(torch.empty(dim, hidden, device=device))
        with torch.no_grad():
            for w in (self.w_gate, self.w_up, self.w_down):
                w.uniform_(-1, 1).mul_(1 / math.sqrt(w.shape[1]))   # as nn.Linear draws its weights

    def forward(self, x, residual=None):
        if residual is None:
            y, total = self.norm(x), x
        else:
            y, total = self.norm(x, residual)
        weights = self.w_gate, self.w_up, self.w_down
        if total.dtype == torch.float32 and _autocast_bf16():      # an fp32 residual stream stays one
            return total + gated_mlp(y, *weights, self.activation)
        return gated_mlp(y, *weights, self.activation, residual=total)

    def int8(self):
        """The same block for serving, with its weights in 8 bits."""
        return Int8GatedFeedForward(self)

    def extra_repr(self):
        return f"dim={self.dim}, hidden={self.hidden}, activation={self.activation!r}"


class Int8GatedFeedForward(nn.Module):
    """A ``GatedFeedForward`` for serving: norm, projections and down projection on int8 rows, the sums between them in the
    rows' type. No gradients."""

    def __init__(self, block):
        super().__init__()
        self.dim, self.hidden, self.activation, self.eps = block.dim, block.hidden, block.activation, block.norm.eps
        with torch.no_grad():
            self.register_buffer("norm_weight", block.norm.weight.detach().clone())
            for name in ("w_gate", "w_up", "w_down"):
                q = quantize_int8(getattr(block, name))
                self.register_buffer(name, q.data)
                self.register_buffer(name + "_scale", q.scale)

    def _apply(self, fn, recurse=True):
        kept = {n: t for n, t in self._buffers.items() if t.dtype == torch.float32}
        super()._apply(fn, recurse)
        for n, t in kept.items():                       # .bfloat16() and the like would round the scales
            if self._buffers[n].dtype != torch.float32:
                self._buffers[n] = t.to(self._buffers[n].device)
        return self

    def _rows(self, name):
        return Int8Rows(getattr(self, name), getattr(self, name + "_scale"))

    def forward(self, x, residual=None):
        if residual is None:
            y, total = rms_norm_int8(x, self.norm_weight, self.eps), x
        else:
            y, total = rms_norm_int8(x, self.norm_weight, self.eps, residual)
        h = gated_linear_int8(y, self._rows("w_gate"), self._rows("w_up"), self.activation, dtype=x.dtype)
        return linear_int8(quantize_int8(h), self._rows("w_down"), residual=total, dtype=x.dtype)

    def extra_repr(self):
        return f"dim={self.dim}, hidden={self.hidden}, activation={self.activation!r}"
