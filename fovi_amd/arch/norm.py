"""Layer norm of token rows on the HIP kernels ``fovi_layer_norm_fwd`` / ``fovi_layer_norm_bwd``.

``y = (x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, statistics and sums
in fp32, one rounding at the output (the reference's token norms: ``fovi/arch/norm.py:125-157``).
Rows in any layout whose channels are adjacent are read where they are (a slice of tokens, a
head-split view); other layouts are copied first. The gradients of weight and bias are summed in a
fixed order: the same inputs give the same bits.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import _lib

__all__ = ["layer_norm", "LayerNorm"]


def _rows(x):
    """``(x, rows0, rows1, stride0, stride1)``: the leading dimensions as two, ``x`` copied where
    its channels are not adjacent or more than two row strides remain."""
    if x.dim() == 2 and x.stride(1) == 1:
        return x, 1, x.shape[0], 0, x.stride(0)
    if x.stride(-1) == 1 or x.shape[-1] == 1:
        dims = []
        for n, s in zip(x.shape[:-1], x.stride()[:-1]):
            if n == 1:
                continue
            if dims and dims[-1][1] == n * s:
                dims[-1] = [dims[-1][0] * n, s]
            else:
                dims.append([n, s])
        if len(dims) <= 2:
            (n0, s0), (n1, s1) = ([[1, 0]] * (2 - len(dims)) + dims)
            return x, n0, n1, s0, s1
    x = x.contiguous()
    c = x.shape[-1]
    return x, 1, x.numel() // c, 0, c


def _args(x, weight, bias, eps):
    x, n0, n1, s0, s1 = _rows(x)
    a = _lib.LayerNormArgs()
    a.x, a.dtype = x.data_ptr(), _lib.dtype_code(x.dtype)
    a.rows0, a.rows1, a.channels = n0, n1, x.shape[-1]
    a.x_stride[:] = (s0, s1)
    param = weight if weight is not None else bias
    a.p_dtype = _lib.F32 if param is None else _lib.dtype_code(param.dtype)
    if weight is not None:
        a.weight = weight.data_ptr()
    if bias is not None:
        a.bias = bias.data_ptr()
    a.eps = eps
    return a, x


class _LayerNormFn(torch.autograd.Function):
    """Forward ``fovi_layer_norm_fwd`` with the rows' statistics kept; backward ``fovi_layer_norm_bwd``."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        a, xr = _args(x, weight, bias, eps)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        c = x.shape[-1]
        a.y = y.data_ptr()
        a.y_stride[:] = (a.rows1 * c, c)
        if keep:
            stats = torch.empty(2, a.rows0 * a.rows1, dtype=torch.float32, device=x.device)
            a.mean, a.rstd = stats.data_ptr(), stats.data_ptr() + 4 * stats.shape[1]
            ctx.save_for_backward(x, weight, bias, stats)
            ctx.eps = eps
        _lib.check(_lib.load().fovi_layer_norm_fwd(a, _lib.stream_handle(x.device)), "fovi_layer_norm_fwd")
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        a, xr = _args(x, weight, bias, ctx.eps)
        # rows of x and dy in the same two levels; the statistics are in row order
        dy = dy.to(x.dtype)
        dyr, n0, n1, s0, s1 = _rows(dy)
        if (n0, n1) != (a.rows0, a.rows1):
            if n0 == 1:                              # one level splits into any two
                n0, n1, s0 = a.rows0, a.rows1, a.rows1 * s1
            elif a.rows0 == 1:
                a.rows0, a.rows1 = n0, n1
                a.x_stride[0] = n1 * a.x_stride[1]
            else:
                dyr = dy.contiguous()
                n0, n1, s0, s1 = a.rows0, a.rows1, a.rows1 * x.shape[-1], x.shape[-1]
        a.dy = dyr.data_ptr()
        a.dy_stride[:] = (s0, s1)
        a.mean, a.rstd = stats.data_ptr(), stats.data_ptr() + 4 * stats.shape[1]
        dx = dw = db = None
        lib = _lib.load()
        if need_x:
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            a.dx = dx.data_ptr()
            a.dx_stride[:] = (n1 * x.shape[-1], x.shape[-1])
        if need_w:
            dw = torch.empty_like(weight, memory_format=torch.contiguous_format)
            a.dweight = dw.data_ptr()
        if need_b:
            db = torch.empty_like(bias, memory_format=torch.contiguous_format)
            a.dbias = db.data_ptr()
        if need_w or need_b:
            nbytes = lib.fovi_layer_norm_workspace_bytes(n0 * n1, x.shape[-1], a.dtype)
            work = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
            a.workspace, a.workspace_bytes = work.data_ptr(), nbytes
        _lib.check(lib.fovi_layer_norm_bwd(a, _lib.stream_handle(x.device)), "fovi_layer_norm_bwd")
        return dx, dw, db, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of ``x [..., C]`` (fp32 or bf16) over its last dimension, in ``x``'s type.

    ``weight`` and ``bias`` ``[C]``, each optional, are fp32 or bf16 whatever ``x`` is (one type for
    both). Differentiable once in all three.
    """
    _lib.require_device(x, weight, bias)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: expected [..., C] with C >= 1, got {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"layer_norm: unsupported dtype {x.dtype}")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != x.shape[-1:]:
            raise ValueError(f"layer_norm: {name} of shape {tuple(t.shape)} for {x.shape[-1]} channels")
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"layer_norm: unsupported {name} dtype {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"layer_norm: {name} on {t.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    if x.numel() == 0:
        y = x * 1
        for t in (weight, bias):
            y = y if t is None else (y * t).to(x.dtype)       # zero gradients for the parameters
        return y
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    keep = torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                        or (bias is not None and bias.requires_grad))
    return _LayerNormFn.apply(x, weight, bias, float(eps), keep)


class LayerNorm(nn.Module):
    """``layer_norm`` with its parameters (fp32 unless ``dtype`` says otherwise)."""

    def __init__(self, dim, eps=1e-5, elementwise_affine=True, bias=True, device="cuda", dtype=torch.float32):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype)) if elementwise_affine and bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.dim}, eps={self.eps}, elementwise_affine={self.weight is not None}"
