"""Layer norm and RMS norm of token rows on the HIP kernels ``fovi_layer_norm_fwd`` / ``fovi_layer_norm_bwd`` and
``fovi_rms_norm_fwd`` / ``fovi_rms_norm_bwd``.

``y = (x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, statistics and sums
in fp32, one rounding at the output (the reference's token norms: ``fovi/arch/norm.py:125-157``).
Rows in any layout whose channels are adjacent are read where they are (a slice of tokens, a
head-split view); other layouts are copied first. The gradients of weight and bias are summed in a
fixed order: the same inputs give the same bits.

``rms_norm`` is ``y = x / sqrt(mean(x^2) + eps) * weight``, with the addition of a residual in front where one is given
(the same reading of rows, statistics and rounding); ``rms_norm_int8`` gives its rows in 8 bits with a
scale each, as the products of ``fovi_amd.arch.int8`` read them.
"""
from __future__ import annotations

import ctypes as C

import torch
import torch.nn as nn

from .. import _lib
from .int8 import Int8Rows, refuse_gradients

__all__ = ["layer_norm", "LayerNorm", "rms_norm", "rms_norm_int8", "RMSNorm"]


def _rows(x):
    """``(x, rows0, rows1, stride0, stride1)``: the leading dimensions as two, ``x`` copied where
    its channels are not adjacent or more than two row strides remain."""
    c = x.shape[-1]
    if x.is_contiguous():
        return x, 1, x.numel() // c, 0, c
    if x.stride(-1) == 1 or c == 1:
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
    return x.contiguous(), 1, x.numel() // c, 0, c


def _forward(x, weight, bias, eps, stats):
    xr, n0, n1, s0, s1 = _rows(x)
    c = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = _lib.LayerNormArgs()
    a.x, a.dtype, a.rows0, a.rows1, a.channels, a.eps = xr.data_ptr(), _lib.dtype_code(x.dtype), n0, n1, c, eps
    a.x_stride[:] = (s0, s1)
    if weight is not None:
        a.weight, a.p_dtype = weight.data_ptr(), _lib.dtype_code(weight.dtype)
    if bias is not None:
        a.bias, a.p_dtype = bias.data_ptr(), _lib.dtype_code(bias.dtype)
    a.y = y.data_ptr()
    a.y_stride[:] = (n1 * c, c)
    if stats is not None:
        a.mean, a.rstd = stats.data_ptr(), stats.data_ptr() + 4 * n0 * n1
    lib = _lib.load()
    _lib.check(lib.fovi_layer_norm_fwd(a, _lib.stream_of(x)), "fovi_layer_norm_fwd")
    return y


def _backward(ctx, saved, dy):
    x, weight, bias, stats = saved
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    c = x.shape[-1]
    xr, n0, n1, s0, s1 = _rows(x)
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    dyr, m0, m1, t0, t1 = _rows(dy)
    if (m0, m1) != (n0, n1):            # rows of x and dy in the same two levels; one splits into any two
        if m0 == 1:
            t0 = n1 * t1
        elif n0 == 1:
            n0, n1, s0 = m0, m1, m1 * s1
        else:
            dyr, t0, t1 = dy.contiguous(), n1 * c, c
    a = _lib.LayerNormArgs()
    a.x, a.dtype, a.rows0, a.rows1, a.channels, a.eps = xr.data_ptr(), _lib.dtype_code(x.dtype), n0, n1, c, ctx.eps
    a.x_stride[:] = (s0, s1)
    a.dy = dyr.data_ptr()
    a.dy_stride[:] = (t0, t1)
    a.mean, a.rstd = stats.data_ptr(), stats.data_ptr() + 4 * n0 * n1
    dx = dw = db = work = None
    lib = _lib.load()
    if need_x:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a.dx = dx.data_ptr()
        a.dx_stride[:] = (n1 * c, c)
    if weight is not None:
        a.weight, a.p_dtype = weight.data_ptr(), _lib.dtype_code(weight.dtype)
        if need_w:
            dw = torch.empty_like(weight)
            a.dweight = dw.data_ptr()
    if need_b:
        db = torch.empty_like(bias)
        a.dbias, a.p_dtype = db.data_ptr(), _lib.dtype_code(bias.dtype)
    if need_w or need_b:
        nbytes = lib.fovi_layer_norm_workspace_bytes(n0 * n1, c, a.dtype)
        work = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        a.workspace, a.workspace_bytes = work.data_ptr(), nbytes
    _lib.check(lib.fovi_layer_norm_bwd(a, _lib.stream_of(x)), "fovi_layer_norm_bwd")
    return dx, dw, db, None


class _LayerNormFn(torch.autograd.Function):
    """Forward ``fovi_layer_norm_fwd`` with the rows' statistics kept; backward ``fovi_layer_norm_bwd``."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        stats = torch.empty(2, x.numel() // x.shape[-1], dtype=torch.float32, device=x.device)
        y = _forward(x, weight, bias, eps, stats)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.eps = eps
        return y

    @staticmethod
    def backward(ctx, dy):
        return _lib.differentiated_once(_backward, ctx, dy)


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
    if (torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                     or (bias is not None and bias.requires_grad))) or _lib.forward_mode():
        return _LayerNormFn.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, eps, None)


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


_Pair = C.c_int64 * 2


def _rms_args(x, weight, eps, residual):
    """The arguments that both directions share, with the tensors that they point into."""
    c = x.shape[-1]
    xr, n0, n1, s0, s1 = _rows(x)
    rr, t0, t1 = None, 0, 0
    if residual is not None:
        rr, m0, m1, t0, t1 = _rows(residual)
        if (m0, m1) != (n0, n1):        # rows of both in the same two levels; one splits into any two
            if m0 == 1:
                t0 = n1 * t1
            elif n0 == 1:
                n0, n1, s0 = m0, m1, m1 * s1
            else:
                rr, t0, t1 = residual.contiguous(), n1 * c, c
    a = _lib.RmsNormArgs(xr.data_ptr(), _lib.dtype_code(x.dtype), 0 if weight is None else _lib.dtype_code(weight.dtype), n0, n1, c,
                         _Pair(s0, s1), None if rr is None else rr.data_ptr(), _Pair(t0, t1),
                         None if weight is None else weight.data_ptr(), eps)
    return a, (xr, rr)


def _rms_forward(x, weight, eps, residual, rstd, quantize=False):
    """``(y, total)``, ``y`` as ``Int8Rows`` with ``quantize``; ``total`` is ``x`` without a residual."""
    a, keep = _rms_args(x, weight, eps, residual)
    total = x
    if residual is not None:
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a.total = total.data_ptr()
    if quantize:
        y = Int8Rows(torch.empty(x.shape, dtype=torch.int8, device=x.device),
                     torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device))
        a.q, a.scale = y.data.data_ptr(), y.scale.data_ptr()
    else:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        a.y = y.data_ptr()
    if rstd is not None:
        a.rstd = rstd.data_ptr()
    _lib.launch(_lib.load().fovi_rms_norm_fwd, (a,), x, "fovi_rms_norm_fwd")
    del keep
    return y, total


def _rms_backward(ctx, saved, dy, dtotal=None):
    total, weight, rstd = saved
    need_x, need_w, need_r = ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[3]
    if dy is None:                                       # nothing comes through the norm
        dx = torch.zeros_like(total) if dtotal is None else dtotal.to(total.dtype)
        return dx if need_x else None, torch.zeros_like(weight) if need_w else None, None, dx if need_r else None
    c = total.shape[-1]
    xr, n0, n1, s0, s1 = _rows(total)
    a = _lib.RmsNormArgs()
    keep = []
    for name, g in (("dy", dy), ("dtotal", dtotal)):
        if g is None:
            continue
        if g.dtype != total.dtype:
            g = g.to(total.dtype)
        gr, m0, m1, t0, t1 = _rows(g)
        if (m0, m1) != (n0, n1):
            if m0 == 1:
                t0 = n1 * t1
            else:
                gr, t0, t1 = g.contiguous(), n1 * c, c
        keep.append(gr)
        setattr(a, name, gr.data_ptr())
        getattr(a, name + "_stride")[:] = (t0, t1)
    a.x, a.dtype, a.rows0, a.rows1, a.channels, a.eps = xr.data_ptr(), _lib.dtype_code(total.dtype), n0, n1, c, ctx.eps
    a.x_stride[:] = (s0, s1)
    a.rstd = rstd.data_ptr()
    dx = dw = work = None
    lib = _lib.load()
    if need_x or need_r:
        dx = torch.empty(total.shape, dtype=total.dtype, device=total.device)
        a.dx = dx.data_ptr()
    if weight is not None:
        a.weight, a.p_dtype = weight.data_ptr(), _lib.dtype_code(weight.dtype)
        if need_w:
            dw = torch.empty_like(weight)
            nbytes = lib.fovi_rms_norm_workspace_bytes(n0 * n1, c)
            work = torch.empty(nbytes, dtype=torch.uint8, device=total.device)
            a.dweight, a.workspace, a.workspace_bytes = dw.data_ptr(), work.data_ptr(), nbytes
    _lib.launch(lib.fovi_rms_norm_bwd, (a,), total, "fovi_rms_norm_bwd")
    del keep
    return dx if need_x else None, dw, None, dx if need_r else None


class _RMSNormFn(torch.autograd.Function):
    """Forward ``fovi_rms_norm_fwd`` with the rows' statistics kept; backward ``fovi_rms_norm_bwd``, which reads the
    gradients that arrive: a block whose ``total`` goes no further has none of it."""

    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        ctx.set_materialize_grads(False)
        rstd = torch.empty(x.numel() // x.shape[-1], dtype=torch.float32, device=x.device)
        y, total = _rms_forward(x, weight, eps, residual, rstd)
        ctx.save_for_backward(total, weight, rstd)
        ctx.eps = eps
        return y if residual is None else (y, total)

    @staticmethod
    def backward(ctx, *grads):
        return _lib.differentiated_once(_rms_backward, ctx, *grads)


def _rms_checks(what, x, weight, eps, residual):
    _lib.require_device(x, weight, residual)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: expected [..., C] with C >= 1, got {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{what}: unsupported dtype {x.dtype}")
    if not eps >= 0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    if weight is not None:
        if weight.shape != x.shape[-1:]:
            raise ValueError(f"{what}: weight of shape {tuple(weight.shape)} for {x.shape[-1]} channels")
        if weight.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"{what}: unsupported weight dtype {weight.dtype}")
        if weight.device != x.device:
            raise ValueError(f"{what}: weight on {weight.device}, x on {x.device}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{what}: residual of shape {tuple(residual.shape)} for rows {tuple(x.shape)}")
        if residual.dtype != x.dtype:
            raise TypeError(f"{what}: residual is {residual.dtype}, x {x.dtype}")
        if residual.device != x.device:
            raise ValueError(f"{what}: residual on {residual.device}, x on {x.device}")


def rms_norm(x, weight=None, eps=1e-6, residual=None):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension of ``x [..., C]`` (fp32 or bf16), in its type.

    With ``residual`` (``x``'s shape and type) the rows are ``total = x + residual``, rounded to that type, and the
    result is ``(y, total)``. ``weight [C]`` is fp32 or bf16 whatever ``x`` is, or None. Differentiable once in
    ``x``, ``weight`` and ``residual``, through both results.
    """
    _rms_checks("rms_norm", x, weight, eps, residual)
    if x.numel() == 0:
        total = x * 1 if residual is None else x + residual
        y = total * 1 if weight is None else (total * weight).to(x.dtype)
        return y if residual is None else (y, total)
    weight = weight if weight is None else weight.contiguous()
    if (torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                     or (residual is not None and residual.requires_grad))) or _lib.forward_mode():
        return _RMSNormFn.apply(x, weight, float(eps), residual)
    y, total = _rms_forward(x, weight, float(eps), residual, None)
    return y if residual is None else (y, total)


def rms_norm_int8(x, weight=None, eps=1e-6, residual=None):
    """``rms_norm`` with its rows as ``Int8Rows`` (``data`` int8 and a ``scale`` for each row: the row's largest value over
    127), quantised from the unrounded norm; with ``residual`` ``(rows, total)``. For serving: no gradient, and
    asking for one raises."""
    _rms_checks("rms_norm_int8", x, weight, eps, residual)
    refuse_gradients("rms_norm_int8", x, weight, residual)
    if x.numel() == 0:
        y = Int8Rows(torch.empty(x.shape, dtype=torch.int8, device=x.device),
                     torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device))
        return y if residual is None else (y, x + residual)
    weight = weight if weight is None else weight.contiguous()
    y, total = _rms_forward(x, weight, float(eps), residual, None, quantize=True)
    return y if residual is None else (y, total)


class RMSNorm(nn.Module):
    """``rms_norm`` with its weight (fp32 unless ``dtype`` says otherwise)."""

    def __init__(self, dim, eps=1e-6, elementwise_affine=True, device="cuda", dtype=torch.float32):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype)) if elementwise_affine else None

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, self.eps, residual)

    def extra_repr(self):
        return f"{self.dim}, eps={self.eps}, elementwise_affine={self.weight is not None}"
