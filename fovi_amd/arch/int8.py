"""Token rows and weights in 8 bits with a scale each, and their products, on the HIP kernels ``fovi_quantize_rows``,
``fovi_dequantize_rows`` and ``fovi_linear_int8``.

For serving: a linear layer's weights are quantised once, one scale for each output channel
(``quantize_int8(weight)``), its inputs at every call, one scale for each token. A row's largest value is 127
steps, values are rounded to the nearest step; the product's sums are exact. Nothing here has gradients.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch
import torch.nn as nn

from .. import _lib

__all__ = ["Int8Rows", "quantize_int8", "linear_int8", "gated_linear_int8", "Int8Linear"]

GATES = {"silu": _lib.GATE_SILU, "gelu": _lib.GATE_GELU}


def refuse_gradients(what, *tensors):
    """Raises where a gradient or tangent is asked for."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what}: no gradients (call it under torch.no_grad())")
    if _lib.forward_mode():
        raise ValueError(f"{what}: no forward-mode derivatives")


def _matrix(t):
    """``t [..., K]`` as rows at one stride, elements adjacent: ``(tensor, rows, stride)``, copied where it is not."""
    k = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // k, k
    if t.stride(-1) == 1 or k == 1:
        rows, stride = 1, 0
        for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if n == 1:
                continue
            if rows == 1:
                rows, stride = n, s
            elif s == rows * stride:
                rows *= n
            else:
                break
        else:
            if rows == 1 or stride >= k:
                return t, rows, max(stride, k)
    return t.contiguous(), t.numel() // k, k


class Int8Rows(NamedTuple):
    """``data``: int8 ``[..., K]``; ``scale``: fp32 ``[...]`` on the same device, so that ``x ~= data * scale[..., None]``."""
    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype=torch.float32):
        """The values that the rows stand for, in fp32 or bf16. No gradient, and asking for one raises."""
        _rows_check("dequantize", self)
        if dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"dequantize: unsupported dtype {dtype}")
        refuse_gradients("dequantize", self.scale)
        y = torch.empty(self.data.shape, dtype=dtype, device=self.data.device)
        if y.numel():
            data, rows, stride = _matrix(self.data)
            scale = self.scale.contiguous()
            _lib.launch(_lib.load().fovi_dequantize_rows, (data.data_ptr(), scale.data_ptr(), rows, data.shape[-1], stride,
                                                           y.data_ptr(), _lib.dtype_code(dtype)), y, "fovi_dequantize_rows")
        return y


def _rows_check(what, rows):
    data, scale = rows
    if not (data.is_cuda and scale.is_cuda):
        _lib.require_device(data, scale)
    if data.dtype is not torch.int8 or scale.dtype is not torch.float32:
        raise TypeError(f"{what}: expected int8 rows with fp32 scales, got {data.dtype} and {scale.dtype}")
    shape = data.shape
    if len(shape) < 1 or shape[-1] < 1 or scale.shape != shape[:-1]:
        raise ValueError(f"{what}: rows {tuple(shape)} with scales {tuple(scale.shape)}")
    if scale.device != data.device:
        raise ValueError(f"{what}: scales on {scale.device}, rows on {data.device}")


def quantize_int8(x):
    """``x [..., K]`` (fp32 or bf16) as ``Int8Rows``: ``scale = max|row| / 127``, ``data = x / scale`` rounded to nearest
    even. A row with an infinity or NaN stands for NaN throughout."""
    _lib.require_device(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize_int8: expected [..., K] with K >= 1, got {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"quantize_int8: unsupported dtype {x.dtype}")
    refuse_gradients("quantize_int8", x)
    q = Int8Rows(torch.empty(x.shape, dtype=torch.int8, device=x.device),
                 torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device))
    if x.numel():
        xr, rows, stride = _matrix(x)
        _lib.launch(_lib.load().fovi_quantize_rows, (xr.data_ptr(), _lib.dtype_code(x.dtype), 1, rows, x.shape[-1],
                                                     (C.c_int64 * 2)(0, stride), q.data.data_ptr(), q.scale.data_ptr()),
                    x, "fovi_quantize_rows")
    return q


def _weight(what, w, k, device):
    """``(data, stride, scale)`` of weights as the kernels read them."""
    _rows_check(what, w)
    data, scale = w
    shape = data.shape
    if len(shape) != 2 or shape[1] != k:
        raise ValueError(f"{what}: weights {tuple(shape)} for {k} inputs")
    if data.device != device:
        raise ValueError(f"{what}: weights on {data.device}, x on {device}")
    s0, s1 = data.stride()
    if s1 != 1 or s0 < k:
        data, s0 = data.contiguous(), k
    return data, s0, scale if scale.is_contiguous() else scale.contiguous()


def _product(what, x, weight, weight2, activation, bias, residual, dtype):
    _rows_check(what, x)
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise TypeError(f"{what}: unsupported dtype {dtype}")
    data, scale = x
    shape, device = data.shape, data.device
    k = shape[-1]
    if k > 131071:
        raise ValueError(f"{what}: {k} inputs, at most 131071 keep the sums exact")
    w, w_stride, w_scale = _weight(what, weight, k, device)
    n = w.shape[0]
    shape = shape[:-1] + (n,)
    refuse_gradients(what, scale, w_scale, None if weight2 is None else weight2.scale, bias, residual)
    w2, w2_stride, w2_scale, act = None, 0, None, 0
    if weight2 is not None:
        w2, w2_stride, w2_scale = _weight(what, weight2, k, device)
        if w2.shape != w.shape:
            raise ValueError(f"{what}: weights {tuple(w.shape)} and {tuple(w2.shape)}")
        if activation not in GATES:
            raise ValueError(f"{what}: unknown activation {activation!r}")
        act = GATES[activation]
    if bias is not None:
        _lib.require_device(bias)
        if bias.shape != (n,) or bias.device != device:
            raise ValueError(f"{what}: bias {tuple(bias.shape)} on {bias.device} for {n} outputs on {device}")
        bias = bias.float().contiguous()
    if residual is not None:
        _lib.require_device(residual)
        if residual.shape != shape or residual.dtype != dtype or residual.device != device:
            raise ValueError(f"{what}: residual {tuple(residual.shape)} {residual.dtype} on {residual.device}, the output is "
                             f"{tuple(shape)} {dtype} on {device}")
    out = torch.empty(shape, dtype=dtype, device=device)
    if out.numel() == 0:
        return out
    data, rows, stride = _matrix(data)
    if not scale.is_contiguous():
        scale = scale.contiguous()
    r_stride = 0
    if residual is not None:
        residual, _, r_stride = _matrix(residual)
    a = _lib.LinearInt8Args(data.data_ptr(), scale.data_ptr(), rows, k, n, stride, w.data_ptr(), w_scale.data_ptr(), w_stride,
                            None if w2 is None else w2.data_ptr(), None if w2 is None else w2_scale.data_ptr(), w2_stride, act, _lib.dtype_code(dtype),
                            None if bias is None else bias.data_ptr(), None if residual is None else residual.data_ptr(), r_stride,
                            out.data_ptr(), n)
    lib = _lib.load()
    nbytes = lib.fovi_linear_int8_workspace_bytes(a)
    work = None
    if nbytes:
        work = torch.empty(nbytes, dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes = work.data_ptr(), nbytes
    _lib.launch(lib.fovi_linear_int8, (a,), out, "fovi_linear_int8")
    del work
    return out


def linear_int8(x, weight, bias=None, residual=None, dtype=torch.bfloat16):
    """``x weight^T + bias + residual`` in ``dtype`` (fp32 or bf16), rounded once.

    ``x``: ``Int8Rows [..., K]``, a scale for each token; ``weight``: ``Int8Rows [N, K]``, a scale for each output channel.
    ``bias [N]`` is taken in fp32; ``residual [..., N]`` is of ``dtype``. Rows of any stride and alignment.
    """
    return _product("linear_int8", x, weight, None, None, bias, residual, dtype)


def gated_linear_int8(x, gate, up, activation="silu", dtype=torch.bfloat16):
    """``act(x gate^T) * (x up^T)`` in ``dtype``, both products over one reading of ``x``; ``activation`` 'silu' or 'gelu'."""
    return _product("gated_linear_int8", x, gate, up, activation, None, None, dtype)


class Int8Linear(nn.Module):
    """An ``nn.Linear`` for serving: its weights in 8 bits, its inputs quantised at every call (``Int8Rows`` are taken as
    they are). Its outputs are in ``dtype``, by default the inputs' type, or for ``Int8Rows`` the residual's (without one
    bf16)."""

    def __init__(self, linear):
        super().__init__()
        with torch.no_grad():
            weight = quantize_int8(linear.weight)
        self.register_buffer("weight", weight.data)
        self.register_buffer("weight_scale", weight.scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().float())

    def _apply(self, fn, recurse=True):
        kept = {n: getattr(self, n) for n in ("weight_scale", "bias")}
        super()._apply(fn, recurse)
        for n, t in kept.items():                       # .bfloat16() and the like would round the scales
            if t is not None and getattr(self, n).dtype != torch.float32:
                setattr(self, n, t.to(getattr(self, n).device))
        return self

    def forward(self, x, residual=None, dtype=None):
        if not isinstance(x, Int8Rows):
            dtype = x.dtype if dtype is None else dtype
            x = quantize_int8(x)
        elif dtype is None:
            dtype = torch.bfloat16 if residual is None else residual.dtype
        return linear_int8(x, Int8Rows(self.weight, self.weight_scale), self.bias, residual, dtype)

    def extra_repr(self):
        return f"in_features={self.weight.shape[1]}, out_features={self.weight.shape[0]}, bias={self.bias is not None}"
