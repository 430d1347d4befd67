"""Attention of queries to the states of an encoder on the HIP kernels ``fovi_attention_fwd`` / ``fovi_attention_bwd``.

Queries and states have lengths of their own: probe or answer tokens over the tokens of several
fixations, or tokens over themselves. Several query heads may share a key head. A row of the score
matrix that keeps no state gives zeros and passes no gradient; what lies in places that a length or
a mask leaves out has no effect, infinities and NaN included. Scores, softmax statistics and sums
are fp32; the sums are in a fixed order, so the same inputs give the same bits.

With bf16 inputs the matrix products take bf16 on both sides: probabilities are rounded to it before the
products with ``v`` and with the incoming gradient, score gradients before those with ``k`` and ``q`` (2^-9
of each value at most), and the part of the output that its rounding takes away is kept for the backward in
bf16. Outputs of normal inputs were 0.0019 to 0.0024 off the exact ones (norm of the difference over the
norm), where fp32 probabilities give 0.0017, most of it the rounding of the output itself.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from .. import _lib

__all__ = ["cross_attention"]


def _strides(t):
    """Strides of batch, token and head, 0 along dimensions of one."""
    s0, s1, s2, _ = t.stride()
    if (s0 | s1 | s2) & 7 == 0:
        return s0, s1, s2
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3]))


def _whole(t):
    """Whether the kernels can read (or write) ``t`` where it is: heads of whole 16-byte pieces at
    aligned addresses, tokens less than 64 MiB apart."""
    rest = (7 if t.dtype == torch.bfloat16 else 3)
    s0, s1, s2 = _strides(t)
    return t.stride(3) == 1 and (s0 | s1 | s2 | t.shape[3]) & rest == 0 and t.data_ptr() & 15 == 0 and s1 < 1 << 24


def _pieces(t):
    """``t`` as the kernels read it. Other layouts are copied, heads padded with zeros to the next
    piece (which no score or sum notices)."""
    if _whole(t):
        return t
    extra = -t.shape[3] % (16 // t.element_size())
    if extra:
        return torch.nn.functional.pad(t, (0, extra))
    return t.clone(memory_format=torch.contiguous_format)


def _like(t):
    """An output of ``t``'s shape, in its layout where that is dense."""
    y = torch.empty_like(t)
    return y if _whole(y) else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _args(a, q, k, v, kv_lengths, mask, scale):
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.dtype = _lib.dtype_code(q.dtype)
    a.batch, a.q_len, a.heads, a.head_dim = q.shape
    _, a.kv_len, a.kv_heads, _ = k.shape
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = _strides(q), _strides(k), _strides(v)
    if mask is not None:
        a.mask_kind = _lib.MASK_KEEP if mask.dtype == torch.int32 else _lib.MASK_BIAS
        a.mask = mask.data_ptr()
        a.mask_stride[:] = mask.stride()
    if kv_lengths is not None:
        a.kv_lengths = kv_lengths.data_ptr()
    a.scale = scale


def _packed(mask, b, h, n, states):
    """A boolean mask as the kernels read it: 32 states a word, broadcast dimensions packed once."""
    s = mask.stride()
    sizes = tuple(1 if step == 0 else m for m, step in zip((b, h, n), s))
    words = torch.empty(sizes + ((states + 31) // 32,), dtype=torch.int32, device=mask.device)
    if words.numel():
        _lib.check(_lib.load().fovi_attention_pack_mask(mask.data_ptr(), (C.c_int64 * 4)(*s), *sizes, states,
                                                        words.data_ptr(), _lib.stream_of(mask)),
                   "fovi_attention_pack_mask")
    return words.expand(b, h, n, words.shape[3])


def _workspace(a, size, device):
    """The call's workspace, kept alive by the caller until the launch."""
    n = size(a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim, a.dtype)
    if n == 0:
        return None
    work = torch.empty(n, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = work.data_ptr(), n
    return work


def _forward(q, k, v, kv_lengths, mask, scale, keep):
    """The output, and with ``keep`` what the backward needs: the rows' statistics and what the
    rounding of a bf16 output takes away."""
    out, stats, rest = _like(q), None, None
    b, n, h, _ = q.shape
    if keep:
        stats = torch.empty(2, b, h, n, dtype=torch.float32, device=q.device)
        if q.dtype == torch.bfloat16:
            rest = torch.empty_strided(out.shape, out.stride(), dtype=out.dtype, device=q.device)
    if b * n == 0:
        return out, stats, rest
    lib = _lib.load()
    a = _lib.AttentionArgs()
    _args(a, q, k, v, kv_lengths, mask, scale)
    a.out = out.data_ptr()
    a.out_stride[:] = _strides(out)
    if keep:
        a.stats = stats.data_ptr()
        if rest is not None:
            a.out_rest = rest.data_ptr()
    work = _workspace(a, lib.fovi_attention_fwd_workspace_bytes, q.device)
    _lib.check(lib.fovi_attention_fwd(a, _lib.stream_of(q)), "fovi_attention_fwd")
    del work
    return out, stats, rest


def _backward(ctx, saved, dout):
    q, k, v, kv_lengths, mask, out, stats, rest = saved
    dq, dk, dv = _like(q), _like(k), _like(v)
    if q.numel() == 0:
        return dq, dk.zero_(), dv.zero_(), None, None, None
    dout = _pieces(dout if dout.dtype == q.dtype else dout.to(q.dtype))
    lib = _lib.load()
    a = _lib.AttentionBwdArgs()
    f = a.fwd
    _args(f, q, k, v, kv_lengths, mask, ctx.scale)
    f.out, f.stats, a.dout = out.data_ptr(), stats.data_ptr(), dout.data_ptr()
    if rest is not None:
        f.out_rest = rest.data_ptr()
    a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    f.out_stride[:], a.dout_stride[:] = _strides(out), _strides(dout)
    a.dq_stride[:], a.dk_stride[:], a.dv_stride[:] = _strides(dq), _strides(dk), _strides(dv)
    work = _workspace(f, lib.fovi_attention_bwd_workspace_bytes, q.device)
    _lib.check(lib.fovi_attention_bwd(a, _lib.stream_of(q)), "fovi_attention_bwd")
    del work
    return dq, dk, dv, None, None, None


class _CrossAttentionFn(torch.autograd.Function):
    """Forward ``fovi_attention_fwd`` with the rows' maxima and sums kept; backward ``fovi_attention_bwd``."""

    @staticmethod
    def forward(ctx, q, k, v, kv_lengths, mask, scale):
        out, stats, rest = _forward(q, k, v, kv_lengths, mask, scale, True)
        ctx.save_for_backward(q, k, v, kv_lengths, mask, out, stats, rest)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, dout):
        return _lib.differentiated_once(_backward, ctx, dout)


def cross_attention(q, k, v, kv_lengths=None, mask=None, scale=None):
    """``softmax(scale q k^T + mask) v``, in the type and layout of ``q [B, Lq, Hq, D]``.

    ``k, v [B, Lk, Hk, D]``, Hq a multiple of Hk (query head h reads key head h // (Hq / Hk)), D up
    to 128, fp32 or bf16 (under bf16 autocast fp32 inputs are taken in bf16). Any strides: heads of
    whole 16-byte pieces at aligned addresses are read where they are (broadcast ones too), others copied.

    ``kv_lengths [B]`` (integers on the device): image b has only its first ``kv_lengths[b]`` states.
    ``mask``, broadcastable to ``[B, Hq, Lq, Lk]``: boolean, True where a row may read a state, or a
    float bias added to the scores (-inf leaves a state out). ``scale`` defaults to D ** -0.5.
    Differentiable once in ``q``, ``k`` and ``v``. bf16 inputs: probabilities and score gradients are rounded to
    bf16 before their products.
    """
    _lib.require_device(q, k, v, kv_lengths, mask)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"cross_attention: expected [B, L, H, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    b, lq, hq, d = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise ValueError(f"cross_attention: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} do not fit")
    lk, hk = k.shape[1], k.shape[2]
    if hq < 1 or hk < 1 or hq % hk:
        raise ValueError(f"cross_attention: {hq} query heads over {hk} key heads")
    if not 1 <= d <= 128:
        raise ValueError(f"cross_attention: heads of {d}, at most 128 are supported")
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
        q, k, v = q.to(torch.bfloat16), k.to(torch.bfloat16), v.to(torch.bfloat16)
    if q.dtype not in (torch.float32, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"cross_attention: unsupported dtypes {q.dtype}, {k.dtype}, {v.dtype}")
    if k.device != q.device or v.device != q.device:
        raise ValueError("cross_attention: q, k and v must be on one device")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError(f"cross_attention: scale must be positive and finite, got {scale}")
    if kv_lengths is not None:
        if kv_lengths.shape != (b,) or kv_lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"cross_attention: kv_lengths must be {b} integers, got {kv_lengths.dtype} {tuple(kv_lengths.shape)}")
        if kv_lengths.device != q.device:
            raise ValueError("cross_attention: kv_lengths must be on the device of q")
        if kv_lengths.dtype != torch.int32:
            kv_lengths = kv_lengths.clamp(0, lk).to(torch.int32)
        if kv_lengths.stride(0) != 1:
            kv_lengths = kv_lengths.contiguous()
    if mask is not None:
        if mask.requires_grad and torch.is_grad_enabled():
            raise ValueError("cross_attention: no gradient for the mask")
        if mask.device != q.device:
            raise ValueError("cross_attention: mask must be on the device of q")
        if mask.dtype == torch.bfloat16:
            mask = mask.float()
        if mask.dtype not in (torch.bool, torch.float32):
            raise TypeError(f"cross_attention: unsupported mask dtype {mask.dtype}")
        try:
            mask = mask.expand(b, hq, lq, lk)
        except RuntimeError:
            raise ValueError(f"cross_attention: mask of shape {tuple(mask.shape)} for {(b, hq, lq, lk)}") from None
        if mask.dtype == torch.bool:
            mask = _packed(mask, b, hq, lq, lk)
    q, k, v = _pieces(q), _pieces(k), _pieces(v)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or _lib.forward_mode():
        out = _CrossAttentionFn.apply(q, k, v, kv_lengths, mask, scale)
    else:
        out = _forward(q, k, v, kv_lengths, mask, scale, False)[0]
    return out if out.shape[3] == d else out[..., :d]
