"""Cross attention forward and backward against float64, over lengths, heads, layouts, masks and types.

Tolerances, from the arithmetic. fp32: a score is a sum of D products (error about sqrt(D) 2^-24 of
|q||k| scale, 1e-6 absolute at the spreads used here), which the exponential turns into a relative
error; with the sums over the states and the gradients' differences 1e-5 relative is allowed. bf16:
probabilities (and score gradients) enter the second product rounded to bf16, at most 2^-9 each, and
the result is rounded once more; independent roundings add to at most 2^-9 (1 + a) with a <= 2 the
ratio of sum p|v| to |sum p v| over these random inputs: 6e-3. A score gradient is the difference
p (do.v - do.o), which may cancel (one state, equal values): its terms' roundings, 2^-21 of
p (|do.v| + |do.o|) in fp32 and 2^-16 in bf16 (o is kept to 2^-18 there), come on top in dq and dk.
"""
import ctypes as C
import math

import pytest
import torch

from fovi_amd import _lib

TOL = {torch.float32: 1e-5, torch.bfloat16: 6e-3}
TERMS = {torch.float32: 2.0 ** -21, torch.bfloat16: 2.0 ** -16}
INF = math.inf


def _reference(q, k, v, lengths=None, mask=None, scale=None, dout=None):
    """out, dq, dk, dv in float64 on the CPU, pair by pair (what is left out is never multiplied), and the
    norms of what dq and dk are with the terms of the score gradients taken absolutely."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    keep = torch.ones(b, hq, lq, lk, dtype=torch.bool)
    bias = torch.zeros(b, hq, lq, lk, dtype=torch.float64)
    if lengths is not None:
        keep &= torch.arange(lk) < lengths.cpu()[:, None, None, None]
    if mask is not None:
        m = mask.cpu().expand(b, hq, lq, lk)
        if m.dtype == torch.bool:
            keep &= m
        else:
            bias = m.double()
            keep &= bias != -INF
    out = torch.zeros(b, lq, hq, d, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(out), torch.zeros_like(k), torch.zeros_like(v)
    tq, tk = torch.zeros_like(out), torch.zeros_like(k)
    for i in range(b):
        for h in range(hq):
            j = h * hk // hq
            for r in range(lq):
                at = keep[i, h, r].nonzero()[:, 0]
                if len(at) == 0:
                    continue
                kk, vv = k[i, at, j], v[i, at, j]
                p = torch.softmax(kk @ q[i, r, h] * scale + bias[i, h, r, at], 0)
                out[i, r, h] = p @ vv
                if dout is not None:
                    g = dout[i, r, h].double().cpu()
                    ds = p * (vv @ g - g @ out[i, r, h])
                    terms = p * ((vv @ g).abs() + (g @ out[i, r, h]).abs())
                    tq[i, r, h] = scale * (terms @ kk.abs())
                    tk[i, at, j] += scale * terms[:, None] * q[i, r, h].abs()
                    dq[i, r, h] = scale * (ds @ kk)
                    dk[i, at, j] += scale * ds[:, None] * q[i, r, h]
                    dv[i, at, j] += p[:, None] * g
    return out, dq, dk, dv, tq.norm(), tk.norm()


def _close(got, want, tol, what, terms=0.0):
    got = got.detach().double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    err, most = (got - want).norm(), tol * want.norm() + terms
    assert err <= most, f"{what}: off by {err:.2e} of {want.norm():.2e}, {most:.2e} allowed"


def _inputs(b, lq, lk, hq, hk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (1.3 * torch.randn(b, lq, hq, d, generator=g)).to(dtype).cuda()
    k, v = (torch.randn(b, lk, hk, d, generator=g).to(dtype).cuda() for _ in range(2))
    return q, k, v, torch.randn(b, lq, hq, d, generator=g).to(dtype).cuda(), g


def _check(q, k, v, dout, tol=None, **kw):
    """Forward without and with gradients, and the gradients, against the reference."""
    from fovi_amd.arch.attention import cross_attention
    tol = TOL[q.dtype] if tol is None else tol
    plain = cross_attention(q, k, v, **kw)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, **kw)
    grads = torch.autograd.grad(out, leaves, dout)
    want = _reference(q, k, v, kw.get("kv_lengths"), kw.get("mask"), kw.get("scale"), dout)
    _close(plain, want[0], tol, "out without gradients")
    _close(out, want[0], tol, "out")
    for name, got, ref, terms in zip(("dq", "dk", "dv"), grads, want[1:4], (want[4], want[5], 0.0)):
        _close(got, ref, tol, name, TERMS[q.dtype] * terms)
    again = torch.autograd.grad(cross_attention(*leaves, **kw), leaves, dout)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))        # sums in a fixed order
    return out, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,lq,lk,hq,hk,d", [
    (1, 1, 1, 1, 1, 64), (1, 1, 64, 6, 6, 64), (2, 3, 65, 4, 2, 32), (1, 33, 31, 2, 2, 64), (2, 70, 129, 4, 1, 64),
    (1, 128, 128, 2, 2, 128), (1, 5, 300, 8, 2, 80), (1, 257, 40, 1, 1, 96), (2, 31, 33, 3, 3, 16), (1, 2, 2, 2, 1, 8),
    (1, 130, 200, 2, 1, 40), (1, 64, 1, 3, 3, 64), (1, 1, 700, 16, 2, 128), (3, 17, 90, 6, 2, 64),
    (1, 9, 20, 2, 2, 1), (1, 12, 50, 2, 1, 33), (2, 8, 70, 1, 1, 127), (1, 40, 77, 2, 2, 5)])
def test_sizes(b, lq, lk, hq, hk, d, dtype):
    _check(*_inputs(b, lq, lk, hq, hk, d, dtype)[:4])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["heads_first", "kv_pair", "padded", "odd_offset", "element_stride", "expanded", "mixed"])
def test_layouts(layout, dtype):
    b, lq, lk, h, d = 2, 37, 75, 3, 32
    q, k, v, dout, g = _inputs(b, lq, lk, h, h, d, dtype, seed=1)

    def randn(*shape):
        return torch.randn(shape, generator=g).to(dtype).cuda()

    if layout in ("heads_first", "mixed"):
        q = randn(b, h, lq, d).transpose(1, 2)
        if layout == "heads_first":
            k, v = randn(b, h, lk, d).transpose(1, 2), randn(b, h, lk, d).transpose(1, 2)
    elif layout == "kv_pair":
        kv = randn(b, lk, 2, h, d)
        k, v = kv[:, :, 0], kv[:, :, 1]
    elif layout == "padded":
        q, k, v = randn(b, lq, h, d + 8)[..., :d], randn(b, lk + 5, h, d)[:, 5:], randn(b, lk, h + 2, d)[:, :, 1:-1]
    elif layout == "odd_offset":
        q, k, v = (randn(b, n, h, d + 3)[..., 3:] for n in (lq, lk, lk))
    elif layout == "element_stride":
        q, k, v = (randn(b, n, d, h).transpose(2, 3) for n in (lq, lk, lk))
        dout = randn(b, lq, d, h).transpose(2, 3)
    elif layout == "expanded":
        k, v = randn(1, lk, 1, d).expand(b, lk, h, d), randn(b, 1, h, d).expand(b, lk, h, d)
        dout = randn(b, lq, 1, 1).expand(b, lq, h, d)
    out, _ = _check(q, k, v, dout)
    if layout == "heads_first":
        assert out.stride() == q.stride()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq", [1, 4, 45])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (2, 2, 128), (1, 1, 32)])
def test_lengths(lq, hq, hk, d, dtype):
    """Images with no state, one, a few, all; beyond the tensor and below zero. What lies behind a
    length is NaN."""
    q, k, v, dout, _ = _inputs(7, lq, 100, hq, hk, d, dtype, seed=2)
    lengths = torch.tensor([0, 1, 33, 64, 100, 1000, -3])
    for i, n in enumerate(lengths.clamp(0, 100).tolist()):
        k[i, n:], v[i, n:] = float("nan"), float("inf")
    out, (_, dk, dv) = _check(q, k, v, dout, kv_lengths=lengths.int().cuda())
    assert not out[0].any() and not dk[0].any() and not dv[1, 1:].any()
    _check(q, k, v, dout, kv_lengths=lengths.cuda())
    from fovi_amd.arch.attention import cross_attention
    assert not cross_attention(q, k, v, kv_lengths=torch.zeros(7, dtype=torch.int32, device="cuda")).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", ["pairs", "heads", "keys", "full", "rows", "strided"])
@pytest.mark.parametrize("lq,lk,d", [(37, 77, 64), (3, 150, 32), (1, 40, 128)])
def test_boolean_masks(shape, lq, lk, d, dtype):
    b, hq, hk = 2, 4, 2
    q, k, v, dout, g = _inputs(b, lq, lk, hq, hk, d, dtype, seed=3)

    def rand(*size):
        return (torch.rand(size, generator=g) < 0.6).cuda()

    mask = {"pairs": lambda: rand(lq, lk), "heads": lambda: rand(1, hq, lq, lk), "keys": lambda: rand(b, 1, 1, lk),
            "full": lambda: rand(b, hq, lq, lk), "rows": lambda: rand(b, 1, lq, 1),
            "strided": lambda: rand(lk, lq, b).permute(2, 1, 0)[:, None]}[shape]()
    mask = mask.clone(memory_format=torch.preserve_format)
    if shape in ("pairs", "full", "strided"):
        mask[..., ::3, :] = False                       # rows that keep nothing
    out, (dq, _, _) = _check(q, k, v, dout, mask=mask)
    empty = ~mask.expand(b, hq, lq, lk).any(-1).transpose(1, 2)
    assert not out[empty].any() and not dq[empty].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq,lk", [(21, 70), (2, 130)])
def test_bias_masks(lq, lk, dtype):
    """A float bias: ordinary values, the type's lowest value, -inf, a row of each alone."""
    b, h, d = 2, 2, 64
    q, k, v, dout, g = _inputs(b, lq, lk, h, h, d, dtype, seed=4)
    bias = torch.randn(b, 1, lq, lk, generator=g)
    bias[:, :, :, 5::7] = -INF
    bias[:, :, :, 3::5] = torch.finfo(torch.float32).min
    bias[0, :, 0] = -INF
    bias[1, :, 1] = torch.finfo(torch.float32).min       # the lowest value alone: every state the same
    bias = bias.cuda()
    out, _ = _check(q, k, v, dout, mask=bias)
    assert not out[0, 0].any()
    assert ((out[1, 1].double() - v[1].double().mean(0)).norm() / v[1].double().mean(0).norm()) < TOL[dtype]
    half = bias[:, :, :1].bfloat16()
    _check(q, k, v, dout, mask=half)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq,lk,d", [(40, 100, 64), (2, 300, 64), (33, 70, 128), (70, 40, 32)])
@pytest.mark.parametrize("kind", ["bool", "bias"])
def test_non_finite_values_in_masked_places(lq, lk, d, kind, dtype):
    """NaN and infinities in states that no row keeps, in states that some rows leave out, and in
    queries (and their incoming gradients) that keep nothing."""
    b, h = 2, 2
    q, k, v, dout, g = _inputs(b, lq, lk, h, h, d, dtype, seed=5)
    keep = torch.rand(b, 1, lq, lk, generator=g) < 0.7
    keep[:, :, 1] = False
    q[:, 1], dout[:, 1] = float("nan"), float("inf")      # a padded query
    keep[:, :, :, 7] = False
    k[:, 7], v[:, 7] = float("inf"), float("nan")
    mask = keep.cuda() if kind == "bool" else torch.zeros(keep.shape).masked_fill(~keep, -INF).cuda()
    _check(q, k, v, dout, mask=mask)
    # a state whose value is not finite, read by the first row alone: the other rows do not see it
    from fovi_amd.arch.attention import cross_attention
    keep[:, :, :, 9] = False
    keep[:, :, 0, 9] = True
    mask = keep.cuda() if kind == "bool" else torch.zeros(keep.shape).masked_fill(~keep, -INF).cuda()
    clean = v.clone()
    clean[:, 9] = 0
    v[:, 9, :, 0], v[:, 9, :, 1], v[:, 9, :, 2] = float("nan"), INF, -INF
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, mask=mask)
    dout[:, 0] = 0
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    assert out[:, 0, :, 0].isnan().all() and (out[:, 0, :, 1] == INF).all() and (out[:, 0, :, 2] == -INF).all()
    want = _reference(q, k, clean, None, mask, None, dout)
    _close(out[:, 1:], want[0][:, 1:], TOL[dtype], "out of the other rows")
    _close(dq[:, 1:], want[1][:, 1:], TOL[dtype], "dq of the other rows")
    other = [i for i in range(lk) if not bool(keep[:, :, 0, i].any())]
    _close(dv[:, other], want[3][:, other], TOL[dtype], "dv of states that row does not read")
    _close(dk[:, other], want[2][:, other], TOL[dtype], "dk of states that row does not read")


@pytest.mark.gpu
def test_infinite_keys_poison_their_readers_only():
    """A key of infinities (kept) in one image: the other image and the other heads do not change."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, _, _ = _inputs(2, 20, 50, 2, 2, 64, torch.float32, seed=6)
    want = cross_attention(q, k, v)
    k[0, 3, 1, 0] = INF
    out = cross_attention(q, k, v)
    assert torch.equal(out[1], want[1]) and torch.equal(out[0, :, 0], want[0, :, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_scores(dtype):
    """Scores to about +-400: the running maximum, no overflow; rows that read one state. fp32 scores of
    400 are off by 400 * 2^-24 * a few, so 2e-4 is allowed there; bf16 products are exact in fp32."""
    q, k, v, dout, _ = _inputs(1, 40, 130, 2, 2, 64, dtype, seed=7)
    _check(12 * q, k, v, dout, tol=2e-4 if dtype == torch.float32 else 6e-3, scale=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq,hq,hk", [(1, 6, 6), (4, 16, 4), (1, 1, 1), (50, 2, 2)])
def test_many_states(lq, hq, hk, dtype):
    """20000 states: the sums over the states, in parts, against float64 on the GPU."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, dout, _ = _inputs(1, lq, 20000, hq, hk, 64, dtype, seed=8)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, dout)
    ref = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
    kk, vv = (t.repeat_interleave(hq // hk, 2).transpose(1, 2) for t in ref[1:])
    want = (torch.softmax(ref[0].transpose(1, 2) @ kk.transpose(2, 3) / 8, -1) @ vv).transpose(1, 2)
    rgrads = torch.autograd.grad(want, ref, dout.double())
    _close(out, want.detach().cpu(), TOL[dtype], "out")
    _close(cross_attention(q, k, v), want.detach().cpu(), TOL[dtype], "out without gradients")
    for name, a, b in zip(("dq", "dk", "dv"), grads, rgrads):
        _close(a, b.cpu(), TOL[dtype], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_queries_over_few_states(dtype):
    """5000 queries over 70 states: the sums of dk and dv over the queries."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, dout, _ = _inputs(1, 5000, 70, 2, 1, 32, dtype, seed=9)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*leaves), leaves, dout)
    ref = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
    kk, vv = (t.repeat_interleave(2, 2).transpose(1, 2) for t in ref[1:])
    want = (torch.softmax(ref[0].transpose(1, 2) @ kk.transpose(2, 3) * 32 ** -0.5, -1) @ vv).transpose(1, 2)
    for name, a, b in zip(("dq", "dk", "dv"), grads, torch.autograd.grad(want, ref, dout.double())):
        _close(a, b.cpu(), TOL[dtype], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_almost_one_state(dtype):
    """Two states, one of them read nearly alone: dq and dk are small differences. The forward's output
    enters them before its rounding."""
    g = torch.Generator().manual_seed(10)
    q = torch.randn(1, 200, 1, 64, generator=g).to(dtype)
    k = torch.cat([q.mean(1, keepdim=True) * 0, 0.5 * torch.randn(1, 1, 1, 64, generator=g).to(dtype)], 1)
    v, dout = (torch.randn(1, n, 1, 64, generator=g).to(dtype) for n in (2, 200))
    _check(q.cuda(), k.cuda(), v.cuda(), dout.cuda(), scale=1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 40])
def test_offsets_beyond_32_bits(lq):
    """States so far apart that their element offsets pass 2^31."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, dout, _ = _inputs(1, lq, 9, 1, 1, 32, torch.bfloat16, seed=11)
    step = (1 << 28) + 8
    room = torch.empty(8 * step + 64, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(room, (1, 9, 1, 32), (0, step, 32, 1))
    far.copy_(k)
    assert torch.equal(cross_attention(q, far, v), cross_attention(q, k, v))
    far.copy_(v)
    assert torch.equal(cross_attention(q, k, far), cross_attention(q, k, v))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(cross_attention(*leaves), leaves, dout)
    far_v = far.detach().requires_grad_(True)
    got = torch.autograd.grad(cross_attention(leaves[0], leaves[1], far_v), leaves[:2], dout)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 40])
def test_long_rows_beyond_32_bits(lq):
    """150 states almost 32 MiB apart, read where they are: byte offsets to 5 * 10^9, element offsets
    past 2^31, within one tensor."""
    from fovi_amd.arch.attention import _whole, cross_attention
    q, k, v, dout, _ = _inputs(1, lq, 150, 1, 1, 32, torch.bfloat16, seed=15)
    step = (1 << 24) - 8
    room = torch.empty(149 * step + 64, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(room, (1, 150, 1, 32), (0, step, 32, 1))
    far.copy_(k)
    assert _whole(far) and 149 * step > 2 ** 31
    leaves = [t.detach().requires_grad_(True) for t in (q, far, v)]
    out = cross_attention(*leaves)
    assert torch.equal(out, cross_attention(q, k, v))
    near = [t.detach().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(cross_attention(*near), near, dout)
    got = torch.autograd.grad(out, [leaves[0], leaves[2]], dout)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[2])


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences in fp32 with step 2e-2: the second-order error is step^2 / 6 times third
    derivatives of order 1 (7e-5), the rounding 2^-24 * 10 / 4e-2 (2e-5) times a few."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, dout, _ = _inputs(2, 3, 5, 2, 1, 8, torch.float32, seed=12)
    mask = torch.ones(2, 1, 3, 5, dtype=torch.bool, device="cuda")
    mask[0, 0, 1], mask[1, 0, 0, 2] = False, False
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*leaves, mask=mask), leaves, dout)

    def f():
        with torch.no_grad():
            return (cross_attention(*leaves, mask=mask).double() * dout.double()).sum().item()

    for t, gt in zip(leaves, grads):
        flat = t.detach().reshape(-1)
        for i in range(0, flat.numel(), 7):
            x = flat[i].item()
            flat[i] = x + 2e-2
            up = f()
            flat[i] = x - 2e-2
            down = f()
            flat[i] = x
            assert abs((up - down) / 4e-2 - gt.reshape(-1)[i].item()) < 1e-3


@pytest.mark.gpu
def test_empty_tensors():
    from fovi_amd.arch.attention import cross_attention
    def z(b, n, h):
        return torch.randn(b, n, h, 16, device="cuda", requires_grad=True)
    for b, lq, lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0), (0, 0, 0)):
        q, k, v = z(b, lq, 2), z(b, lk, 1), z(b, lk, 1)
        out = cross_attention(q, k, v)
        assert out.shape == (b, lq, 2, 16) and not out.any()
        for g, t in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
            assert g.shape == t.shape and not g.any()


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 50])
def test_streams_and_capture(lq):
    """On a side stream; and captured, replayed with new inputs and with work of its own between."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, _, g = _inputs(2, lq, 3000, 4, 2, 64, torch.bfloat16, seed=13)
    want = cross_attention(q, k, v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = cross_attention(q, k, v)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cross_attention(q, k, v)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g).cuda())
        want = cross_attention(q, k, v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


@pytest.mark.gpu
def test_autocast_takes_bf16():
    from fovi_amd.arch.attention import cross_attention
    q, k, v, _, _ = _inputs(1, 9, 33, 2, 2, 32, torch.float32, seed=14)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = cross_attention(q, k, v)
    assert out.dtype == torch.bfloat16
    assert torch.equal(out, cross_attention(q.bfloat16(), k.bfloat16(), v.bfloat16()))


@pytest.mark.gpu
def test_refusals():
    from fovi_amd.arch.attention import cross_attention
    q, k, v, _, _ = _inputs(2, 5, 7, 4, 2, 16, torch.float32)
    lengths = torch.tensor([3, 7], device="cuda")
    cross_attention(q, k, v, kv_lengths=lengths)
    big = torch.zeros(2, 5, 4, 136, device="cuda")
    mask = torch.ones(5, 7, dtype=torch.bool, device="cuda")
    for args, kw, kind, match in [
            ((q.cpu(), k, v), {}, RuntimeError, "no CPU fallback"), ((q[0], k, v), {}, ValueError, "expected"),
            ((q, k, v[:, :6]), {}, ValueError, "do not fit"), ((q, k[..., :8], v[..., :8]), {}, ValueError, "do not fit"),
            ((q[:, :, :3], k, v), {}, ValueError, "heads"), ((big, big, big), {}, ValueError, "128"),
            ((q.half(), k.half(), v.half()), {}, TypeError, "dtypes"), ((q.bfloat16(), k, v), {}, TypeError, "dtypes"),
            ((q, k, v), {"scale": 0.0}, ValueError, "scale"), ((q, k, v), {"scale": INF}, ValueError, "scale"),
            ((q, k, v), {"kv_lengths": lengths[:1]}, ValueError, "kv_lengths"),
            ((q, k, v), {"kv_lengths": lengths.float()}, ValueError, "kv_lengths"),
            ((q, k, v), {"mask": mask[:, :6]}, ValueError, "mask of shape"),
            ((q, k, v), {"mask": mask.to(torch.uint8)}, TypeError, "mask dtype"),
            ((q, k, v), {"mask": mask.float().requires_grad_(True)}, ValueError, "no gradient"),
            ((q, k, v), {"mask": mask.cpu()}, RuntimeError, "no CPU fallback")]:
        with pytest.raises(kind, match=match):
            cross_attention(*args, **kw)


def test_c_arguments_are_refused():
    lib = _lib.load()
    a = _lib.AttentionArgs()
    assert lib.fovi_attention_fwd(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.q = a.k = a.v = a.out = 16
    a.dtype = 9
    assert lib.fovi_attention_fwd(a, None) != 0 and b"dtype" in lib.fovi_last_error()
    a.dtype = _lib.BF16
    assert lib.fovi_attention_fwd(a, None) != 0 and b"bad sizes" in lib.fovi_last_error()
    a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim = 1, 4, 4, 3, 2, 64
    assert lib.fovi_attention_fwd(a, None) != 0 and b"multiple" in lib.fovi_last_error()
    a.heads, a.head_dim = 4, 129
    assert lib.fovi_attention_fwd(a, None) != 0 and b"head_dim" in lib.fovi_last_error()
    a.head_dim = 64
    assert lib.fovi_attention_fwd(a, None) != 0 and b"scale" in lib.fovi_last_error()
    a.scale, a.mask_kind = 1.0, 3
    assert lib.fovi_attention_fwd(a, None) != 0 and b"mask_kind" in lib.fovi_last_error()
    a.mask_kind = _lib.MASK_KEEP
    assert lib.fovi_attention_fwd(a, None) != 0 and b"null mask" in lib.fovi_last_error()
    b = _lib.AttentionBwdArgs()
    assert lib.fovi_attention_bwd(b, None) != 0 and b"null pointer" in lib.fovi_last_error()


def _pattern(kind, lq, lk):
    i, j = torch.arange(lq)[:, None], torch.arange(lk)[None]
    at = i * lk // lq                                    # the state beside row i
    if kind == "causal":
        return j <= at
    if kind == "band":
        return (j - at).abs() <= 9
    if kind == "blocks":                                 # three groups that see only themselves, 34 rows that see nothing
        return (i * 3 // lq == j * 3 // lk) & ((i < lq // 3) | (i >= lq // 3 + 34))
    return (j >= lk - 5) & (i % 2 == 0)                  # "end": the last states, for every other row


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["causal", "band", "blocks", "end"])
@pytest.mark.parametrize("lq,lk,d", [(150, 333, 64), (301, 140, 32), (131, 260, 128), (2, 1500, 64), (9, 700, 40)])
@pytest.mark.parametrize("as_bias", [False, True])
def test_masks_that_leave_whole_tiles_empty(lq, lk, d, kind, dtype, as_bias):
    b, hq, hk = 1, 4, 2
    q, k, v, dout, g = _inputs(b, lq, lk, hq, hk, d, dtype, seed=11)
    mask = _pattern(kind, lq, lk)
    if as_bias:
        mask = torch.randn(lq, lk, generator=g).masked_fill(~mask, -INF)
    out, (dq, dk, dv) = _check(q, k, v, dout, mask=mask.cuda(), kv_lengths=torch.tensor([lk - 3], device="cuda"))
    keep = _pattern(kind, lq, lk) & (torch.arange(lk) < lk - 3)
    rows, states = ~keep.any(1), ~keep.any(0)
    assert not out[:, rows].any() and not dq[:, rows].any() and not dk[:, states].any() and not dv[:, states].any()


@pytest.mark.gpu
def test_mask_per_head_and_image_of_many_tiles():
    """Patterns that differ by head and image, shared key heads (rows of two heads in one tile)."""
    b, lq, lk, hq, hk, d = 2, 70, 200, 4, 2, 64
    q, k, v, dout, _ = _inputs(b, lq, lk, hq, hk, d, torch.bfloat16, seed=12)
    kinds = ["causal", "band", "end", "blocks", "band", "causal", "causal", "end"]
    mask = torch.stack([_pattern(kind, lq, lk) for kind in kinds]).view(b, hq, lq, lk).cuda()
    _check(q, k, v, dout, mask=mask)
    _check(q[:, :3], k, v, dout[:, :3], mask=mask[:, :, :3])


def test_c_layouts_workspaces_and_masks_are_refused():
    lib = _lib.load()
    a = _lib.AttentionArgs()
    a.q = a.k = a.v = a.out = 4096
    a.dtype, a.scale = _lib.BF16, 0.125
    a.batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim = 1, 4, 100000, 2, 2, 64
    for f in (a.q_stride, a.k_stride, a.v_stride, a.out_stride):
        f[:] = (1 << 30, 128, 64)

    def refused(match, **kw):
        keep = {name: getattr(a, name) for name in kw}
        for name, value in kw.items():
            setattr(a, name, value)
        assert lib.fovi_attention_fwd(a, None) != 0 and match in lib.fovi_last_error(), lib.fovi_last_error()
        for name, value in keep.items():
            setattr(a, name, value)

    refused(b"16-byte", q=4098)
    refused(b"16-byte", head_dim=63)
    a.k_stride[1] = 129
    refused(b"16-byte")
    a.k_stride[1] = 1 << 25                              # 64 MiB of bf16
    refused(b"64 MiB")
    a.k_stride[1] = 128
    refused(b"workspace")
    refused(b"too many", q_len=1 << 40)
    refused(b"too many", batch=1 << 62)
    refused(b"scale", scale=float("nan"))
    need = lib.fovi_attention_fwd_workspace_bytes(1, 4, 100000, 2, 2, 64, _lib.BF16)
    assert need > 0
    refused(b"workspace", workspace=4096, workspace_bytes=need - 1)
    refused(b"workspace", workspace=4104, workspace_bytes=need)
    stride = (C.c_int64 * 4)(0, 0, 0, 1)
    assert lib.fovi_attention_pack_mask(None, stride, 1, 1, 1, 8, 4096, None) != 0 and b"null pointer" in lib.fovi_last_error()
    assert lib.fovi_attention_pack_mask(4096, stride, 1, -1, 1, 8, 4096, None) != 0 and b"bad sizes" in lib.fovi_last_error()
    assert lib.fovi_attention_pack_mask(4096, stride, 1 << 30, 1 << 30, 1, 8, 4096, None) != 0
    assert b"too large" in lib.fovi_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", [_lib.MASK_NONE, _lib.MASK_KEEP, _lib.MASK_BIAS])
@pytest.mark.parametrize("lk,hq,hk,d", [(1, 1, 1, 8), (70, 4, 2, 64), (300, 3, 1, 128)])
def test_no_queries_in_the_c_backward(lk, hq, hk, d, kind, dtype):
    """States without a query: dk and dv are written whole, as zeros, without a workspace. Queries,
    statistics and masks have no element; their pointers have a place of their own all the same."""
    b, lib = 2, _lib.load()
    k = torch.randn(b, lk, hk, d, device="cuda").to(dtype)
    dk, dv = torch.full_like(k, 7.0), torch.full_like(k, 7.0)
    place = torch.zeros(1024, device="cuda")
    a = _lib.AttentionBwdArgs()
    f = a.fwd
    f.q = f.out = f.stats = f.mask = a.dout = a.dq = place.data_ptr()
    if dtype == torch.bfloat16:
        f.out_rest = place.data_ptr()
    f.k = f.v = k.data_ptr()
    f.dtype, f.mask_kind, f.scale = _lib.dtype_code(dtype), kind, 0.125
    f.batch, f.q_len, f.kv_len, f.heads, f.kv_heads, f.head_dim = b, 0, lk, hq, hk, d
    for s in (f.k_stride, f.v_stride, a.dk_stride, a.dv_stride):
        s[:] = k.stride()[:3]
    for s in (f.q_stride, f.out_stride, a.dout_stride, a.dq_stride):
        s[:] = (0, hq * d, d)
    a.dk, a.dv = dk.data_ptr(), dv.data_ptr()
    assert lib.fovi_attention_bwd_workspace_bytes(b, 0, lk, hq, hk, d, f.dtype) == 0
    _lib.check(lib.fovi_attention_bwd(a, _lib.stream_of(k)), "fovi_attention_bwd")
    torch.cuda.synchronize()
    assert not dk.any() and not dv.any() and not place.any()


@pytest.mark.gpu
@pytest.mark.parametrize("constant", [True, False])
def test_differentiating_twice_raises(constant):
    """With a constant incoming gradient and with one that has a gradient itself, in every input; a
    gradient that is only recorded, and not differentiated, is the gradient."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, dout, _ = _inputs(2, 5, 9, 2, 1, 16, torch.float32, seed=20)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dout.requires_grad_(not constant)
    out = cross_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, dout, create_graph=True)
    want = torch.autograd.grad(cross_attention(*leaves), leaves, dout.detach())
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    for g in grads:
        for leaf in leaves + ([] if constant else [dout]):
            with pytest.raises(RuntimeError, match="differentiated once"):
                torch.autograd.grad(cross_attention(*leaves).sum() + dout.sum() + g.square().sum(), leaf, retain_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_raises(which, grad):
    """A tangent of any input, the bias among them, is refused, not dropped; with a level open and no tangent the call
    is the ordinary one."""
    from torch.autograd import forward_ad
    from fovi_amd.arch.attention import cross_attention
    q, k, v, _, g = _inputs(1, 3, 5, 2, 2, 16, torch.float32, seed=21)
    args = [q, k, v, torch.randn(3, 5, generator=g).cuda()]
    want = cross_attention(*args[:3], mask=args[3])
    if grad and which < 3:
        args[which].requires_grad_(True)
    leaf = args[0].detach().requires_grad_(True)
    y = cross_attention(leaf, *args[1:3], mask=args[3])
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(want), torch.ones_like(want)))
    with forward_ad.dual_level():
        assert torch.equal(cross_attention(*args[:3], mask=args[3]), want)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for off in (False, True):
            with torch.set_grad_enabled(not off), pytest.raises(NotImplementedError, match="forward mode"):
                cross_attention(*args[:3], mask=args[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq,lk", [(1, 40), (7, 70), (45, 130), (3, 9000), (45, 3000)])
def test_extreme_biases(lq, lk, dtype):
    """Biases of the size of the type's limits: differences among them count as any others do, and so does one
    state with the largest value; long rows of the lowest value alone, in parts that are joined, read all alike."""
    b, hq, hk, d = 2, 2, 1, 32
    q, k, v, dout, g = _inputs(b, lq, lk, hq, hk, d, dtype, seed=23)
    top = torch.finfo(torch.float32).max
    bias = torch.full((b, hq, lq, lk), -top)
    bias[0, 0] = -2.5e38 - 0.8e38 * torch.rand(lq, lk, generator=g)          # one state of each row is read
    bias[0, 1] = torch.randn(lq, lk, generator=g)
    bias[0, 1, :, lk // 2] = top
    bias[1, 0, :, ::3] = torch.finfo(torch.bfloat16).min                     # a third of the states, alike
    out, _ = _check(q, k, v, dout, mask=bias.cuda())
    want = v[0, :, 0].double().cpu()[bias[0, 0].argmax(-1)]
    assert ((out[0, :, 0].double().cpu() - want).norm() / want.norm()) < TOL[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq,lk", [(2, 40), (45, 130), (2, 9000)])
def test_nan_bias_is_seen(lq, lk, dtype):
    """A bias that is not a number makes its row so, and the gradients that the row enters; other rows stay."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, dout, g = _inputs(1, lq, lk, 2, 2, 32, dtype, seed=24)
    bias = torch.randn(1, 1, lq, lk, generator=g).cuda()
    bad = bias.clone()
    bad[..., 1, lk // 2] = float("nan")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out, clean = cross_attention(*leaves, mask=bad), cross_attention(*leaves, mask=bias)
    rows = [i for i in range(lq) if i != 1]
    assert out[:, 1].isnan().all() and torch.equal(out[:, rows], clean[:, rows])
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    want = torch.autograd.grad(clean, leaves, dout)[0]
    assert dq[:, 1].isnan().all() and torch.equal(dq[:, rows], want[:, rows])
    assert dk.isnan().all() and dv.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["key", "bias"])
@pytest.mark.parametrize("lq,lk", [(2, 40), (45, 130)])
def test_infinite_scores_have_no_gradient_of_zero(lq, lk, kind, dtype):
    """A score of +inf that a row keeps (from a key under a boolean mask, or from a bias) leaves its output NaN, and so its
    gradients, not zeros; rows and states that do not meet it stay as they are."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, dout, g = _inputs(1, lq, lk, 1, 1, 32, dtype, seed=29)
    keep = torch.rand(lq, lk, generator=g) < 0.7
    keep[1, :lk // 2], keep[1, lk // 2:] = True, False    # row 1 reads the first half, others all but state 3
    keep[:, 3] = False
    keep[1, 3] = True
    mask = keep if kind == "key" else torch.zeros(lq, lk).masked_fill(~keep, -INF)
    mask = mask.cuda()
    bad, far = mask.clone(), k.clone()
    if kind == "key":
        far[0, 3] = INF * q[0, 1, 0].sign()
    else:
        bad[1, 3] = INF
    leaves = [t.requires_grad_(True) for t in (q, far, v)]
    out = cross_attention(*leaves, mask=bad)
    rows = [i for i in range(lq) if i != 1]
    mask[:, 3] = False if kind == "key" else -INF
    assert out[:, 1].isnan().all() and torch.equal(out[:, rows], cross_attention(q, k, v, mask=mask)[:, rows])
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    want = torch.autograd.grad(cross_attention(q, leaves[1], v, mask=mask), [q, v], dout)
    assert dq[:, 1].isnan().all() and torch.equal(dq[:, rows], want[0][:, rows])
    assert dk[:, :lk // 2].isnan().all() and dv[:, :lk // 2].isnan().all()
    assert torch.equal(dv[:, lk // 2:], want[1][:, lk // 2:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 65), (45, 33), (150, 127), (3, 1000)])
def test_infinities_at_the_last_place(lq, lk, d, dtype):
    """No mask, and an infinite value in the last state (behind which a tile has nothing more): outputs of that
    element are infinite, not NaN, all others as without it. The same of the last query's incoming gradient and dv."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, dout, _ = _inputs(2, lq, lk, 2, 2, d, dtype, seed=25)
    lengths = torch.tensor([lk, max(1, lk - 30)], device="cuda")
    other = [0] + list(range(2, d))
    want = cross_attention(q, k, v, kv_lengths=lengths)
    far = v.clone()
    for i, n in enumerate(lengths.tolist()):
        far[i, n - 1, :, 1] = INF
    out = cross_attention(q, k, far, kv_lengths=lengths)
    assert (out[..., 1] == INF).all() and torch.equal(out[..., other], want[..., other])
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(cross_attention(*leaves, kv_lengths=lengths), leaves, dout)[2]
    dout[:, -1, :, 1] = -INF
    dv = torch.autograd.grad(cross_attention(*leaves, kv_lengths=lengths), leaves, dout)[2]
    for i, n in enumerate(lengths.tolist()):
        assert (dv[i, :n, :, 1] == -INF).all() and not dv[i, n:].any()
    assert torch.equal(dv[..., other], want[..., other])


@pytest.mark.gpu
def test_learned_bias_without_gradients():
    """A bias that is a parameter (learned elsewhere) is taken where no gradient is asked for."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, _, g = _inputs(1, 5, 9, 2, 2, 16, torch.float32, seed=26)
    bias = torch.nn.Parameter(torch.randn(2, 5, 9, generator=g).cuda())
    want = cross_attention(q, k, v, mask=bias.detach())
    with torch.no_grad():
        assert torch.equal(cross_attention(q, k, v, mask=bias), want)
    with torch.inference_mode():
        assert torch.equal(cross_attention(q, k, v, mask=bias), want)
    with pytest.raises(ValueError, match="no gradient"):
        cross_attention(q, k, v, mask=bias)


def _poison():
    """Leaves NaN in the allocator's free memory, where the next workspaces come from."""
    torch.cuda.synchronize()
    held = [torch.full((1 << 26,), float("nan"), device="cuda")]
    held += [torch.full((1 << n,), float("nan"), device="cuda") for n in range(8, 19) for _ in range(4)]
    torch.cuda.synchronize()
    del held


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["none", "bool", "bias"])
@pytest.mark.parametrize("lq,lk,hq,hk", [(1, 3000, 1, 1), (45, 3000, 2, 1), (45, 3000, 6, 6), (3, 3000, 6, 6), (2, 9000, 2, 1),
                                         (200, 3000, 2, 2)])
def test_lengths_that_end_before_later_parts(lq, lk, hq, hk, kind, dtype):
    """States split over workgroups (joins of fewer than 16 parts and of more) and images that have none, one, one
    part, whole parts and a state, half or all of them: parts that an image does not have are not read."""
    from fovi_amd.arch.attention import cross_attention
    lengths = torch.tensor([0, 1, 128, 513, lk // 2, lk])
    q, k, v, dout, g = _inputs(6, lq, lk, hq, hk, 32, dtype, seed=27)
    mask = None
    if kind != "none":
        mask = torch.rand(lq, lk, generator=g) < 0.8
        mask[lq // 2] = False
        if kind == "bias":
            mask = torch.randn(lq, lk, generator=g).masked_fill(~mask, -INF)
        mask = mask.cuda()
    kw = dict(kv_lengths=lengths.cuda(), mask=mask)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    _poison()
    plain = cross_attention(q, k, v, **kw)
    _poison()
    out = cross_attention(*leaves, **kw)
    _poison()
    grads = torch.autograd.grad(out, leaves, dout)
    want = _reference(q, k, v, lengths, mask, None, dout)
    _close(plain, want[0], TOL[dtype], "out without gradients")
    _close(out, want[0], TOL[dtype], "out")
    for name, got, ref, terms in zip(("dq", "dk", "dv"), grads, want[1:4], (want[4], want[5], 0.0)):
        _close(got, ref, TOL[dtype], name, TERMS[dtype] * terms)
    assert not out[0].any() and not grads[0][0].any()
    for i, n in enumerate(lengths.tolist()):
        assert not grads[1][i, n:].any() and not grads[2][i, n:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq", [2, 50])
def test_capture_with_gradients(lq, dtype):
    """Forward under a mask and backward, captured; replayed with new inputs and with work of its own between."""
    from fovi_amd.arch.attention import cross_attention
    q, k, v, dout, g = _inputs(2, lq, 700, 4, 2, 64, dtype, seed=28)
    mask = (torch.rand(lq, 700, generator=g) < 0.7).cuda()
    lengths = torch.tensor([700, 130], device="cuda", dtype=torch.int32)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        out = cross_attention(*leaves, kv_lengths=lengths, mask=mask)
        return (out.detach(),) + torch.autograd.grad(out, leaves, dout)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        with torch.no_grad():
            for t in leaves + [dout]:
                t.copy_(torch.randn(t.shape, generator=g))
            lengths.copy_(torch.tensor([700 - 100 * i, 33 * i]))
            mask.copy_(torch.rand(mask.shape, generator=g) < 0.7)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
