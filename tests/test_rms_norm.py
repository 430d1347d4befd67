"""RMS norm, with the residual's addition and with rows in 8 bits, against float64.

Tolerances, from the arithmetic. u is half a step of the rows' type, relative: 2^-24 (fp32) or 2^-8 (bf16). The mean of
squares is a sum of up to C positive terms, each addition off by 2^-24 of it at most; the root halves that, and a handful of
products follow: a value is off by (C / 2 + 8) 2^-24 of itself, plus u for its rounding. The sum with the residual is
rounded once, and what follows is compared on the rounded sum. Gradients: dx = dtotal + rstd (g - h mean(g h)); the mean is a
sum of C terms of either sign, off by (C + 8) 2^-24 of the mean of |g h|.  A weight gradient is a sum over the rows: off by
(rows + C / 2 + 8) 2^-24 of the sum of |dy h|.
"""
import ctypes as C
import shutil

import pytest
import torch

from fovi_amd import _lib
from tests.test_abi import _c_layout

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24


def _data(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, r, dy, dt = (torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(4))
    w = (1 + 0.2 * torch.randn(shape[-1], generator=g)).cuda()
    return x, r, w, dy, dt


def _within(got, want, bound, what):
    over = ((got.detach().double().cpu() - want).abs() - bound).max().item() if want.numel() else 0.0
    assert got.shape == want.shape and over <= 0, f"{what}: {over:.3e} over the bound"


def _check(x, r, w, dy, dt, y, total, dx, dw, eps=1e-6):
    """y, total and the gradients (each may be None) against float64."""
    c, u = x.shape[-1], U[x.dtype]
    t = x.detach().double().cpu() + (0 if r is None else r.detach().double().cpu())
    if r is not None:
        _within(total, t, u * t.abs() * (1 + 2.0 ** -20), "total")
        t = total.detach().double().cpu()
    wd = torch.ones(c, dtype=torch.float64) if w is None else w.detach().double().cpu()
    rstd = 1 / (t.square().mean(-1, keepdim=True) + eps).sqrt()
    h = t * rstd
    rel = (c / 2 + 8) * E
    want = h * wd
    if y is not None:
        _within(y, want, (u + rel) * 1.001 * want.abs() + 1e-38, "y")
    if dx is None and dw is None:
        return
    d = dy.detach().double().cpu()
    g = d * wd
    mean = (g * h).mean(-1, keepdim=True)
    want = rstd * (g - h * mean) + (0 if dt is None else dt.detach().double().cpu())
    slack = rstd * (g.abs() * rel + h.abs() * ((g * h).abs().mean(-1, keepdim=True) * (c + 8) * E + mean.abs() * 2 * rel)) + \
        4 * E * (rstd * (g.abs() + (h * mean).abs()))
    if dx is not None:
        _within(dx, want, (u * want.abs() + slack) * 1.01 + 1e-38, "dx")
    if dw is not None:
        uw = U[dw.dtype]
        want = (d * h).reshape(-1, c).sum(0)
        rows = d.numel() // c
        bound = (d * h).abs().reshape(-1, c).sum(0) * (rows + c / 2 + 8) * E
        _within(dw, want, (uw * want.abs() + bound) * 1.01 + 1e-38, "dw")


SHAPES = [(1, 1), (3, 2), (1, 17), (5, 64), (64, 384), (257, 384), (33, 771), (7, 1000), (4100, 7), (4097, 385), (4099, 61),
          (20, 1537), (5, 4095), (3, 8191), (2, 8192), (2, 9001), (3, 20000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,c", SHAPES)
def test_values_and_gradients(rows, c, dtype, residual):
    from fovi_amd.arch.norm import rms_norm
    x, r, w, dy, dt = _data((rows, c), dtype)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)] + ([r.requires_grad_(True)] if residual else [])
    if residual:
        y, total = rms_norm(x, w, residual=r)
        dx, dw, dr = torch.autograd.grad((y, total), leaves, (dy, dt))
        assert torch.equal(dx, dr)
        _check(x, r, w, dy, dt, y, total, dx, dw)
    else:
        y = rms_norm(x, w)
        dx, dw = torch.autograd.grad(y, leaves, dy)
        _check(x, None, w, dy, None, y, None, dx, dw)
    with torch.no_grad():
        again = rms_norm(x, w, residual=r if residual else None)
    assert torch.equal(again[0] if residual else again, y)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [40, 771, 9000])
@pytest.mark.parametrize("which", ["none", "bf16", "frozen", "only_y", "only_total", "only_residual"])
def test_parameters_and_parts(c, which):
    """Without a weight, with one in bf16 beside fp32 rows, with parts of the gradients asked for, and with a gradient that
    reaches one of the two results only."""
    from fovi_amd.arch.norm import rms_norm
    x, r, w, dy, dt = _data((9, c), torch.float32, 3)
    w = {"none": None, "bf16": w.bfloat16()}.get(which, w)
    x.requires_grad_(which != "only_residual")
    r.requires_grad_(which == "only_residual")
    if w is not None and which != "frozen":
        w.requires_grad_(True)
    y, total = rms_norm(x, w, residual=r)
    leaves = [t for t in (x, w, r) if t is not None and t.requires_grad]
    outs, grads = (y, total), (dy, dt)
    if which == "only_y":
        outs, grads = (y,), (dy,)
    if which == "only_total":
        outs, grads = (total,), (dt,)
    got = dict(zip([id(t) for t in leaves], torch.autograd.grad(outs, leaves, grads, allow_unused=True)))
    d = torch.zeros_like(dy) if which == "only_total" else dy
    e = None if which == "only_y" else dt
    dx = got.get(id(x), got.get(id(r)))
    _check(x, r, w, d, e, y, total, dx, got.get(id(w)) if w is not None else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_gradient_that_does_not_arrive_is_not_read(dtype, monkeypatch):
    """Only y's gradient: the kernel is given none of total's, and the rows are those of one of zeros. Only total's: it is the rows'
    gradient, without a kernel, and the weight's is zero. Neither: zeros."""
    from fovi_amd.arch import norm
    x, r, w, dy, dt = _data((300, 40), dtype, 13)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    calls, launch = [], _lib.launch
    monkeypatch.setattr(_lib, "launch", lambda entry, args, t, what: calls.append((what, args[0].dtotal)) or launch(entry, args, t, what))
    y, total = norm.rms_norm(x, w, residual=r)
    want = torch.autograd.grad((y, total), leaves, (dy, torch.zeros_like(dt)), retain_graph=True)
    assert calls[-1][0] == "fovi_rms_norm_bwd" and calls[-1][1] is not None
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert calls[-1] == ("fovi_rms_norm_bwd", None) and all(torch.equal(a, b) for a, b in zip(got, want))
    n = len(calls)
    dx, dr, dw = torch.autograd.grad(total, leaves, dt, retain_graph=True)
    assert len(calls) == n and torch.equal(dx, dt) and torch.equal(dr, dt) and dw.shape == w.shape and not dw.any()

    class Nothing(torch.autograd.Function):
        @staticmethod
        def forward(ctx, *args):
            return args[0].sum()

        @staticmethod
        def backward(ctx, g):
            return None, None

    assert not any(g.any() for g in torch.autograd.grad(Nothing.apply(y, total), leaves, retain_graph=True))
    assert len(calls) == n
    for g in torch.autograd.grad(total, leaves, dt.requires_grad_(True), create_graph=True):
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(g.sum(), [dt, x], allow_unused=True, retain_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["tokens", "padded", "odd_offset", "channels_first", "four_dims", "expanded", "one_dim"])
def test_layouts(layout, dtype):
    """Rows where they are, with a residual and gradients of other layouts; the values of the contiguous call."""
    from fovi_amd.arch.norm import rms_norm, rms_norm_int8
    g = torch.Generator().manual_seed(5)

    def rows(kind):
        make = {"tokens": lambda: torch.randn(3, 9, 40, generator=g)[:, 2:7], "padded": lambda: torch.randn(3, 5, 48, generator=g)[..., :40],
                "odd_offset": lambda: torch.randn(3, 5, 47, generator=g)[..., 3:43],
                "channels_first": lambda: torch.randn(3, 40, 5, generator=g).transpose(1, 2),
                "four_dims": lambda: torch.randn(3, 7, 5, 40, generator=g)[:, 3], "expanded": lambda: torch.randn(1, 5, 40, generator=g).expand(3, 5, 40),
                "one_dim": lambda: torch.randn(40, generator=g)}[kind]
        t = make()
        return t.to(dtype).cuda() if t.is_contiguous() else torch.empty_strided(t.shape, t.stride(), dtype=dtype, device="cuda").copy_(t) \
            if 0 not in t.stride() else t[:1].to(dtype).cuda().expand(t.shape)

    other = "one_dim" if layout == "one_dim" else "tokens" if layout != "tokens" else "channels_first"
    x, r, dy, dt = rows(layout), rows(other), rows(other), rows(layout)
    w = torch.randn(40, generator=g).cuda()

    def run(x, r, dy, dt):
        x, r, v = x.detach().requires_grad_(True), r.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y, total = rms_norm(x, v, residual=r)
        q, total8 = rms_norm_int8(x.detach(), w, residual=r.detach())
        alone = rms_norm(x, v)
        return (y, total, q.data, q.scale, total8, alone) + torch.autograd.grad((y, total, alone), (x, r, v), (dy, dt, dy))

    got, want = run(x, r, dy, dt), run(*(t.contiguous() for t in (x, r, dy, dt)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _eight_bits(y, q, scale, c):
    """The rows in 8 bits against the unrounded y (float64): half a step and what fp32 loses."""
    top = y.abs().amax(-1)
    rel = (c / 2 + 16) * E
    _within(scale, top / 127, top / 127 * rel + 2.0 ** -149, "scale")
    s = scale.double().cpu()
    _within(q.double() * s.cuda()[..., None], y, (0.5 * s[..., None] + 2 * rel * top[..., None]) * 1.0001 + 2.0 ** -149, "values")
    assert q.abs().max() <= 127
    assert (q.abs().amax(-1).cpu()[top > 2.0 ** -120] == 127).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c", SHAPES)
def test_rows_in_8_bits(rows, c, dtype):
    from fovi_amd.arch.int8 import quantize_int8
    from fovi_amd.arch.norm import rms_norm_int8
    x, r, w, _, _ = _data((rows, c), dtype, 7)
    q, total = rms_norm_int8(x, w, residual=r)
    _check(x, r, w, None, None, None, total, None, None)
    t = total.double().cpu()
    _eight_bits(t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double().cpu(), q.data, q.scale, c)
    alone = rms_norm_int8(total, w)
    assert torch.equal(alone.data, q.data) and torch.equal(alone.scale, q.scale)
    p = quantize_int8(x)
    _eight_bits(x.double().cpu(), p.data, p.scale, c)
    for dt in (torch.float32, torch.bfloat16):
        want = (p.data.float() * p.scale[:, None]).to(dt)
        assert torch.equal(p.dequantize(dt), want)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [5, 64, 9000])
def test_extreme_rows_in_8_bits(c):
    """Zeros, numbers near both ends of fp32, infinities and NaN, each in rows of their own."""
    from fovi_amd.arch.int8 import quantize_int8
    x = torch.randn(10, c, generator=torch.Generator().manual_seed(1)).cuda()
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e-37 / x[2].abs().max()
    x[3] *= 1e-41 / x[3].abs().max()
    x[4] *= 3e38 / x[4].abs().max()
    x[5, c // 2] = float("inf")
    x[6, c - 1] = float("-inf")
    x[7, 0] = float("nan")
    x[8] = 2.0 ** -149
    q = quantize_int8(x)
    fine = [0, 1, 2, 3, 4, 8, 9]
    xd, s = x.double().cpu(), q.scale.double().cpu()
    values = q.dequantize().double().cpu()
    for i in fine:
        top = xd[i].abs().max()
        assert abs(s[i] - top / 127) <= top / 127 * 2 * E + 2.0 ** -149
        # a step below the smallest numbers is rounded to a whole multiple of 2^-149: 127 of them are off by 63.5
        assert ((values[i] - xd[i]).abs() <= 0.5 * s[i] * 1.0001 + 127 * 2.0 ** -149).all(), i
    for i in (5, 6, 7):
        assert values[i].isnan().all() and not s[i].isfinite()
        assert (q.data[i] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [4e17, 3e19, 1e30, 1e36])
@pytest.mark.parametrize("rows,c", [(5, 40), (4099, 1024), (3, 8192), (2, 9001)])
def test_large_rows(rows, c, top, dtype):
    """Rows whose sum of squares is past fp32's range, beside others: the norm is that of the formula, in both directions and in
    8 bits. (Their 1 / sqrt is a normal number, as the bounds assume.)"""
    from fovi_amd.arch.norm import rms_norm, rms_norm_int8
    x, r, w, dy, dt = _data((rows, c), dtype, 23)
    x[1::2] *= top
    dy[1::2] *= min(top, 1e30)                                       # (g h is summed in fp32 too)
    dt.zero_()
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    y, total = rms_norm(x, w, residual=r)
    assert y.isfinite().all() and (y[1].abs().amax() > 0.5)
    dx, dw, _ = torch.autograd.grad((y, total), leaves, (dy, dt))
    _check(x, r, w, dy, dt, y, total, dx, dw)
    with torch.no_grad():
        q, total = rms_norm_int8(x, w, residual=r)
    t = total.double().cpu()
    _eight_bits(t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.detach().double().cpu(), q.data, q.scale, c)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [3, 384, 9001])
def test_the_largest_rows(c):
    """Rows of the type's largest value: 1 / sqrt of their mean of squares, 2^-128, has 22 bits."""
    from fovi_amd.arch.norm import rms_norm
    for dtype in (torch.float32, torch.bfloat16):
        y = rms_norm(torch.full((2, c), torch.finfo(dtype).max, dtype=dtype, device="cuda"), torch.full((c,), 3.0, device="cuda"), eps=0.0)
        assert ((y.double() - 3).abs() <= 3 * (2.0 ** -22 + (c / 2 + 8) * E + U[dtype])).all()


@pytest.mark.gpu
def test_infinities_stay_in_their_rows():
    from fovi_amd.arch.norm import rms_norm
    x, r, w, dy, dt = _data((6, 48), torch.float32, 9)
    want = rms_norm(x, w, residual=r)
    bad = x.clone()
    bad[1, 3], bad[4, 0] = float("nan"), float("inf")
    got = rms_norm(bad, w, residual=r)
    keep = [0, 2, 3, 5]
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])
    assert got[0][1].isnan().all() and got[0][4, 0].isnan() and (got[0][4, 1:] == 0).all()


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the float64 formula that the kernels are held to, in a few directions."""
    from fovi_amd.arch.norm import rms_norm
    x, r, w, dy, dt = _data((4, 33), torch.float32, 11)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    grads = torch.autograd.grad(rms_norm(x, w, residual=r), leaves, (dy, dt))

    def loss(x, r, w):
        t = x + r
        return (t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w * dy.double()).sum() + (t * dt.double()).sum()

    base = [t.detach().double() for t in leaves]
    for i in range(3):
        v = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
        h = 1e-5
        at = [[t + s * h * v if j == i else t for j, t in enumerate(base)] for s in (1, -1)]
        want = ((loss(*at[0]) - loss(*at[1])) / (2 * h)).item()
        assert abs((grads[i].double() * v).sum().item() - want) < 1e-4 * max(1.0, abs(want))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 16), (3, 0, 16)])
def test_empty_inputs(shape):
    from fovi_amd.arch.int8 import quantize_int8
    from fovi_amd.arch.norm import rms_norm, rms_norm_int8
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y, total = rms_norm(x, w, residual=torch.zeros(shape, device="cuda"))
    assert y.shape == total.shape == x.shape
    (y.sum() + total.sum()).backward()
    assert x.grad.shape == x.shape and (w.grad == 0).all()
    with torch.no_grad():
        q, total = rms_norm_int8(x, w, residual=x)
        assert q.data.shape == shape and q.scale.shape == shape[:-1] and total.shape == shape
        assert quantize_int8(x).dequantize().shape == shape


@pytest.mark.gpu
def test_module_and_stream():
    from fovi_amd.arch.norm import RMSNorm, rms_norm
    m = RMSNorm(40)
    x = torch.randn(300, 40, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, total = m(x, residual=x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, rms_norm(x + x, m.weight)) and torch.equal(total, x + x)
    assert "40" in repr(m) and RMSNorm(8, elementwise_affine=False).weight is None


@pytest.mark.gpu
def test_refusals():
    from fovi_amd.arch.int8 import Int8Rows, quantize_int8
    from fovi_amd.arch.norm import rms_norm, rms_norm_int8
    x = torch.zeros(4, 16, device="cuda")
    with pytest.raises(TypeError, match="dtype"):
        rms_norm(x.half())
    with pytest.raises(ValueError, match="weight of shape"):
        rms_norm(x, torch.ones(15, device="cuda"))
    with pytest.raises(TypeError, match="weight dtype"):
        rms_norm(x, torch.ones(16, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError, match="eps"):
        rms_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="C >= 1"):
        rms_norm(torch.zeros(4, 0, device="cuda"))
    with pytest.raises(ValueError, match="residual of shape"):
        rms_norm(x, residual=x[:2])
    with pytest.raises(TypeError, match="residual is"):
        rms_norm(x, residual=x.bfloat16())
    leaf = x.clone().requires_grad_(True)
    for call in (lambda: rms_norm_int8(leaf), lambda: rms_norm_int8(x, residual=leaf), lambda: quantize_int8(leaf)):
        with pytest.raises(ValueError, match="no gradients"):
            call()
    with pytest.raises(TypeError, match="int8 rows"):
        Int8Rows(x, x[:, 0]).dequantize()
    with pytest.raises(ValueError, match="scales"):
        Int8Rows(x.to(torch.int8), x[:2, 0]).dequantize()
    with pytest.raises(TypeError, match="dtype"):
        quantize_int8(x).dequantize(torch.float16)
    with pytest.raises(TypeError, match="dtype"):
        quantize_int8(x.half())


def test_cpu_tensors_and_c_arguments_are_refused():
    from fovi_amd.arch.int8 import Int8Rows, quantize_int8
    from fovi_amd.arch.norm import rms_norm, rms_norm_int8
    x = torch.zeros(2, 4)
    for call in (lambda: rms_norm(x), lambda: rms_norm_int8(x), lambda: quantize_int8(x),
                 lambda: Int8Rows(x.to(torch.int8), x[:, 0]).dequantize()):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    lib = _lib.load()
    a = _lib.RmsNormArgs()
    assert lib.fovi_rms_norm_fwd(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.x, a.dtype = 16, 7
    assert lib.fovi_rms_norm_fwd(a, None) != 0 and b"dtypes" in lib.fovi_last_error()
    a.dtype, a.rows0, a.rows1 = _lib.F32, 1, 1
    assert lib.fovi_rms_norm_fwd(a, None) != 0 and b"bad sizes" in lib.fovi_last_error()
    a.channels, a.eps = 8, -1.0
    assert lib.fovi_rms_norm_fwd(a, None) != 0 and b"eps" in lib.fovi_last_error()
    a.eps = 1e-5
    assert lib.fovi_rms_norm_fwd(a, None) != 0 and b"either y" in lib.fovi_last_error()
    a.y, a.residual = 16, 16
    assert lib.fovi_rms_norm_fwd(a, None) != 0 and b"total with residual" in lib.fovi_last_error()
    assert lib.fovi_rms_norm_bwd(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.dy, a.rstd, a.dweight = 16, 16, 16
    assert lib.fovi_rms_norm_bwd(a, None) != 0 and b"workspace" in lib.fovi_last_error()
    assert lib.fovi_rms_norm_workspace_bytes(0, 8) == 0
    stride = (C.c_int64 * 2)(0, 8)
    assert lib.fovi_quantize_rows(None, _lib.F32, 1, 1, 8, stride, 16, 16, None) != 0 and b"null" in lib.fovi_last_error()
    assert lib.fovi_quantize_rows(16, 9, 1, 1, 8, stride, 16, 16, None) != 0 and b"dtype" in lib.fovi_last_error()
    assert lib.fovi_quantize_rows(16, _lib.F32, 1, 1, 0, stride, 16, 16, None) != 0 and b"bad sizes" in lib.fovi_last_error()
    assert lib.fovi_dequantize_rows(16, 16, 1, 0, 8, 16, _lib.F32, None) != 0 and b"bad sizes" in lib.fovi_last_error()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("py,c", [(_lib.RmsNormArgs, "fovi_rms_norm_args"), (_lib.LinearInt8Args, "fovi_linear_int8_args"),
                                  (_lib.GatedMlpArgs, "fovi_gated_mlp_args")])
def test_struct_layout_matches_header(py, c, tmp_path):
    fields = [f for f, _ in py._fields_]
    size, offs = _c_layout(c, fields, tmp_path)
    assert C.sizeof(py) == size
    for f, off in zip(fields, offs):
        assert getattr(py, f).offset == off, f


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c", [(5, 3), (4099, 13), (9, 385), (2, 1030), (2, 20001)])
def test_writes_its_rows_only(rows, c, dtype):
    """Outputs inside larger buffers: what lies in front and behind keeps its value."""
    x, r, w, dy, dt = _data((rows, c), dtype)
    lib, n = _lib.load(), rows * c
    t, y, dx = (torch.full((n + 32,), 7.0, dtype=dtype, device="cuda") for _ in range(3))
    q = torch.full((n + 32,), 7, dtype=torch.int8, device="cuda")
    scale, rstd = (torch.full((rows + 32,), 7.0, device="cuda") for _ in range(2))
    es = x.element_size()
    a = _lib.RmsNormArgs()
    a.x, a.residual, a.dtype, a.rows0, a.rows1, a.channels, a.eps = x.data_ptr(), r.data_ptr(), _lib.dtype_code(dtype), 1, rows, c, 1e-6
    a.weight, a.p_dtype = w.data_ptr(), _lib.F32
    a.x_stride[:] = a.residual_stride[:] = a.dy_stride[:] = a.dtotal_stride[:] = (0, c)
    a.total, a.y, a.rstd = t.data_ptr() + 16 * es, y.data_ptr() + 16 * es, rstd.data_ptr() + 64
    _lib.check(lib.fovi_rms_norm_fwd(a, _lib.stream_of(x)), "forward")
    a.y, a.q, a.scale = None, q.data_ptr() + 16, scale.data_ptr() + 64
    _lib.check(lib.fovi_rms_norm_fwd(a, _lib.stream_of(x)), "forward in 8 bits")
    a.x, a.dy, a.dtotal, a.dx = a.total, dy.data_ptr(), dt.data_ptr(), dx.data_ptr() + 16 * es
    _lib.check(lib.fovi_rms_norm_bwd(a, _lib.stream_of(x)), "backward")
    _check(x, r, w, dy, dt, y[16:16 + n].view(rows, c), t[16:16 + n].view(rows, c), dx[16:16 + n].view(rows, c), None)
    for b, m in ((t, n), (y, n), (dx, n), (q, n), (scale, rows), (rstd, rows)):
        assert (b[:16] == 7).all() and (b[16 + m:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("constant", [True, False])
def test_differentiating_twice_raises(constant):
    from fovi_amd.arch.norm import rms_norm
    x, r, w, dy, dt = _data((7, 40), torch.float32, 20)
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    dy.requires_grad_(not constant)
    grads = torch.autograd.grad(rms_norm(x, w, residual=r), leaves, (dy, dt), create_graph=True)
    want = torch.autograd.grad(rms_norm(x, w, residual=r), leaves, (dy.detach(), dt))
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    for got in grads:
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(got.square().sum(), w, retain_graph=True, allow_unused=True)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
def test_forward_mode_raises(which):
    from torch.autograd import forward_ad
    from fovi_amd.arch.norm import rms_norm, rms_norm_int8
    args = [torch.randn(s, device="cuda") for s in ((4, 24), (24,), (4, 24))]
    want = rms_norm(args[0], args[1], residual=args[2])
    with forward_ad.dual_level():
        got = rms_norm(args[0], args[1], residual=args[2])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for off in (False, True):
            with torch.set_grad_enabled(not off), pytest.raises(NotImplementedError, match="forward mode"):
                rms_norm(args[0], args[1], residual=args[2])
        with pytest.raises(ValueError, match="forward-mode"):
            rms_norm_int8(args[0], args[1], residual=args[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c", [(5, 48), (5000, 385), (9, 20000)])
def test_capture(rows, c, dtype):
    """Forward, backward and the 8-bit form captured; replayed with new inputs and with work of its own between."""
    from fovi_amd.arch.norm import rms_norm, rms_norm_int8
    x, r, w, dy, dt = _data((rows, c), dtype, 21)
    leaves = [t.requires_grad_(True) for t in (x, w, r)]

    def step():
        y, total = rms_norm(x, w, residual=r)
        with torch.no_grad():
            q, _ = rms_norm_int8(x, w, residual=r)
        return (y.detach(), total.detach(), q.data, q.scale, q.dequantize()) + torch.autograd.grad((y, total), leaves, (dy, dt))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    g = torch.Generator().manual_seed(22)
    for i in range(4):
        with torch.no_grad():
            for t in leaves + [dy, dt]:
                t.copy_(torch.randn(t.shape, generator=g))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows of more than 2^31 elements in all; only the last have an incoming gradient, so that the weight's comes from them."""
    from fovi_amd.arch.norm import rms_norm, rms_norm_int8
    m, c, last = 2 ** 21 + 70, 1024, 70
    x, r, w, dy, dt = _data((last, c), torch.bfloat16)

    def behind(t, value):
        rows = torch.full((m, c), value, device="cuda", dtype=torch.bfloat16)
        rows[-last:] = t
        return rows

    leaves = [behind(x, 1.0).requires_grad_(True), w.requires_grad_(True), behind(r, 0.5).requires_grad_(True)]
    y, total = rms_norm(leaves[0], leaves[1], residual=leaves[2])
    dx, dw, dr = torch.autograd.grad((y, total), leaves, (behind(dy, 0.0), behind(dt, 0.0)))
    _check(x, r, w, dy, dt, y[-last:], total[-last:], dx[-last:], dw)
    assert not dx[:-last].any() and torch.equal(dr[-last:], dx[-last:])
    with torch.no_grad():
        q, again = rms_norm_int8(leaves[0], leaves[1], residual=leaves[2])
    assert torch.equal(again, total)
    values, scale = q.dequantize()[-last:].double(), q.scale[-last:, None].double()
    y = y[-last:].detach().double()
    assert ((values - y).abs() <= 0.501 * scale + 1.01 * U[torch.bfloat16] * y.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("c", [2 ** 27 + 24, 2 ** 30])
def test_the_widest_weight_gradients(c):
    """Columns for which a launch along one dimension would have 2^32 threads or more (32 for each in the join, 4 in the sums)."""
    from fovi_amd.arch.norm import rms_norm
    x, dy = (torch.zeros(1, c, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    w = torch.ones(c, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    at = torch.tensor([0, 2 ** 23, 2 ** 27 - 1, c - 1], device="cuda")
    x[0, at], dy[0, at] = 2.0 ** 13, torch.tensor([1.0, 2.0, 3.0, 4.0], device="cuda").bfloat16()
    (dw,) = torch.autograd.grad(rms_norm(x, w, eps=0.0), w, dy)
    h = (c / 4) ** 0.5                                     # the root mean square is 2^13 (4 / c)^0.5
    assert torch.equal(dw[at], (dy[0, at].double() * h).bfloat16()) and dw.count_nonzero() == 4
