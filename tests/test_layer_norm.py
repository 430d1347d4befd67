"""Layer norm forward and backward against float64, over types, widths, layouts and row counts.

Tolerances, from the arithmetic: fp32 outputs and gradients carry a few roundings of 2^-24 and sums
of up to a few thousand terms (error growth about sqrt(n) * 2^-24): 2e-6 relative. bf16 outputs are
rounded once, at most 2^-9 of each value: 2^-9 in the norm, with 5% for the fp32 part; the weight
gradients of bf16 rows are fp32 sums of exact products, so they keep 2e-6.
"""
import ctypes as C
import shutil

import pytest
import torch

from fovi_amd import _lib
from tests.test_abi import _c_layout

F32_TOL, BF16_TOL = 2e-6, 2.05e-3


def _reference(x, w, b, eps, dy=None):
    """(y, dx, dw, db) in float64."""
    x = x.detach().double().cpu()
    c = x.shape[-1]
    w = torch.ones(c, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(c, dtype=torch.float64) if b is None else b.detach().double().cpu()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    h = (x - mean) * rstd
    y = h * w + b
    if dy is None:
        return y, None, None, None
    dy = dy.double().cpu()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return y, dx, (dy * h).reshape(-1, c).sum(0), dy.reshape(-1, c).sum(0)


def _close(got, want, tol, what):
    got = got.detach().double().cpu()
    err = (got - want).norm() / want.norm().clamp_min(1e-30)
    assert torch.isfinite(got).all() and err <= tol, f"{what}: {err:.2e} > {tol:.1e}"


def _data(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * 1.5 + 0.3
    return x.to(dtype).cuda(), torch.randn(shape, generator=g).to(dtype).cuda(), g


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 2), (1, 17), (5, 64), (64, 384), (257, 384), (33, 771), (7, 1000),
                                    (130, 1024), (9, 2047), (6, 4096), (3, 4099), (2, 8192), (2, 16385), (1, 40000),
                                    (4096, 24), (3001, 8)])
def test_values_and_gradients(rows, c, dtype):
    from fovi_amd.arch.norm import layer_norm
    x, dy, g = _data((rows, c), dtype)
    w, b = (1 + 0.2 * torch.randn(c, generator=g)).cuda(), (0.2 * torch.randn(c, generator=g)).cuda()
    y0 = layer_norm(x, w, b)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    assert y.dtype == dtype and torch.equal(y, y0)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    ry, rdx, rdw, rdb = _reference(x, w, b, 1e-5, dy)
    tol = F32_TOL if dtype == torch.float32 else BF16_TOL
    _close(y, ry, tol, "y")
    if c > 2:             # of one or two channels the exact gradient is (nearly) zero: all cancellation
        _close(dx, rdx, tol, "dx")
        _close(dw, rdw, F32_TOL, "dw")
    _close(db, rdb, F32_TOL, "db")
    again = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))      # sums in a fixed order


@pytest.mark.gpu
@pytest.mark.parametrize("c", [40, 384, 771, 5000])
@pytest.mark.parametrize("params", ["none", "weight", "bias", "bf16"])
def test_parameters_of_each_kind(c, params):
    from fovi_amd.arch.norm import layer_norm
    x, dy, g = _data((37, c), torch.bfloat16, seed=3)
    w = b = None
    if params in ("weight", "bf16"):
        w = (1 + 0.2 * torch.randn(c, generator=g)).cuda()
    if params in ("bias", "bf16"):
        b = (0.2 * torch.randn(c, generator=g)).cuda()
    if params == "bf16":
        w, b = w.bfloat16(), b.bfloat16()
    leaves = [t if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    wrt = [t for t in leaves if t is not None]
    grads = list(torch.autograd.grad(y, wrt, dy))
    ry, rdx, rdw, rdb = _reference(x, w, b, 1e-5, dy)
    _close(y, ry, BF16_TOL, "y")
    _close(grads.pop(0), rdx, BF16_TOL, "dx")
    tol = BF16_TOL if params == "bf16" else F32_TOL
    if w is not None:
        _close(grads.pop(0), rdw, tol, "dw")
    if b is not None:
        _close(grads.pop(0), rdb, tol, "db")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["tokens", "padded", "odd_offset", "channels_first", "four_dims", "expanded"])
def test_layouts(layout, dtype):
    """Rows that are slices, padded, not 16-byte aligned, channel planes, split heads, broadcast;
    the incoming gradient in another layout than the rows."""
    from fovi_amd.arch.norm import layer_norm
    c = 48
    g = torch.Generator().manual_seed(7)

    def randn(*shape):
        return torch.randn(shape, generator=g).to(dtype).cuda()

    x = {"tokens": lambda: randn(5, 20, c)[:, 3:], "padded": lambda: randn(6, 9, c + 16)[..., :c],
         "odd_offset": lambda: randn(6, 9, c + 3)[..., 3:], "channels_first": lambda: randn(4, c, 11).transpose(1, 2),
         "four_dims": lambda: randn(3, 7, 2, 5, c).transpose(1, 3)[:, ::2],
         "expanded": lambda: randn(1, 13, c).expand(4, 13, c)}[layout]()
    w, b = torch.randn(c, generator=g).cuda(), torch.randn(c, generator=g).cuda()
    dy = randn(*x.shape)
    for grad in (dy, dy.transpose(0, 1).contiguous().transpose(0, 1), dy[..., :1].expand(dy.shape)):
        leaf = x.detach().requires_grad_(True)
        y = layer_norm(leaf, w, b)
        (dx,) = torch.autograd.grad(y, leaf, grad)
        ry, rdx, _, _ = _reference(x, w, b, 1e-5, grad)
        tol = F32_TOL if dtype == torch.float32 else BF16_TOL
        _close(y, ry, tol, "y")
        _close(dx, rdx, tol, "dx")


@pytest.mark.gpu
def test_many_rows_sum_in_32_bits():
    """70001 rows of 24 channels: the weight gradients' long sums; rows beyond one grid."""
    from fovi_amd.arch.norm import layer_norm
    x, dy, g = _data((70001, 24), torch.bfloat16, seed=5)
    w, b = torch.randn(24, generator=g).cuda(), torch.zeros(24).cuda()
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    _, rdx, rdw, rdb = _reference(x, w, b, 1e-5, dy)
    for got, want, tol in zip(grads, (rdx, rdw, rdb), (BF16_TOL, F32_TOL, F32_TOL)):
        _close(got, want, tol, "gradient")


@pytest.mark.gpu
def test_large_mean_keeps_the_variance():
    """Rows at 1000 with spread 1: fp32 holds x to 2^-14, so h is off by about 6e-5 / sqrt(3) from the
    rounding of the inputs alone, which the reference reads too; the mean's own rounding (2^-15 at
    worst) shifts h by 3e-5. E[x^2] - mean^2 would lose three digits more."""
    from fovi_amd.arch.norm import layer_norm
    x = (torch.randn(50, 384, generator=torch.Generator().manual_seed(1)) + 1000).cuda()
    ry = _reference(x, None, None, 1e-5)[0]
    _close(layer_norm(x), ry, 6e-5, "y")


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of a scalar of the output in fp32, step 1e-2: error step^2 (third
    derivatives of order 1) plus 2^-24 * |f| / step, |f| about 3: 2e-4 absolute on gradients of order 1."""
    from fovi_amd.arch.norm import layer_norm
    g = torch.Generator().manual_seed(11)
    x, r = torch.randn(3, 12, generator=g).cuda(), torch.randn(3, 12, generator=g).double()
    w, b = torch.rand(12, generator=g).cuda() + 0.5, torch.randn(12, generator=g).cuda()
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, r.float().cuda())

    def f():
        with torch.no_grad():
            return (layer_norm(*leaves).double().cpu() * r).sum().item()

    for t, gt in zip(leaves, grads):
        flat = t.detach().reshape(-1)
        for i in range(0, flat.numel(), 5):
            v = flat[i].item()
            flat[i] = v + 1e-2
            up = f()
            flat[i] = v - 1e-2
            down = f()
            flat[i] = v
            assert abs((up - down) / 2e-2 - gt.reshape(-1)[i].item()) < 1e-3


@pytest.mark.gpu
def test_infinities_stay_in_their_rows():
    from fovi_amd.arch.norm import layer_norm
    x = torch.randn(6, 384, generator=torch.Generator().manual_seed(2)).cuda()
    x[1, 5], x[4, 7] = float("inf"), float("nan")
    y = layer_norm(x)
    assert y[[1, 4]].isnan().all()
    keep = [0, 2, 3, 5]
    _close(y[keep], _reference(x[keep], None, None, 1e-5)[0], F32_TOL, "y")


@pytest.mark.gpu
def test_empty_inputs():
    from fovi_amd.arch.norm import layer_norm
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.randn(0, 5, 16, device="cuda", requires_grad=True)
    y = layer_norm(x, w)
    assert y.shape == (0, 5, 16)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros(16, device="cuda"))


@pytest.mark.gpu
def test_module_and_stream():
    from fovi_amd.arch.norm import LayerNorm
    m = LayerNorm(384)
    assert {n: tuple(p.shape) for n, p in m.named_parameters()} == {"weight": (384,), "bias": (384,)}
    x = torch.randn(300, 384, generator=torch.Generator().manual_seed(4)).cuda()
    want = _reference(x, None, None, 1e-5)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = m(x)
    torch.cuda.current_stream().wait_stream(s)
    _close(y, want, F32_TOL, "y")
    assert LayerNorm(8, elementwise_affine=False).weight is None and LayerNorm(8, bias=False).bias is None


@pytest.mark.gpu
def test_refusals():
    from fovi_amd.arch.norm import layer_norm
    x = torch.zeros(4, 16, device="cuda")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layer_norm(x.cpu())
    with pytest.raises(TypeError, match="unsupported dtype"):
        layer_norm(x.half())
    with pytest.raises(TypeError, match="weight dtype"):
        layer_norm(x, torch.ones(16, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError, match="weight of shape"):
        layer_norm(x, torch.ones(15, device="cuda"))
    with pytest.raises(TypeError, match="weight is"):
        layer_norm(x, torch.ones(16, device="cuda"), torch.ones(16, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="C >= 1"):
        layer_norm(torch.zeros(4, 0, device="cuda"))


def test_cpu_tensors_and_c_arguments_are_refused():
    from fovi_amd.arch.norm import layer_norm
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layer_norm(torch.zeros(2, 4))
    lib = _lib.load()
    a = _lib.LayerNormArgs()
    assert lib.fovi_layer_norm_fwd(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.x = 16
    a.dtype = 7
    assert lib.fovi_layer_norm_fwd(a, None) != 0 and b"dtypes" in lib.fovi_last_error()
    a.dtype, a.rows0, a.rows1 = _lib.F32, 1, 1
    assert lib.fovi_layer_norm_fwd(a, None) != 0 and b"bad sizes" in lib.fovi_last_error()
    a.channels, a.eps = 8, -1.0
    assert lib.fovi_layer_norm_fwd(a, None) != 0 and b"eps" in lib.fovi_last_error()
    a.eps = 1e-5
    assert lib.fovi_layer_norm_fwd(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    assert lib.fovi_layer_norm_bwd(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.dy, a.mean, a.rstd, a.dweight = 16, 16, 16, 16
    assert lib.fovi_layer_norm_bwd(a, None) != 0 and b"workspace" in lib.fovi_last_error()
    assert lib.fovi_layer_norm_workspace_bytes(0, 8, _lib.F32) == 0


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("py,c", [(_lib.LayerNormArgs, "fovi_layer_norm_args"), (_lib.RotaryArgs, "fovi_rotary_args"),
                                  (_lib.AttentionArgs, "fovi_attention_args"),
                                  (_lib.AttentionBwdArgs, "fovi_attention_bwd_args")])
def test_struct_layout_matches_header(py, c, tmp_path):
    fields = [f for f, _ in py._fields_]
    size, offs = _c_layout(c, fields, tmp_path)
    assert C.sizeof(py) == size
    for f, off in zip(fields, offs):
        assert getattr(py, f).offset == off, f


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c", [(4100, 3), (4097, 7), (4100, 9), (4099, 61), (4100, 131), (4100, 255), (4097, 385),
                                    (40, 255), (70, 513), (33, 1023), (20, 1537), (20, 2046), (5, 4095), (3, 8191)])
def test_odd_widths(rows, c, dtype):
    """Rows that end inside a 16-byte piece, in each shape of the kernels (16, 64 and 256 lanes a row)."""
    test_values_and_gradients(rows, c, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c", [(5, 3), (4099, 13), (9, 385), (2, 1030), (2, 20001)])
def test_writes_its_rows_only(rows, c, dtype):
    """y and dx are slices of wider rows, at odd offsets: what lies around them keeps its value."""
    x, dy, _ = _data((rows, c), dtype)
    lib = _lib.load()
    outs = [torch.full((rows + 2, c + 11), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    y, dx = (t[1:-1, 5:5 + c] for t in outs)
    stats = torch.empty(2, rows, device="cuda")
    a = _lib.LayerNormArgs()
    a.x, a.dtype, a.rows0, a.rows1, a.channels, a.eps = x.data_ptr(), _lib.dtype_code(dtype), 1, rows, c, 1e-5
    a.x_stride[:] = a.dy_stride[:] = (0, c)
    a.y_stride[:] = a.dx_stride[:] = (0, c + 11)
    a.y, a.dy, a.dx, a.mean, a.rstd = y.data_ptr(), dy.data_ptr(), dx.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr()
    _lib.check(lib.fovi_layer_norm_fwd(a, _lib.stream_of(x)), "forward")
    _lib.check(lib.fovi_layer_norm_bwd(a, _lib.stream_of(x)), "backward")
    ry, rdx, _, _ = _reference(x, None, None, 1e-5, dy)
    tol = F32_TOL if dtype == torch.float32 else BF16_TOL
    _close(y, ry, tol, "y")
    _close(dx, rdx, tol, "dx")
    for t, inner in zip(outs, (y, dx)):
        inner.fill_(7.0)
        assert (t == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("constant", [True, False])
def test_differentiating_twice_raises(constant):
    """With a constant incoming gradient and with one that has a gradient itself, in every input; a
    gradient that is only recorded, and not differentiated, is the gradient."""
    from fovi_amd.arch.norm import layer_norm
    g = torch.Generator().manual_seed(20)
    leaves = [torch.randn(s, generator=g).cuda().requires_grad_(True) for s in ((7, 40), (40,), (40,))]
    dy = torch.randn(7, 40, generator=g).cuda().requires_grad_(not constant)
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy, create_graph=True)
    want = torch.autograd.grad(layer_norm(*leaves), leaves, dy.detach())
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    for got in grads:
        for leaf in leaves + ([] if constant else [dy]):
            with pytest.raises(RuntimeError, match="differentiated once"):
                torch.autograd.grad(layer_norm(*leaves).sum() + dy.sum() + got.square().sum(), leaf, retain_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_raises(which, grad):
    """A tangent of any input is refused, not dropped; with a level open and no tangent the call is the
    ordinary one."""
    from torch.autograd import forward_ad
    from fovi_amd.arch.norm import layer_norm
    args = [torch.randn(s, device="cuda") for s in ((4, 24), (24,), (24,))]
    want = layer_norm(*args)
    args[which].requires_grad_(grad)
    leaf = args[0].detach().requires_grad_(True)
    y = layer_norm(leaf, *args[1:])
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(want), torch.ones_like(want)))
    with forward_ad.dual_level():
        assert torch.equal(layer_norm(*args), want)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for off in (False, True):
            with torch.set_grad_enabled(not off), pytest.raises(NotImplementedError, match="forward mode"):
                layer_norm(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c", [(5, 48), (5000, 385), (9, 20000)])
def test_capture(rows, c, dtype):
    """Forward and backward captured; replayed with new inputs and with work of its own between."""
    from fovi_amd.arch.norm import layer_norm
    g = torch.Generator().manual_seed(21)
    leaves = [torch.randn(rows, c, generator=g).to(dtype).cuda().requires_grad_(True)]
    leaves += [torch.randn(c, generator=g).cuda().requires_grad_(True) for _ in range(2)]
    dy = torch.randn(rows, c, generator=g).to(dtype).cuda()

    def step():
        y = layer_norm(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

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
            for t in leaves + [dy]:
                t.copy_(torch.randn(t.shape, generator=g))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
