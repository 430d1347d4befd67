"""The gated feed-forward block and its gradients against float64, and the block in training and in 8-bit serving.

Tolerances are bounds of the arithmetic, worked out in float64 beside the values. A sum of n products in fp32 is off by at most
(n + 2) 2^-23 of the sum of their magnitudes (the matrix unit's additions may truncate: 2^-23 each); u is half a step of the
tensors' type. bf16 calls round the gated product and its two gradients (u of each) before the next product. Slopes of
the activations are at most 1.13, their second derivatives at most 0.8; their exponentials and reciprocals (or erf) are off by
2^-20 relative to 1 + |z|. From 768 channels on bf16 calls keep gate and up for the backward, rounded: u of each more in what
the gradients are formed from.
"""
import pytest
import torch

from fovi_amd import _lib

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _data(m, c, f, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, r, dy = (torch.randn(m, c, generator=g).to(dtype).cuda() for _ in range(3))
    w = [(torch.randn(s, generator=g) / s[1] ** 0.5).to(dtype).cuda() for s in ((f, c), (f, c), (c, f))]
    return x, w, r, dy


def _act(z, name):
    """(value, slope)"""
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    half = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
    return z * half, half + z * (-0.5 * z * z).exp() / (2 * torch.pi) ** 0.5


def _sum_error(a, b):
    """What a product of these magnitudes may lose in fp32."""
    return (a.shape[1] + 2) * 2.0 ** -23 * (a @ b)


def _expected(x, w, r, dy, act):
    """{name: (value, bound)} in float64."""
    dtype = x.dtype
    u = U[dtype]
    ub = u if dtype == torch.bfloat16 else 2.0 ** -23              # what rounding between the products loses
    x, (wg, wu, wd), dy = x.detach().double(), [t.detach().double() for t in w], dy.double()
    gate, up = x @ wg.t(), x @ wu.t()
    eg, eu = _sum_error(x.abs(), wg.abs().t()), _sum_error(x.abs(), wu.abs().t())
    value, slope = _act(gate, act)
    ev = 1.13 * eg + 2.0 ** -20 * (1 + gate.abs()) * value.abs() + 2.0 ** -22 * gate.abs()
    es = 0.8 * eg + 2.0 ** -20 * (1 + gate.abs()) ** 2
    h = value * up
    eh = ev * up.abs() + value.abs() * eu + ev * eu + ub * h.abs()
    y = h @ wd.t()
    ey = eh @ wd.abs().t() + _sum_error(h.abs() + eh, wd.abs().t())
    if r is not None:
        y = y + r.detach().double()
        ey = ey + 2.0 ** -23 * (y.abs() + r.detach().double().abs())
    if dtype == torch.bfloat16 and x.shape[1] >= 768:
        eg, eu = eg + u * (gate.abs() + eg), eu + u * (up.abs() + eu)
        ev = 1.13 * eg + 2.0 ** -20 * (1 + gate.abs()) * value.abs() + 2.0 ** -22 * gate.abs()
        es = 0.8 * eg + 2.0 ** -20 * (1 + gate.abs()) ** 2
        eh = ev * up.abs() + value.abs() * eu + ev * eu + ub * h.abs()
    dh = dy @ wd
    edh = _sum_error(dy.abs(), wd.abs())
    dgate, dup = dh * up * slope, dh * value
    edg = edh * (up * slope).abs() + dh.abs() * (eu * slope.abs() + up.abs() * es + eu * es) + edh * eu + (ub + 2.0 ** -22) * dgate.abs()
    edu = edh * value.abs() + dh.abs() * ev + edh * ev + (ub + 2.0 ** -22) * dup.abs()
    dx = dgate @ wg + dup @ wu
    edx = edg @ wg.abs() + edu @ wu.abs() + _sum_error(torch.cat([dgate.abs() + edg, dup.abs() + edu], 1), torch.cat([wg.abs(), wu.abs()]))
    out = {"y": (y, ey), "dx": (dx, edx)}
    for name, a, ea, b, eb in (("dw_gate", dgate, edg, x, 0), ("dw_up", dup, edu, x, 0), ("dw_down", dy, 0, h, eh)):
        v = a.t() @ b
        e = _sum_error((a.abs() + ea).t(), b.abs() + eb)
        e = e + (ea.t() @ b.abs() if torch.is_tensor(ea) else a.abs().t() @ eb)
        out[name] = (v, e)
    return {k: (v, 1.01 * (e + u * (v.abs() + e)) + 1e-38) for k, (v, e) in out.items()}


def _within(got, want, what):
    v, bound = want
    assert got.shape == v.shape
    over = ((got.detach().double() - v).abs() - bound).max().item()
    assert over <= 0, f"{what}: {over:.3e} over the bound of {bound.max().item():.3e}"


NAMES = ("dx", "dw_gate", "dw_up", "dw_down")
SIZES = [(1, 1, 1), (1, 384, 1024), (2, 8, 24), (3, 5, 7), (16, 64, 64), (17, 33, 129), (31, 2048, 200), (64, 384, 1024), (65, 96, 64),
         (100, 771, 129), (129, 128, 257), (300, 387, 1031), (1000, 64, 96), (2049, 40, 72), (700, 256, 384), (5000, 8, 16),
         (40, 16, 5504), (33, 1030, 8), (70, 24, 16500), (200, 131, 4100), (256, 640, 96), (200, 100, 67), (300, 768, 512), (2000, 776, 260)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,c,f", SIZES)
def test_values_and_gradients(m, c, f, act, dtype):
    from fovi_amd.arch.feed_forward import gated_mlp
    x, w, r, dy = _data(m, c, f, dtype)
    residual = r if m % 2 else None
    want = _expected(x, w, residual, dy, act)
    y = gated_mlp(x, *w, activation=act, residual=residual)
    _within(y, want["y"], "y")
    leaves = [t.requires_grad_(True) for t in [x] + w]
    if residual is not None:
        residual.requires_grad_(True)
    out = gated_mlp(*leaves, activation=act, residual=residual)
    _within(out, want["y"], "y of training")
    grads = torch.autograd.grad(out, leaves + ([] if residual is None else [residual]), dy)
    for name, g in zip(NAMES, grads):
        _within(g, want[name], name)
    if residual is not None:
        assert torch.equal(grads[-1], dy)
    again = torch.autograd.grad(gated_mlp(*leaves, activation=act, residual=residual), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["whole", "odd"])
@pytest.mark.parametrize("m", [1, 40, 64, 300])
def test_fp32_sums_are_taken_by_stages(m, layout):
    """One product of 2^27 in front of 16383 or so of 1, each lost on its own beside it (half a step is 8): sums by stages lose those
    of its own stage, of 128 at most, a rest of fewer than 16 behind the last one, and the rounding of the result. In the two
    first products (x [.., C] by up [1, C], behind a gate of 32, whose silu is 32), and in the last one (over F)."""
    from fovi_amd.arch.feed_forward import gated_mlp
    k = 16384 if layout == "whole" else 16383
    lost = 128 + 8 + 8

    def wide(rows, cols):                                            # odd: rows that start anywhere
        return torch.zeros(rows, cols + 3, device="cuda")[:, 3:] if layout == "odd" else torch.zeros(rows, cols, device="cuda")

    x, wg, wu = wide(m, k), wide(1, k), wide(1, k)
    wd = torch.full((k, 1), 2.0 ** -5, device="cuda")
    x.fill_(1.0)
    wu.fill_(1.0)
    x[:, 0], wg[:, 0], wu[:, 0] = 2.0 ** 13, 2.0 ** -8, 2.0 ** 14
    with torch.no_grad():
        y = gated_mlp(x, wg, wu, wd)
    assert (y.double() - (2.0 ** 27 + k - 1)).abs().max() <= lost

    x, wg, wu, wd = (torch.ones(m, 4, device="cuda"), torch.zeros(k, 4, device="cuda"), torch.zeros(k, 4, device="cuda"), wide(4, k))
    wg[:, 0], wu[:, 1], wu[0, 1] = 32.0, 2.0 ** -5, 2.0 ** 22
    wd.fill_(1.0)
    with torch.no_grad():
        y = gated_mlp(x, wg, wu, wd)
    assert (y.double() - (2.0 ** 27 + k - 1)).abs().max() <= lost


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,c,f", [(40, 24, 16500), (70, 24, 16500), (70, 17, 16501), (300, 32, 8192), (1025, 8, 5504), (20000, 24, 40),
                                   (40000, 17, 264)])
def test_split_sums_are_whole(m, c, f, dtype):
    """Long reductions, split over workgroups, of small whole numbers: every product and sum is exact in either type (what is
    rounded to bf16 in between is at most 128; sums stay below 2^24 times what all their parts are multiples of), so that a lost
    or doubled stage shows whatever its size. Gates of 32 have silu 32 and slope 1."""
    from fovi_amd.arch.feed_forward import gated_mlp
    g = torch.Generator().manual_seed(m + f)

    def whole(rows, cols, at):                                       # -1, 0 and 1 in the columns from `at` on
        t = torch.randint(-1, 2, (rows, cols), generator=g).double()
        t[:, :at] = 0
        return t

    x, wu, wd, dy = whole(m, c, 1), whole(f, c, 1), whole(c, f, 0), whole(m, c, 0)
    wu[:, 4:] = 0                                                    # up is -3 .. 3
    dy[:, 4:] = 0                                                    # dh is -4 .. 4
    wg = torch.zeros(f, c, dtype=torch.float64)
    x[:, 0], wg[:, 0] = 32, 1
    up, dh = x @ wu.t(), dy @ wd
    h, dgate, dup = 32 * up, dh * up, dh * 32
    want = [h @ wd.t(), dgate @ wg + dup @ wu, dgate.t() @ x, dup.t() @ x, dy.t() @ h]
    for a, b in ((h.abs(), wd.abs().t()), (dup.abs(), wu.abs()), (dgate.abs(), wg), (dgate.abs().t(), x.abs()), (dup.abs().t() / 32, x.abs()),
                 (dy.abs().t(), h.abs())):
        assert (a @ b).max() < 2 ** 24
    leaves = [t.to(dtype).cuda().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_mlp(*leaves)
    got = (y,) + torch.autograd.grad(y, leaves, dy.to(dtype).cuda())
    for name, a, b in zip(("y",) + NAMES, got, want):
        assert torch.equal(a.detach().cpu(), b.to(dtype)), name


@pytest.mark.gpu
@pytest.mark.parametrize("c,f", [(1024, 1032), (384, 2056)])
def test_offsets_past_32_bits(c, f):
    """Rows, gate and up, and their gradients of more than 2^31 elements. Only the last rows have an incoming gradient, so that
    every result comes from them."""
    from fovi_amd.arch.feed_forward import gated_mlp
    m, last = 2 ** 21 + 70, 70
    x, w, r, dy = _data(last, c, f, torch.bfloat16)
    rows = torch.randn(m, c, device="cuda", dtype=torch.bfloat16)
    rows[-last:] = x
    grads = torch.zeros(m, c, device="cuda", dtype=torch.bfloat16)
    grads[-last:] = dy
    want = _expected(x, w, None, dy, "silu")
    leaves = [t.requires_grad_(True) for t in [rows] + w]
    y = gated_mlp(*leaves)
    _within(y[-last:], want["y"], "y")
    dx, *dw = torch.autograd.grad(y, leaves, grads)
    _within(dx[-last:], want["dx"], "dx")
    assert not dx[:-last].any()
    for name, g in zip(NAMES[1:], dw):
        _within(g, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", [(0,), (1,), (2,), (3,), (0, 3), (1, 2)])
def test_parts_of_the_gradients(which, dtype):
    """Each of the inputs alone and some together: the same bits as all at once."""
    from fovi_amd.arch.feed_forward import gated_mlp
    x, w, r, dy = _data(300, 64, 96, dtype)
    leaves = [x] + w
    all_of = [t.detach().requires_grad_(True) for t in leaves]
    want = torch.autograd.grad(gated_mlp(*all_of), all_of, dy)
    some = [t.detach().requires_grad_(i in which) for i, t in enumerate(leaves)]
    got = torch.autograd.grad(gated_mlp(*some), [some[i] for i in which], dy)
    assert all(torch.equal(a, want[i]) for a, i in zip(got, which))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [5, 200])
@pytest.mark.parametrize("layout", ["padded", "odd_offset", "tokens", "expanded", "columns"])
def test_layouts(layout, m, dtype):
    """Rows, weights and incoming gradients where they are: the values of the contiguous call."""
    from fovi_amd.arch.feed_forward import gated_mlp
    g = torch.Generator().manual_seed(5)
    c, f = 40, 48

    def make(rows, width, at, n):
        return torch.randn(rows, width, generator=g).to(dtype).cuda()[:, at:at + n]

    pad, at = {"padded": (8, 0), "odd_offset": (11, 3)}.get(layout, (0, 0))
    x, r, dy = (make(m, c + pad, at, c) for _ in range(3))
    w = [make(a, b + pad, at, b) for a, b in ((f, c), (f, c), (c, f))]
    if layout == "tokens":
        x, r, dy = (make(2 * m, c, 0, c).view(2, m, c)[:, 1:] for _ in range(3))
    if layout == "expanded":
        dy, x = dy[:1].expand(m, c), x[:1].expand(m, c)
    if layout == "columns":
        w = [t.t().contiguous().t() for t in w]

    def run(x, r, dy, *w):
        leaves = [t.detach().requires_grad_(True) for t in (x, *w, r)]
        y = gated_mlp(*leaves[:4], residual=leaves[4])
        with torch.no_grad():
            assert (gated_mlp(*leaves[:4], residual=leaves[4]).double() - y.double()).norm() <= 2.0 ** -6 * y.double().norm()
        return (y,) + torch.autograd.grad(y, leaves, dy)

    got, want = run(x, r, dy, *w), run(*(t.contiguous() for t in (x, r, dy, *w)))
    for i, (a, b) in enumerate(zip(got, want)):      # other loads take other kernels: the same sums in another order
        assert a.shape == b.shape
        assert (a.double() - b.double()).norm() <= (2.0 ** -7 if dtype == torch.bfloat16 else 1e-6) * b.double().norm(), i


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the float64 formula, in a direction of each input."""
    from fovi_amd.arch.feed_forward import gated_mlp
    for act in ("silu", "gelu"):
        x, w, r, dy = _data(9, 12, 20, torch.float32, 3)
        leaves = [t.requires_grad_(True) for t in [x] + w]
        grads = torch.autograd.grad(gated_mlp(*leaves, activation=act), leaves, dy)
        base = [t.detach().double() for t in leaves]

        def loss(x, wg, wu, wd):
            return (((_act(x @ wg.t(), act)[0] * (x @ wu.t())) @ wd.t()) * dy.double()).sum().item()

        for i in range(4):
            v = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
            h = 1e-5
            up, down = ([t + s * h * v if j == i else t for j, t in enumerate(base)] for s in (1, -1))
            want = (loss(*up) - loss(*down)) / (2 * h)
            assert abs((grads[i].double() * v).sum().item() - want) < 1e-4 * max(1.0, abs(want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [6, 200])
def test_what_is_not_finite_stays_in_its_rows(m, dtype):
    """Rows with infinities and NaN, and large gates, leave the other rows as they are; the last rows of a tile take no part."""
    from fovi_amd.arch.feed_forward import gated_mlp
    x, w, r, dy = _data(m, 72, 100, dtype)
    want = gated_mlp(x, *w)
    bad = x.clone()
    bad[1, 3], bad[m - 1, 5] = float("nan"), float("inf")
    bad[2] *= 1000
    with torch.no_grad():
        y = gated_mlp(bad, *w)
    keep = [i for i in range(m) if i not in (1, 2, m - 1)]
    assert torch.equal(y[keep], want[keep])
    assert y[1].isnan().all() and not y[m - 1].isfinite().any() and y[2].isfinite().all()
    leaf = bad.requires_grad_(True)
    (dx,) = torch.autograd.grad(gated_mlp(leaf, *w), leaf, dy)
    assert dx[keep].isfinite().all() and dx[1].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,c,f", [(3, 21, 37), (70, 40, 100), (130, 131, 67), (300, 64, 128)])
def test_writes_its_rows_only(m, c, f, dtype):
    """y at a stride of its own inside a larger buffer, gradients between guards."""
    x, w, r, dy = _data(m, c, f, dtype)
    lib, es = _lib.load(), x.element_size()
    want = _expected(x, w, r, dy, "silu")
    out = torch.full((m + 2, c + 9), 7.0, dtype=dtype, device="cuda")
    y = out[1:-1, 3:3 + c]
    a = _lib.GatedMlpArgs()
    a.x, a.w_gate, a.w_up, a.w_down = (t.data_ptr() for t in (x, *w))
    a.dtype, a.rows, a.dim, a.hidden = _lib.dtype_code(dtype), m, c, f
    a.x_stride = a.w_gate_stride = a.w_up_stride = a.residual_stride = a.dy_stride = c
    a.w_down_stride, a.residual, a.y, a.y_stride = f, r.data_ptr(), y.data_ptr(), c + 9
    sizes = m, c, f, a.dtype
    saved = torch.empty(max(1, lib.fovi_gated_mlp_saved_bytes(*sizes)), dtype=torch.uint8, device="cuda")
    a.dy = dy.data_ptr()
    work = [torch.full((n + 512,), 3, dtype=torch.uint8, device="cuda") for n in (lib.fovi_gated_mlp_fwd_workspace_bytes(a),
                                                                                lib.fovi_gated_mlp_bwd_workspace_bytes(a))]
    a.saved = saved.data_ptr() if lib.fovi_gated_mlp_saved_bytes(*sizes) else None
    a.workspace, a.workspace_bytes = work[0].data_ptr() + 256, work[0].numel() - 512
    _lib.check(lib.fovi_gated_mlp_fwd(a, _lib.stream_of(x)), "forward")
    _within(y, want["y"], "y")
    y.fill_(7.0)
    assert (out == 7.0).all()
    grads = [torch.full((t.numel() + 32,), 7.0, dtype=dtype, device="cuda") for t in (x, *w)]
    a.dx, a.dw_gate, a.dw_up, a.dw_down = (t.data_ptr() + 16 * es for t in grads)
    a.workspace, a.workspace_bytes = work[1].data_ptr() + 256, work[1].numel() - 512
    _lib.check(lib.fovi_gated_mlp_bwd(a, _lib.stream_of(x)), "backward")
    for name, t, like in zip(NAMES, grads, (x, *w)):
        _within(t[16:-16].view(like.shape), want[name], name)
        assert (t[:16] == 7).all() and (t[-16:] == 7).all(), name
    for t in work:
        assert (t[:256] == 3).all() and (t[-256:] == 3).all()


@pytest.mark.gpu
def test_empty_and_autocast():
    from fovi_amd.arch.feed_forward import gated_mlp
    x, w, r, dy = _data(20, 24, 40, torch.float32)
    leaves = [t.requires_grad_(True) for t in [x] + w]
    none = x[:0]
    y = gated_mlp(none, *leaves[1:], residual=r[:0])
    assert y.shape == (0, 24)
    assert all((g == 0).all() for g in torch.autograd.grad(y.sum(), leaves[1:]))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = gated_mlp(*leaves)
    assert y.dtype == torch.bfloat16
    grads = torch.autograd.grad(y, leaves, dy.bfloat16())
    half = [t.detach().bfloat16().requires_grad_(True) for t in leaves]
    want = torch.autograd.grad(gated_mlp(*half), half, dy.bfloat16())
    assert all(a.dtype == torch.float32 and torch.equal(a, b.float()) for a, b in zip(grads, want))


@pytest.mark.gpu
@pytest.mark.parametrize("constant", [True, False])
def test_differentiating_twice_raises(constant):
    from fovi_amd.arch.feed_forward import gated_mlp
    x, w, r, dy = _data(7, 24, 40, torch.float32)
    leaves = [t.requires_grad_(True) for t in [x] + w]
    dy.requires_grad_(not constant)
    grads = torch.autograd.grad(gated_mlp(*leaves), leaves, dy, create_graph=True)
    want = torch.autograd.grad(gated_mlp(*leaves), leaves, dy.detach())
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    for got in grads:
        for leaf in leaves + ([] if constant else [dy]):
            with pytest.raises(RuntimeError, match="differentiated once"):
                torch.autograd.grad(gated_mlp(*leaves).sum() + dy.sum() + got.square().sum(), leaf, retain_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(5))
def test_forward_mode_raises(which):
    from torch.autograd import forward_ad
    from fovi_amd.arch.feed_forward import gated_mlp
    x, w, r, dy = _data(7, 24, 40, torch.float32)
    args = [x, *w, r]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for off in (False, True):
            with torch.set_grad_enabled(not off), pytest.raises(NotImplementedError, match="forward mode"):
                gated_mlp(*args[:4], residual=args[4])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,c,f", [(1, 64, 96), (40, 128, 300), (3000, 64, 96), (600, 387, 130)])
def test_capture(m, c, f, dtype):
    """Forward and backward captured; replayed with new inputs and with work of its own between. Two graphs of one step keep
    their workspaces apart."""
    from fovi_amd.arch.feed_forward import gated_mlp
    x, w, r, dy = _data(m, c, f, dtype)
    leaves = [t.requires_grad_(True) for t in [x] + w]

    def step():
        with torch.no_grad():
            served = gated_mlp(*leaves, residual=r)
        y = gated_mlp(*leaves, residual=r)
        return (served, y.detach()) + torch.autograd.grad(y, leaves, dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs, results = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            results.append(step())
    g = torch.Generator().manual_seed(22)
    for i in range(4):
        with torch.no_grad():
            for t in leaves + [dy, r]:
                t.copy_(torch.randn(t.shape, generator=g) / 8)
        want = step()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in results:
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_together(dtype):
    """Norm, residual and block in training, against float64 (norm-wise: three roundings of u a value in bf16, and the products'
    averages of such; fp32 sums of some hundred terms), and the same block in 8 bits for serving, step by step."""
    from fovi_amd.arch.feed_forward import GatedFeedForward
    from fovi_amd.arch.int8 import gated_linear_int8, linear_int8, quantize_int8
    from fovi_amd.arch.norm import rms_norm_int8
    torch.manual_seed(2)
    block = GatedFeedForward(72, 200).to(dtype)
    assert block.hidden == 200 and GatedFeedForward(384).hidden == 1024 and "72" in repr(block)
    x, r, dy = (torch.randn(3, 50, 72, device="cuda").to(dtype).requires_grad_(i < 2) for i in range(3))
    leaves = [x, r, block.norm.weight, block.w_gate, block.w_up, block.w_down]
    y = block(x, r)
    grads = torch.autograd.grad(y, leaves, dy)
    d = [t.detach().double().requires_grad_(True) for t in leaves]
    total = d[0] + d[1]
    n = total / (total.square().mean(-1, keepdim=True) + 1e-6).sqrt() * d[2]
    want = total + (torch.nn.functional.silu(n @ d[3].t()) * (n @ d[4].t())) @ d[5].t()
    tol = 3e-6 if dtype == torch.float32 else 4 * 2.0 ** -8
    for a, b in zip((y,) + grads, (want,) + torch.autograd.grad(want, d, dy.double())):
        assert (a.double() - b).norm() <= tol * b.norm()
    alone = block(x.detach() + r.detach())
    assert (alone.double() - y.double()).norm() <= 2 * U[dtype] * y.double().norm() + 1e-12

    served = block.int8().bfloat16()
    with torch.no_grad():
        got = served(x, r)
        q, total = rms_norm_int8(x, block.norm.weight, residual=r)
        wg, wu, wd = (quantize_int8(w) for w in (block.w_gate, block.w_up, block.w_down))
        h = gated_linear_int8(q, wg, wu, dtype=dtype)
        assert torch.equal(got, linear_int8(quantize_int8(h), wd, residual=total, dtype=dtype))
        assert torch.equal(served(total), linear_int8(quantize_int8(h), wd, residual=total, dtype=dtype))
    # steps of a 127th of a row's largest value, about 3 of its root mean square: 0.29 / 127 * 3 of a value at each of five
    # places in the way of the block's part, itself less than the whole
    assert (got.double() - y.double()).norm() <= 0.03 * y.double().norm()


@pytest.mark.gpu
def test_autocast_keeps_an_fp32_residual_stream():
    from fovi_amd.arch.feed_forward import GatedFeedForward, gated_mlp
    torch.manual_seed(2)
    block = GatedFeedForward(64, 128)
    x, r = torch.randn(30, 64, device="cuda"), 1000 * torch.randn(30, 64, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        y = block(x, r)
        n, total = block.norm(x, r)
        want = total + gated_mlp(n, block.w_gate, block.w_up, block.w_down)
    assert y.dtype == torch.float32 and torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reader_with_a_feed_forward_block(dtype):
    """The reader's block behind its attention: its own parts put together by hand, gradients everywhere, and 8-bit serving
    through the same call."""
    from fovi_amd.arch.reader import FixationReader, fixation_positions
    from fovi_amd.sensing.coords import SamplingCoords
    torch.manual_seed(4)
    reader = FixationReader(64, 48, heads=2, head_dim=32, hidden=96).to(dtype)
    pos = fixation_positions(SamplingCoords(16, 2.78, 8, style="logpolar"), 2)
    x = torch.randn(3, 5, 64, device="cuda").to(dtype).requires_grad_(True)
    states = torch.randn(3, len(pos), 48, device="cuda").to(dtype)
    y = reader(x, states, pos)
    block, reader.feed_forward = reader.feed_forward, None
    read = reader(x, states, pos)
    reader.feed_forward = block
    # block(read - x, x) sums to what the reader without the block gives, up to its rounding
    assert (block(read).double() - y.double()).norm() <= 4 * U[dtype] * y.double().norm()
    grads = torch.autograd.grad(y.float().square().mean(), [x] + list(reader.parameters()))
    assert len(grads) > 8 and all(g.isfinite().all() and g.abs().max() > 0 for g in grads)
    reader.feed_forward = reader.feed_forward.int8()
    with torch.no_grad():
        served = reader(x, states, pos)
    assert served.dtype == dtype and (served.double() - y.double()).norm() <= 0.03 * y.double().norm()


@pytest.mark.gpu
def test_refusals():
    from fovi_amd.arch.feed_forward import GatedFeedForward, gated_mlp
    x, w, r, dy = _data(4, 16, 24, torch.float32)
    with pytest.raises(ValueError, match="weights"):
        gated_mlp(x, w[0], w[1], w[0])
    with pytest.raises(ValueError, match="weights"):
        gated_mlp(x, w[0], w[1][:20], w[2])
    with pytest.raises(ValueError, match="activation"):
        gated_mlp(x, *w, activation="relu")
    with pytest.raises(ValueError, match="activation"):
        GatedFeedForward(16, activation="relu")
    with pytest.raises(ValueError, match="residual"):
        gated_mlp(x, *w, residual=r[:2])
    with pytest.raises(TypeError, match="dtypes"):
        gated_mlp(x, w[0].bfloat16(), w[1], w[2])
    with pytest.raises(TypeError, match="dtypes"):
        gated_mlp(x.half(), *(t.half() for t in w))
    with pytest.raises(ValueError, match="C >= 1"):
        gated_mlp(x[:, :0], *w)
    with pytest.raises(ValueError, match="no gradients"):
        GatedFeedForward(16, 24).int8()(x.requires_grad_(True))


def test_cpu_tensors_and_c_arguments_are_refused():
    from fovi_amd.arch.feed_forward import gated_mlp
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        gated_mlp(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(3, 4), torch.zeros(4, 3))
    lib = _lib.load()
    a = _lib.GatedMlpArgs()
    assert lib.fovi_gated_mlp_fwd(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.x = a.w_gate = a.w_up = a.w_down = 16
    a.dtype = 9
    assert lib.fovi_gated_mlp_fwd(a, None) != 0 and b"dtype" in lib.fovi_last_error()
    a.dtype, a.activation = _lib.BF16, 7
    assert lib.fovi_gated_mlp_fwd(a, None) != 0 and b"activation" in lib.fovi_last_error()
    a.activation, a.rows = _lib.GATE_SILU, 4
    assert lib.fovi_gated_mlp_fwd(a, None) != 0 and b"bad sizes" in lib.fovi_last_error()
    a.dim, a.hidden = 8, 16
    assert lib.fovi_gated_mlp_fwd(a, None) != 0 and b"workspace" in lib.fovi_last_error()
    assert lib.fovi_gated_mlp_bwd(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.dy = 16
    assert lib.fovi_gated_mlp_bwd(a, None) != 0 and b"workspace" in lib.fovi_last_error()
    a.dtype = _lib.F32
    assert lib.fovi_gated_mlp_bwd(a, None) != 0 and b"gate and up" in lib.fovi_last_error()
    a.rows = 0
    assert lib.fovi_gated_mlp_bwd(a, None) != 0 and b"no rows" in lib.fovi_last_error()
    assert lib.fovi_gated_mlp_saved_bytes(0, 8, 16, _lib.F32) == 0
    assert lib.fovi_gated_mlp_fwd_workspace_bytes(a) == 0 and lib.fovi_gated_mlp_bwd_workspace_bytes(a) == 0
