"""Rotary positions on several axes against float64 (complex turns), over types, layouts, sections and positions.

Tolerances: the angle reaches the sine with fp32 accuracy, and each output is two products and a
sum, so fp32 outputs are within 5e-7 of the pair's length; bf16 outputs are rounded once, 2^-9 at
most of each value (2.05e-3 with the fp32 part).
"""
import math

import pytest
import torch

from fovi_amd import _lib

TOL = {torch.float32: 5e-7, torch.bfloat16: 2.05e-3}


def _reference(x, positions, freqs, sections, pairing, sign=1):
    x = x.detach().double().cpu().clone()
    pos, freqs = positions.detach().float().double().cpu(), freqs.double().cpu()
    if pos.dim() == 2:
        pos = pos.expand(x.shape[0], *pos.shape)
    p = sum(sections)
    angle = torch.empty(x.shape[0], x.shape[1], p, dtype=torch.float64)
    at = 0
    for a, n in enumerate(sections):
        angle[..., at:at + n] = pos[..., a:a + 1] * freqs[at:at + n]
        at += n
    angle = sign * angle[:, :, None]
    iu = torch.arange(p) if pairing == "half" else 2 * torch.arange(p)
    iv = iu + p if pairing == "half" else iu + 1
    u, v = x[..., iu], x[..., iv]
    x[..., iu], x[..., iv] = u * angle.cos() - v * angle.sin(), v * angle.cos() + u * angle.sin()
    return x


def _close(got, want, dtype):
    err = (got.detach().double().cpu() - want).norm() / want.norm().clamp_min(1e-30)
    assert got.dtype == dtype and err <= TOL[dtype], f"{err:.2e}"


def _inputs(b, l, h, d, axes, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, l, h, d, generator=g).to(dtype).cuda()
    pos = (2 * torch.rand(b, l, axes, generator=g) - 1) * spread
    return x, pos.cuda(), g


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("b,l,h,d,sections", [
    (1, 1, 1, 2, (1,)), (2, 5, 3, 7, (1, 2)), (64, 1, 6, 64, (8, 12, 12)), (3, 70, 6, 64, (16, 16)),
    (2, 33, 5, 80, (7, 11, 11)), (1, 257, 2, 128, (64,)), (2, 19, 4, 32, (4, 4, 4, 4)), (1, 40, 3, 96, (0, 20, 12)),
    (2, 9, 1, 250, (60, 60)), (1, 3, 40, 64, (32,)), (5, 301, 12, 64, (10, 11, 11))])
def test_values_and_gradient(b, l, h, d, sections, pairing, dtype):
    from fovi_amd.arch.rotary import rotary
    x, pos, g = _inputs(b, l, h, d, len(sections), dtype)
    freqs = (6.3 * torch.rand(sum(sections), generator=g)).cuda()
    y0 = rotary(x, pos, freqs, sections, pairing)
    leaf = x.detach().requires_grad_(True)
    y = rotary(leaf, pos, freqs, sections, pairing)
    assert torch.equal(y, y0)
    dy = torch.randn(x.shape, generator=g).to(dtype).cuda()
    (dx,) = torch.autograd.grad(y, leaf, dy)
    _close(y, _reference(x, pos, freqs, sections, pairing), dtype)
    _close(dx, _reference(dy, pos, freqs, sections, pairing, -1), dtype)
    rest = 2 * sum(sections)
    assert torch.equal(y[..., rest:], x[..., rest:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["heads_first", "kv_slice", "odd_offset", "element_stride", "expanded", "shared_positions"])
def test_layouts(layout, dtype):
    from fovi_amd.arch.rotary import rotary
    b, l, h, d, sections = 3, 37, 4, 32, (4, 6, 6)
    x, pos, g = _inputs(b, l, h, d, 3, dtype, seed=1)

    def randn(*shape):
        return torch.randn(shape, generator=g).to(dtype).cuda()

    if layout == "heads_first":
        x = randn(b, h, l, d).transpose(1, 2)
    elif layout == "kv_slice":
        x = randn(b, l, 2, h, d)[:, :, 1]
    elif layout == "odd_offset":
        x = randn(b, l, h, d + 3)[..., 3:]
    elif layout == "element_stride":
        x = randn(b, l, d, h).transpose(2, 3)
    elif layout == "expanded":
        x = randn(1, l, h, d).expand(b, l, h, d)
    elif layout == "shared_positions":
        pos = pos[0].t().contiguous().t()
    freqs = torch.rand(16, generator=g).cuda() * 6
    leaf = x.detach().requires_grad_(True)
    y = rotary(leaf, pos, freqs, sections)
    dy = randn(b, h, l, d).transpose(1, 2)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    _close(y, _reference(x, pos, freqs, sections, "half"), dtype)
    _close(dx, _reference(dy, pos, freqs, sections, "half", -1), dtype)
    if layout == "heads_first":
        assert y.stride() == x.stride()


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [1e3, 1e5, 1.6e7])
def test_far_positions_keep_fp32_accuracy(spread):
    """An fp32 angle of 1e7 is a multiple of one radian; reduced in fp64 it is as good as a small one."""
    from fovi_amd.arch.rotary import rotary
    x, pos, g = _inputs(2, 50, 2, 64, 2, torch.float32, seed=2, spread=spread)
    freqs = torch.rand(32, generator=g).cuda() * 6.3
    _close(rotary(x, pos, freqs, (16, 16)), _reference(x, pos, freqs, (16, 16), "half"), torch.float32)


@pytest.mark.gpu
def test_whole_positions_and_fp64_coordinates():
    from fovi_amd.arch.rotary import rotary
    x, _, g = _inputs(2, 11, 3, 32, 2, torch.float32, seed=3)
    freqs = torch.rand(16, generator=g).cuda()
    whole = torch.randint(0, 1000, (11, 2), generator=g).cuda()
    _close(rotary(x, whole, freqs, (8, 8)), _reference(x, whole, freqs, (8, 8), "half"), torch.float32)
    wide = torch.rand(11, 2, generator=g, dtype=torch.float64).cuda()
    _close(rotary(x, wide, freqs, (8, 8)), _reference(x, wide, freqs, (8, 8), "half"), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_position_zero_and_inverse(pairing):
    """A token at 0 stays as it is, bit for bit; the gradient's rotation undoes the rotation."""
    from fovi_amd.arch.rotary import AxialRotary
    rope = AxialRotary(64, (8, 12, 12), pairing=pairing)
    x, pos, _ = _inputs(2, 21, 3, 64, 3, torch.float32, seed=4)
    pos[:, 0] = 0
    leaf = x.detach().requires_grad_(True)
    y = rope(leaf, pos)
    assert torch.equal(y[:, 0], x[:, 0])
    (back,) = torch.autograd.grad(y, leaf, y.detach())
    assert ((back - x).norm() / x.norm()).item() < 1e-6       # two rotations, 5e-7 each


@pytest.mark.gpu
def test_relative_positions():
    """Products of rotated queries and keys depend on the difference of positions alone."""
    from fovi_amd.arch.rotary import AxialRotary
    rope = AxialRotary(64, (16, 16), base=100.0)
    g = torch.Generator().manual_seed(5)
    q, k = torch.randn(1, 9, 1, 64, generator=g).cuda(), torch.randn(1, 9, 1, 64, generator=g).cuda()
    pos = torch.rand(9, 2, generator=g).cuda()
    shift = torch.tensor([0.25, -0.5], device="cuda")
    a = (rope(q, pos).double() * rope(k, pos + shift).double()).sum(-1)
    b = (rope(q, pos + shift).double() * rope(k, pos + 2 * shift).double()).sum(-1)
    assert (a - b).abs().max().item() < 64 * 2e-6            # |q||k| about 64; position sums round to 2^-24


@pytest.mark.gpu
def test_default_frequencies_are_the_backbone_rope():
    """The defaults give the angles of the DINOv3 patch positions (two axes, base 100, 2 pi times
    coordinates in [-1, 1], pairs (j, j + D/2)); the backbone library applies them to the patch
    tokens behind its prefix tokens, which have position 0 here."""
    transformers = pytest.importorskip("transformers.models.dinov3_vit.modeling_dinov3_vit")
    from fovi_amd.arch.rotary import AxialRotary
    g = torch.Generator().manual_seed(6)
    q, k = torch.randn(2, 3, 5 + 49, 64, generator=g), torch.randn(2, 3, 5 + 49, 64, generator=g)
    coords = 2 * torch.rand(49, 2, generator=g) - 1
    inv = 1 / 100.0 ** torch.arange(0, 1, 4 / 64, dtype=torch.float32)
    angles = (2 * math.pi * coords[:, :, None] * inv[None, None]).flatten(1, 2).tile(2)
    want, _ = transformers.apply_rotary_pos_emb(q, k, angles.cos(), angles.sin())
    pos = torch.cat([torch.zeros(5, 2), coords]).cuda()
    got = AxialRotary(64)(q.transpose(1, 2).cuda(), pos).transpose(1, 2).cpu()
    assert ((got - want).norm() / want.norm()).item() < 2e-6     # fp32 angles of up to 6.3 there


@pytest.mark.gpu
def test_empty_and_stream():
    from fovi_amd.arch.rotary import AxialRotary
    rope = AxialRotary(32)
    assert rope(torch.zeros(2, 0, 3, 32, device="cuda"), torch.zeros(0, 2, device="cuda")).shape == (2, 0, 3, 32)
    x, pos, _ = _inputs(4, 300, 3, 32, 2, torch.float32, seed=8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = rope(x, pos)
    torch.cuda.current_stream().wait_stream(s)
    _close(y, _reference(x, pos, rope.freqs, rope.sections, "half"), torch.float32)


@pytest.mark.gpu
def test_refusals():
    from fovi_amd.arch.rotary import AxialRotary, rotary
    x, pos, _ = _inputs(2, 5, 3, 32, 2, torch.float32)
    freqs = torch.ones(16, device="cuda")
    ok = (x, pos, freqs, (8, 8))
    rotary(*ok)
    for args, kind, match in [((x[0],) + ok[1:], ValueError, "expected"), ((x.half(),) + ok[1:], TypeError, "dtype"),
                              ((x, pos[:, :4], freqs, (8, 8)), ValueError, "positions"),
                              ((x, pos[..., :1], freqs, (8, 8)), ValueError, "positions"),
                              ((x, pos, freqs[:15], (8, 8)), ValueError, "freqs"),
                              ((x, pos, torch.ones(17, device="cuda"), (8, 9)), ValueError, "do not fit"),
                              ((x, pos, freqs, (-1, 17)), ValueError, "negative"),
                              ((x, torch.zeros(5, 5, device="cuda"), freqs, (4, 4, 4, 2, 2)), ValueError, "axes"),
                              (ok + ("quarter",), ValueError, "pairing"), ((x.cpu(),) + ok[1:], RuntimeError, "no CPU fallback"),
                              ((x, pos.clone().requires_grad_(True), freqs, (8, 8)), ValueError, "no gradient")]:
        with pytest.raises(kind, match=match):
            rotary(*args)
    with pytest.raises(ValueError, match="built for"):
        AxialRotary(64)(x, pos)
    with pytest.raises(ValueError, match="two axes"):
        AxialRotary(30)
    with pytest.raises(ValueError, match="do not fit"):
        AxialRotary(32, (8, 9))
    with pytest.raises(ValueError, match="bases"):
        AxialRotary(32, (8, 8), base=(10.0,))


def test_c_arguments_are_refused():
    lib = _lib.load()
    a = _lib.RotaryArgs()
    assert lib.fovi_rotary(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.x = a.y = a.positions = a.freqs = 16
    a.dtype = 5
    assert lib.fovi_rotary(a, None) != 0 and b"dtype" in lib.fovi_last_error()
    a.dtype, a.pairing = _lib.F32, 2
    assert lib.fovi_rotary(a, None) != 0 and b"pairing" in lib.fovi_last_error()
    a.pairing, a.n_axes = 0, 5
    assert lib.fovi_rotary(a, None) != 0 and b"axes" in lib.fovi_last_error()
    a.n_axes, a.head_dim = 2, 8
    a.section_end[:] = [3, 2, 0, 0]
    assert lib.fovi_rotary(a, None) != 0 and b"section_end" in lib.fovi_last_error()
    a.section_end[:] = [3, 5, 0, 0]
    assert lib.fovi_rotary(a, None) != 0 and b"bad sizes" in lib.fovi_last_error()


def test_launches_past_the_limit_are_refused():
    """2^24 workgroups of 256 threads, one for each token of 8192 channels: more than one launch holds."""
    lib, a = _lib.load(), _lib.RotaryArgs()
    a.x = a.y = a.positions = a.freqs = 4096
    a.dtype, a.n_axes, a.batch, a.length, a.heads, a.head_dim = _lib.BF16, 1, 1 << 24, 1, 64, 128
    a.section_end[:] = [64, 64, 64, 64]
    assert lib.fovi_rotary(a, None) != 0 and b"too many tokens" in lib.fovi_last_error(), lib.fovi_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("d,sections", [(3, (1,)), (6, (3,)), (10, (5,)), (17, (8,)), (18, (9,)), (22, (4, 4)), (30, (15,)),
                                        (34, (8, 9)), (41, (3, 9, 4)), (64, (13, 8, 8)), (66, (16, 16)), (90, (1, 30)),
                                        (128, (3,)), (129, (60, 4))])
def test_odd_runs(d, sections, pairing, dtype):
    """Turned and copied runs that are not whole 16-byte pieces, shorter than one, and odd heads."""
    test_values_and_gradient(3, 21, 3, d, sections, pairing, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pairing", [0, 1])
@pytest.mark.parametrize("d,pairs", [(7, 3), (24, 8), (30, 15), (37, 9), (64, 29)])
def test_writes_its_heads_only(d, pairs, pairing, dtype):
    """Heads inside wider rows, at odd offsets: what lies around them keeps its value."""
    b, l, h = 2, 9, 3
    x, pos, g = _inputs(b, l, h, d, 1, dtype, seed=9)
    freqs = torch.rand(pairs, generator=g).cuda()
    wide = torch.full((b, l, h, d + 11), 7.0, dtype=dtype, device="cuda")
    y = wide[..., 5:5 + d]
    a = _lib.RotaryArgs()
    a.x, a.dtype, a.pairing = x.data_ptr(), _lib.dtype_code(dtype), pairing
    a.batch, a.length, a.heads, a.head_dim = b, l, h, d
    a.x_stride[:], a.y_stride[:] = x.stride()[:3], y.stride()[:3]
    a.positions, a.freqs, a.y = pos.data_ptr(), freqs.data_ptr(), y.data_ptr()
    a.pos_stride[:] = pos.stride()[:2]
    a.n_axes, a.section_end[0] = 1, pairs
    _lib.check(_lib.load().fovi_rotary(a, _lib.stream_of(x)), "fovi_rotary")
    _close(y, _reference(x, pos, freqs, (pairs,), ("half", "adjacent")[pairing]), dtype)
    y.fill_(7.0)
    assert (wide == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("constant", [True, False])
def test_second_gradients(constant):
    """A penalty on a gradient. The rotation is linear, so that its gradient is differentiable as it is. Six
    turns of 5e-7 follow one another at most (y enters squared), with ten roundings of 6e-8: 4e-6."""
    from fovi_amd.arch.rotary import rotary
    x, pos, g = _inputs(2, 9, 3, 24, 2, torch.float32, seed=20)
    freqs = torch.rand(11, generator=g).cuda() * 6
    dy = torch.randn(x.shape, generator=g).cuda()

    def penalty(x, dy, turn):
        if constant:
            (dx,) = torch.autograd.grad((turn(x) * dy).sum(), x, create_graph=True)
            return (turn(x) ** 3).sum() + dx.square().sum()
        (dx,) = torch.autograd.grad((turn(x) ** 3 * dy).sum(), x, create_graph=True)
        return dx.square().sum()

    def plain(x):
        p = pos.double().cpu()
        angle = torch.cat([p[..., :1] * freqs[:5].double().cpu(), p[..., 1:] * freqs[5:].double().cpu()], -1)[:, :, None]
        u, v, rest = x[..., :11], x[..., 11:22], x[..., 22:]
        return torch.cat([u * angle.cos() - v * angle.sin(), v * angle.cos() + u * angle.sin(), rest], -1)

    x.requires_grad_(True)
    dy.requires_grad_(not constant)
    got = torch.autograd.grad(penalty(x, dy, lambda t: rotary(t, pos, freqs, (5, 6))), [x] if constant else [x, dy])
    rx, ry = x.detach().double().cpu().requires_grad_(True), dy.detach().double().cpu().requires_grad_(True)
    want = torch.autograd.grad(penalty(rx, ry, plain), [rx] if constant else [rx, ry])
    for a, b in zip(got, want):
        assert ((a.double().cpu() - b).norm() / b.norm()).item() < 4e-6


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_raises(which, grad):
    """A tangent of any input, positions and frequencies among them, is refused, not dropped; with a level open and
    no tangent the call is the ordinary one."""
    from torch.autograd import forward_ad
    from fovi_amd.arch.rotary import rotary
    x, pos, g = _inputs(1, 4, 2, 16, 2, torch.float32, seed=21)
    args = [x, pos, torch.rand(8, generator=g).cuda()]
    want = rotary(*args, (4, 4))
    if grad and which == 0:
        x.requires_grad_(True)
    leaf = args[0].detach().requires_grad_(True)
    y = rotary(leaf, *args[1:], (4, 4))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(want), torch.ones_like(want)))
    with forward_ad.dual_level():
        assert torch.equal(rotary(*args, (4, 4)), want)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for off in (False, True):
            with torch.set_grad_enabled(not off), pytest.raises(NotImplementedError, match="forward mode"):
                rotary(*args, (4, 4))


@pytest.mark.parametrize("convert", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
                                     lambda m: torch.nn.Sequential(m).bfloat16()[0]])
def test_converted_modules_keep_their_frequencies(convert):
    """A reader in bf16 turns its heads as it did in fp32: frequencies are not parameters to be rounded."""
    from fovi_amd.arch.rotary import AxialRotary
    want = AxialRotary(64, (8, 12, 12), device="cpu").freqs
    got = convert(AxialRotary(64, (8, 12, 12), device="cpu")).freqs
    assert got.dtype == torch.float32 and torch.equal(got, want)


@pytest.mark.gpu
def test_converted_modules_turn_alike():
    from fovi_amd.arch.rotary import AxialRotary
    x, pos, _ = _inputs(2, 30, 3, 64, 3, torch.bfloat16, seed=22, spread=20.0)
    rope = AxialRotary(64, (8, 12, 12), device="cpu")
    want = rope.cuda()(x, pos)
    assert rope.freqs.is_cuda and torch.equal(rope.bfloat16()(x, pos), want)
    assert list(rope.state_dict()) == []


@pytest.mark.gpu
def test_learned_positions_without_gradients():
    """Positions and frequencies that are parameters are taken where no gradient is asked for."""
    from fovi_amd.arch.rotary import rotary
    x, pos, g = _inputs(2, 5, 3, 32, 2, torch.float32, seed=23)
    freqs = torch.rand(16, generator=g).cuda()
    want = rotary(x, pos, freqs, (8, 8))
    pos, freqs = torch.nn.Parameter(pos), torch.nn.Parameter(freqs)
    for args in ((x, pos, freqs.detach(), (8, 8)), (x, pos.detach(), freqs, (8, 8))):
        with torch.no_grad():
            assert torch.equal(rotary(*args), want)
        with pytest.raises(ValueError, match="no gradient"):
            rotary(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_capture(pairing, dtype):
    """Both directions captured; replayed with new inputs and positions and with work of its own between."""
    from fovi_amd.arch.rotary import rotary
    x, pos, g = _inputs(3, 70, 4, 64, 3, dtype, seed=24)
    freqs = torch.rand(32, generator=g).cuda() * 6
    dy = torch.randn(x.shape, generator=g).to(dtype).cuda()
    x.requires_grad_(True)

    def step():
        y = rotary(x, pos, freqs, (8, 12, 12), pairing)
        return (y.detach(),) + torch.autograd.grad(y, x, dy)

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
            for t in (x, dy, pos):
                t.copy_(torch.randn(t.shape, generator=g))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
