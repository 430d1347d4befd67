"""Products of 8-bit rows with 8-bit weights, against float64 (where the integer sums are exact).

Tolerances, from the arithmetic. The integer sum is exact and becomes a float once (2^-24 of it); times two scales, plus bias
and residual: with the rounding of each step, 6 * 2^-24 of the sum of the parts' magnitudes. Outputs are rounded once more (u,
half a step: 2^-24 or 2^-8 of the value). The gate's exponential and reciprocal add 2^-20 of the value and, by the error of the
exponent's argument, 2^-22 (1 + |gate|) of it.
"""
import pytest
import torch

from fovi_amd import _lib

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24


def _rows(n, k, seed):
    from fovi_amd.arch.int8 import Int8Rows
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8)
    return Int8Rows(q.cuda(), (0.01 * (0.5 + torch.rand(n, generator=g))).cuda())


def _sum(x, w):
    """The product times the scales, in float64 (sums of integers below 2^53 are exact there)."""
    return (x.data.double() @ w.data.double().t()) * x.scale.double()[:, None] * w.scale.double()


def _within(got, want, bound, what):
    assert got.shape == want.shape
    over = ((got.double() - want).abs() - bound).max().item()
    assert over <= 0, f"{what}: {over:.3e} over the bound"


def _act(z, name):
    return z / (1 + (-z).exp()) if name == "silu" else 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))


SIZES = [(1, 1, 1), (1, 64, 384), (1, 4096, 100), (2, 16, 16), (3, 17, 5), (16, 1024, 384), (17, 771, 33), (48, 2048, 1003), (64, 128, 129),
         (65, 128, 128), (100, 15, 64), (129, 129, 257), (300, 771, 1537), (1000, 640, 384), (257, 8192, 70), (513, 384, 1024),
         (64, 12288, 40), (2000, 96, 2752), (1, 65536, 17), (40, 33000, 3), (70, 80, 16500),
         (200, 33, 4100), (200, 100, 257), (256, 640, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("extras", ["none", "bias", "residual", "both"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(m, k, n, extras, dtype):
    from fovi_amd.arch.int8 import linear_int8
    x, w = _rows(m, k, 1), _rows(n, k, 2)
    g = torch.Generator().manual_seed(3)
    bias = torch.randn(n, generator=g).cuda() if extras in ("bias", "both") else None
    residual = torch.randn(m, n, generator=g).to(dtype).cuda() if extras in ("residual", "both") else None
    y = linear_int8(x, w, bias=bias, residual=residual, dtype=dtype)
    want = _sum(x, w)
    parts = want.abs()
    for t in (bias, residual):
        if t is not None:
            want, parts = want + t.double(), parts + t.double().abs()
    _within(y, want, 1.01 * (U[dtype] * want.abs() + 6 * E * parts) + 1e-38, "y")
    assert torch.equal(linear_int8(x, w, bias=bias, residual=residual, dtype=dtype), y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_gated(m, k, n, activation, dtype):
    from fovi_amd.arch.int8 import Int8Rows, gated_linear_int8
    x, gate, up = _rows(m, k, 1), _rows(n, k, 2), _rows(n, k, 4)
    gate = Int8Rows(gate.data, gate.scale / (73 * k) ** 0.5)          # gates of a few units, where the activation bends
    y = gated_linear_int8(x, gate, up, activation, dtype)
    g, u = _sum(x, gate), _sum(x, up)
    want = _act(g, activation) * u
    # value of the gate: act' is at most 1.13, the sums are off by 4 E
    bound = U[dtype] * want.abs() + u.abs() * g.abs() * 1.13 * 4 * E + want.abs() * (4 * E + 2.0 ** -20 + 2.0 ** -22 * (1 + g.abs()))
    if activation == "gelu":                                             # 1 + erf cancels for negative gates
        bound = bound + (g * u).abs() * 4 * E
    _within(y, want, 1.01 * bound + 1e-38, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(5, 16), (40, 21), (300, 32)])
def test_gate_of_fp32_outputs(m, k):
    """Gates that are exact, between -40 and 40: what is left is the activation's. The library's exponential is off by 2^-23,
    the sum below it, the division, the product and the output by 2^-24 each, so 6 * 2^-24 in all. (An exponential of base 2 loses
    half a step of its argument, which is |gate| 2^-24 of its value.)"""
    from fovi_amd.arch.int8 import Int8Rows, gated_linear_int8
    n = 24
    x, gate, up = (torch.zeros(r, k, dtype=torch.int8) for r in (m, n, n))
    x[:, 0], x[:, 1] = (torch.arange(m) * 37 % 255 - 127).to(torch.int8), (1 + torch.arange(m) % 127).to(torch.int8)
    gate[:, 0], up[:, 1] = 1, (1 + torch.arange(n)).to(torch.int8)
    one = torch.ones(max(m, n), device="cuda")
    x, gate, up = Int8Rows(x.cuda(), one[:m]), Int8Rows(gate.cuda(), one[:n] * 0.3125), Int8Rows(up.cuda(), one[:n] * 0.125)
    y = gated_linear_int8(x, gate, up, "silu", torch.float32)
    want = _act(_sum(x, gate), "silu") * _sum(x, up)
    _within(y, want, 6 * E * want.abs(), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("k", [131071, 131056])
@pytest.mark.parametrize("m", [3, 70, 300])
def test_sums_are_exact(m, k):
    """Rows of -128 and 127 of the largest lengths (the second is of whole 16-byte pieces), whose sums come near 2^31, and one
    that nearly cancels."""
    from fovi_amd.arch.int8 import Int8Rows, linear_int8
    x = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.stack([torch.full((k,), v, dtype=torch.int8, device="cuda") for v in (-128, 127, 127)])
    w[2, : k // 2] = -127
    x[1, 0], w[2, 0] = 1, 1
    one = torch.ones(m, device="cuda")
    y = linear_int8(Int8Rows(x, one), Int8Rows(w, one[:1].expand(3)), dtype=torch.float32)
    want = (x.double() @ w.double().t()).float()
    assert torch.equal(y, want)
    assert y[0, 0] == 128.0 * 128 * k


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 200])
@pytest.mark.parametrize("layout", ["padded", "odd_offset", "tokens", "expanded", "columns"])
def test_layouts(m, layout):
    """Rows and weights where they are, whatever lies between and behind them; the values of the contiguous call."""
    from fovi_amd.arch.int8 import Int8Rows, linear_int8, gated_linear_int8
    g = torch.Generator().manual_seed(5)
    k, n = 83, 37

    def make(r, width, cols):
        t = torch.randint(-127, 128, (r, width), generator=g, dtype=torch.int32).to(torch.int8).cuda()
        return t[:, cols:cols + k]

    if layout == "padded":
        x, w, u = make(m, 96, 0), make(n, 96, 0), make(n, 128, 0)
    elif layout == "odd_offset":
        x, w, u = make(m, 101, 5), make(n, 90, 3), make(n, 97, 1)
    elif layout == "tokens":
        x, w, u = make(m * 2, 83, 0).view(2, m, k)[:, : m - 1], make(n, 83, 0), make(n, 83, 0)
    elif layout == "expanded":
        x, w, u = make(1, 83, 0).expand(m, k), make(1, 83, 0).expand(n, k), make(n, 83, 0)
    else:
        x, w, u = make(m, 83, 0), make(n, 83, 0).t().contiguous().t(), make(n, 83, 0)
    xs = torch.rand(x.shape[:-1] + (2,), generator=g).cuda()[..., 0]
    ws = torch.rand(n, 3, generator=g).cuda()[:, 1]
    residual = torch.randn(x.shape[:-1] + (n + 5,), generator=g).cuda()[..., 2:2 + n]
    bias = torch.randn(2 * n, generator=g).cuda()[::2]
    got = linear_int8(Int8Rows(x, xs), Int8Rows(w, ws), bias=bias, residual=residual, dtype=torch.float32)
    both = gated_linear_int8(Int8Rows(x, xs), Int8Rows(w, ws), Int8Rows(u, ws), dtype=torch.float32)
    c = [t.contiguous() for t in (x, xs, w, ws, u, residual, bias)]
    assert torch.equal(got, linear_int8(Int8Rows(c[0], c[1]), Int8Rows(c[2], c[3]), bias=c[6], residual=c[5], dtype=torch.float32))
    assert torch.equal(both, gated_linear_int8(Int8Rows(c[0], c[1]), Int8Rows(c[2], c[3]), Int8Rows(c[4], c[3]), dtype=torch.float32))
    want = (c[0].double() @ c[2].double().t()) * c[1].double()[..., None] * c[3].double() + c[6].double() + c[5].double()
    assert (got.double() - want).abs().max() <= 1e-5 * want.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(3, 100, 21), (70, 64, 100), (129, 77, 131), (300, 256, 260)])
def test_writes_its_rows_only(m, k, n):
    """Outputs of one stride inside a wider buffer: what lies around them keeps its value."""
    x, w = _rows(m, k, 1), _rows(n, k, 2)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((m + 2, n + 9), 7.0, dtype=dtype, device="cuda")
        y = out[1:-1, 3:3 + n]
        for two in (False, True):
            a = _lib.LinearInt8Args()
            a.x, a.x_scale, a.rows, a.inputs, a.outputs, a.x_stride = x.data.data_ptr(), x.scale.data_ptr(), m, k, n, k
            a.weight, a.weight_scale, a.weight_stride = w.data.data_ptr(), w.scale.data_ptr(), k
            if two:
                a.weight2, a.weight2_scale, a.weight2_stride = a.weight, a.weight_scale, k
            a.out, a.out_dtype, a.out_stride = y.data_ptr(), _lib.dtype_code(dtype), n + 9
            size = _lib.load().fovi_linear_int8_workspace_bytes(a)
            work = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
            a.workspace, a.workspace_bytes = work.data_ptr(), size
            _lib.check(_lib.load().fovi_linear_int8(a, _lib.stream_of(y)), "product")
            want = _sum(x, w)
            want = _act(want, "silu") * want if two else want
            assert (y.double() - want).abs().max() <= 5e-3 * want.abs().max()
            y.fill_(7.0)
            assert (out == 7.0).all()


@pytest.mark.gpu
def test_scales_that_are_not_finite_stay_in_their_rows():
    from fovi_amd.arch.int8 import Int8Rows, linear_int8, quantize_int8
    x = torch.randn(80, 64, device="cuda")
    x[7, 3] = float("inf")
    w = _rows(50, 64, 2)
    y = linear_int8(quantize_int8(x), w, dtype=torch.float32)
    assert y[7].isnan().all() and y[:7].isfinite().all() and y[8:].isfinite().all()


@pytest.mark.gpu
def test_empty():
    from fovi_amd.arch.int8 import linear_int8
    assert linear_int8(_rows(0, 8, 1), _rows(5, 8, 2)).shape == (0, 5)
    assert linear_int8(_rows(3, 8, 1), _rows(0, 8, 2)).shape == (3, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_module(dtype):
    """Against the same steps by hand, through a conversion of the module's type."""
    from fovi_amd.arch.int8 import Int8Linear, Int8Rows, linear_int8, quantize_int8
    torch.manual_seed(1)
    lin = torch.nn.Linear(72, 40, device="cuda")
    mod = Int8Linear(lin).bfloat16()
    x = torch.randn(3, 5, 72, device="cuda").to(dtype)
    r = torch.randn(3, 5, 40, device="cuda").to(dtype)
    with torch.no_grad():
        y = mod(x, residual=r)
        w = quantize_int8(lin.weight)
        assert torch.equal(y, linear_int8(quantize_int8(x), w, bias=lin.bias, residual=r, dtype=dtype))
        assert torch.equal(mod(quantize_int8(x)), linear_int8(quantize_int8(x), w, bias=lin.bias))
        # each side of every product is off by half a step, a 254th of its row's largest value
        exact = torch.nn.functional.linear(x.double(), lin.weight.double(), lin.bias.double()) + r.double()
    top = x.double().abs().amax(-1)[..., None] / 254
    wtop = lin.weight.double().abs().amax(-1) / 254
    bound = top * lin.weight.double().abs().sum(-1) + wtop * x.double().abs().sum(-1)[..., None] + 72 * top * wtop
    assert ((y.double() - exact).abs() <= 1.01 * bound + 2 * U[dtype] * exact.abs() + 1e-5).all()
    assert "72" in repr(mod) and mod.weight_scale.dtype == torch.float32
    other = Int8Linear(torch.nn.Linear(72, 40, device="cuda"))
    other.load_state_dict(mod.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x, residual=r), y)


@pytest.mark.gpu
def test_module_output_types():
    """Rows in 8 bits: the output's type is the residual's, bf16 without one, or what is asked for; other rows: their type, or that."""
    from fovi_amd.arch.int8 import Int8Linear, Int8Rows, linear_int8, quantize_int8
    torch.manual_seed(1)
    mod = Int8Linear(torch.nn.Linear(72, 40, device="cuda"))
    x, r = torch.randn(5, 72, device="cuda"), torch.randn(5, 40, device="cuda")
    q, w = quantize_int8(x), Int8Rows(mod.weight, mod.weight_scale)
    for dtype in (torch.float32, torch.bfloat16):
        want = linear_int8(q, w, bias=mod.bias, residual=r.to(dtype), dtype=dtype)
        assert torch.equal(mod(q, residual=r.to(dtype)), want)
        assert torch.equal(mod(q, residual=r.to(dtype), dtype=dtype), want)
        assert torch.equal(mod(x, residual=r.to(dtype), dtype=dtype), want)
        assert torch.equal(mod(q, dtype=dtype), linear_int8(q, w, bias=mod.bias, dtype=dtype))
    assert mod(q).dtype == torch.bfloat16 and mod(x).dtype == torch.float32
    with pytest.raises(ValueError, match="residual"):
        mod(q, residual=r, dtype=torch.bfloat16)


@pytest.mark.gpu
def test_stream_and_capture():
    """The smallest, few-row and tiled calls on another stream and captured, with their workspaces; replayed with new inputs."""
    from fovi_amd.arch.int8 import gated_linear_int8, linear_int8
    calls = [(_rows(m, k, 1), _rows(n, k, 2)) for m, k, n in ((1, 640, 40), (30, 4096, 100), (100, 2048, 128), (600, 128, 300))]

    def step():
        return [t for x, w in calls for t in (linear_int8(x, w), gated_linear_int8(x, w, w))]

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        for x, w in calls:
            x.data.copy_(torch.randint(-127, 128, x.data.shape, device="cuda", dtype=torch.int32).to(torch.int8))
            x.scale.uniform_(0.1, 1)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(40, 1024, 2 ** 21 + 100), (40, 1023, 2 ** 21 + 4200), (2 ** 21 + 70, 1024, 24), (2 ** 21 + 4200, 1023, 24),
                                   (70000, 16, 32000)])
def test_offsets_past_32_bits(m, k, n):
    """Weights, rows (as they are and copied) and outputs of more than 2^31 elements: the last rows and outputs as a small call
    gives them (the sums are exact)."""
    from fovi_amd.arch.int8 import Int8Rows, gated_linear_int8, linear_int8
    x, w = (Int8Rows(torch.randint(-127, 128, (r, k), dtype=torch.int8, device="cuda"), torch.rand(r, device="cuda")) for r in (m, n))
    a, b = Int8Rows(x.data[-33:].clone(), x.scale[-33:]), Int8Rows(w.data[-21:].clone(), w.scale[-21:])
    assert torch.equal(linear_int8(x, w)[-33:, -21:], linear_int8(a, b))
    assert torch.equal(gated_linear_int8(x, w, w)[-33:, -21:], gated_linear_int8(a, b, b))


@pytest.mark.gpu
def test_dequantize_asked_for_gradients():
    from torch.autograd import forward_ad
    from fovi_amd.arch.int8 import Int8Rows
    x = _rows(4, 16, 1)
    leaf = x.scale.clone().requires_grad_(True)
    with pytest.raises(ValueError, match="no gradients"):
        Int8Rows(x.data, leaf).dequantize()
    with torch.no_grad():
        assert torch.equal(Int8Rows(x.data, leaf).dequantize(), x.dequantize())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.scale, torch.ones_like(x.scale))
        with pytest.raises(ValueError, match="forward-mode"):
            Int8Rows(x.data, dual).dequantize()


@pytest.mark.gpu
def test_refusals():
    from fovi_amd.arch.int8 import Int8Rows, gated_linear_int8, linear_int8
    x, w = _rows(4, 16, 1), _rows(8, 16, 2)
    with pytest.raises(TypeError, match="dtype"):
        linear_int8(x, w, dtype=torch.float16)
    with pytest.raises(ValueError, match="weights"):
        linear_int8(x, _rows(8, 15, 2))
    with pytest.raises(ValueError, match="bias"):
        linear_int8(x, w, bias=torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError, match="residual"):
        linear_int8(x, w, residual=torch.zeros(4, 8, device="cuda"))
    with pytest.raises(ValueError, match="activation"):
        gated_linear_int8(x, w, w, "relu")
    with pytest.raises(ValueError, match="weights"):
        gated_linear_int8(x, w, _rows(7, 16, 3))
    with pytest.raises(TypeError, match="int8"):
        linear_int8(Int8Rows(x.data.float(), x.scale), w)
    with pytest.raises(ValueError, match="scales"):
        linear_int8(Int8Rows(x.data, x.scale[:3]), w)
    with pytest.raises(ValueError, match="no gradients"):
        linear_int8(x, w, bias=torch.zeros(8, device="cuda", requires_grad=True))
    with pytest.raises(ValueError, match="at most 131071"):
        linear_int8(_rows(1, 131072, 1), _rows(1, 131072, 1))


def test_cpu_tensors_and_c_arguments_are_refused():
    from fovi_amd.arch.int8 import Int8Rows, linear_int8
    x = Int8Rows(torch.zeros(2, 4, dtype=torch.int8), torch.zeros(2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_int8(x, x)
    lib = _lib.load()
    a = _lib.LinearInt8Args()
    assert lib.fovi_linear_int8(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.x = a.x_scale = a.weight = a.weight_scale = a.out = 16
    a.out_dtype = 9
    assert lib.fovi_linear_int8(a, None) != 0 and b"out_dtype" in lib.fovi_last_error()
    a.out_dtype, a.rows, a.outputs = _lib.F32, 1, 1
    assert lib.fovi_linear_int8(a, None) != 0 and b"bad sizes" in lib.fovi_last_error()
    a.inputs = 131072
    assert lib.fovi_linear_int8(a, None) != 0 and b"bad sizes" in lib.fovi_last_error()
    a.inputs, a.weight2 = 8, 16
    assert lib.fovi_linear_int8(a, None) != 0 and b"null pointer" in lib.fovi_last_error()
    a.weight2_scale, a.bias = 16, 16
    assert lib.fovi_linear_int8(a, None) != 0 and b"no bias" in lib.fovi_last_error()
    a.bias, a.activation = None, 5
    assert lib.fovi_linear_int8(a, None) != 0 and b"activation" in lib.fovi_last_error()


@pytest.mark.parametrize("k,n", [(16, 2 ** 31), (15, 2 ** 31), (1296, 2 ** 31), (1297, 2 ** 31)])
@pytest.mark.parametrize("two", [False, True])
def test_launches_past_the_limit_are_refused(k, n, two):
    """Outputs of one row for which the launch would have 2^32 threads or more. (The host refuses: nothing is read or launched.)"""
    lib, a = _lib.load(), _lib.LinearInt8Args()
    a.x = a.x_scale = a.weight = a.weight_scale = a.out = 16
    if two:
        a.weight2 = a.weight2_scale = 16
    a.rows, a.inputs, a.outputs, a.x_stride, a.weight_stride, a.weight2_stride, a.out_stride = 1, k, n, k, k, k, n
    assert lib.fovi_linear_int8(a, None) != 0 and b"exceed one launch" in lib.fovi_last_error()


def test_launch_is_on_the_tensors_device(monkeypatch):
    """An entry point runs with the device of its tensors as the current one, which it leaves as it was."""
    current, calls = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 100 + t.device.index)
    for index in (0, 1):
        t = type("T", (), {"device": torch.device("cuda", index)})()
        _lib.launch(lambda *a: calls.append((current[0],) + a) or 0, (7, 8), t, "entry")
    assert calls == [(0, 7, 8, 100), (1, 7, 8, 101)] and current == [0]
    with pytest.raises(RuntimeError, match="entry"):
        _lib.launch(lambda *a: 1, (), t, "entry")
    assert current == [0]
