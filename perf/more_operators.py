"""Cases of the feed-forward half of a token block: RMS norm with the residual's addition, the gated
feed-forward block, and products of 8-bit integers with a scale for each token and channel.

Where ``own`` is false, ``run`` computes an operator in elementary torch operations in fp32,
rounded once at the end; where it is true, it calls the framework's operators. ``exact`` gives
the definition in float64.

Kinds of case:

* ``norm``: ``total = x + residual`` (in the type of x), ``y = total / sqrt(mean(total^2) + eps) * weight``
  of tokens ``[rows, C]``, the weight in fp32. ``mode``: 'forward'; 'train', with the gradients of x (which
  is the residual's too) and weight; 'int8', where y is held in 8 bits with a scale a row: the scales and the
  values it stands for are the outputs.
* ``product``: int8 tokens ``[rows, k]`` with a scale each by int8 weights ``[n, k]`` with a scale a row;
  ``gated``: silu of one such product times another; ``extras``: bias and residual.
* ``mlp``: ``(act(x Wg^T) * (x Wu^T)) Wd^T`` of tokens ``[rows, C]``, with ``residual`` the residual's addition;
  ``train``: also the gradients of x and of the three weights.
"""
import math

import torch

own = False

DEV = "cuda"
_DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-6


# ------------------------------------------------------------------------------ the cases ---
def listed():
    return [
        # the tokens of one serving step, in front of a product in 8 bits: latency
        dict(name="norm_step", kind="norm", rows=64, c=384, dtype="bf16", mode="int8", residual=True),
        # every token of 512 views (128 images, 4 fixations) in training, behind the attention
        dict(name="norm_train", kind="norm", rows=512 * 256, c=384, dtype="bf16", mode="train", residual=True),
        # fp32 training at a width that no vector load divides, the block's first norm
        dict(name="norm_odd", kind="norm", rows=7421, c=771, dtype="fp32", mode="train", residual=False),
        # many tokens of a wider model in 8-bit serving
        dict(name="norm_int8", kind="norm", rows=32768, c=1024, dtype="bf16", mode="int8", residual=True),
        # one token by the weights of an output projection: the smallest product, latency
        dict(name="int8_token", kind="product", rows=1, k=1024, n=384, gated=False, extras=True, out="bf16"),
        # the tokens of a serving step by a wide layer: the weights' bytes
        dict(name="int8_few", kind="product", rows=48, k=4096, n=11008, gated=False, extras=False, out="bf16"),
        # both first projections for every token of 64 images
        dict(name="int8_gated", kind="product", rows=16384, k=1024, n=2752, gated=True, extras=False, out="bf16"),
        # odd sizes, fp32 outputs
        dict(name="int8_odd", kind="product", rows=2571, k=771, n=1537, gated=False, extras=True, out="fp32"),
        # one token in bf16 serving: latency
        dict(name="mlp_token", kind="mlp", rows=1, c=384, hidden=1024, dtype="bf16", act="silu", residual=True, train=False),
        # the tokens of a serving step in a wide block: the weights' bytes
        dict(name="mlp_few", kind="mlp", rows=32, c=2048, hidden=5504, dtype="bf16", act="silu", residual=True, train=False),
        # every token of 512 views in training: the largest
        dict(name="mlp_train", kind="mlp", rows=512 * 256, c=384, hidden=1024, dtype="bf16", act="silu", residual=False,
             train=True),
        # fp32 training, odd sizes, the other activation
        dict(name="mlp_odd", kind="mlp", rows=2571, c=387, hidden=1031, dtype="fp32", act="gelu", residual=False, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step):
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.4 else step * max(1, n // step)


def draw(rng):
    kind = rng.choice(["norm", "product", "mlp"])
    if kind == "norm":
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        c = _size(rng, 17, 8192, 64)
        rows = max(1, min(_log(rng, 1, 512 * 256), 512 * 256 * 384 // (c * (2 if dtype == "fp32" else 1))))
        return dict(kind=kind, rows=rows, c=c, dtype=dtype, mode=rng.choice(["forward", "train", "int8"]),
                    residual=rng.random() < 0.6)
    if kind == "product":
        k, n = _size(rng, 64, 8192, 64), _size(rng, 64, 11008, 64)
        rows = rng.randint(1, 64) if rng.random() < 0.4 else _log(rng, 65, 32768)
        gated = rng.random() < 0.4
        rows = max(1, min(rows, 16384 * 1024 * 2752 * 2 // (k * n * (2 if gated else 1))))
        return dict(kind=kind, rows=rows, k=k, n=n, gated=gated, extras=not gated and rng.random() < 0.5,
                    out=rng.choice(["bf16", "bf16", "fp32"]))
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    c, hidden = _size(rng, 64, 2048, 64), _size(rng, 64, 5504, 64)
    few = rng.random() < 0.3
    rows = rng.randint(1, 64) if few else _log(rng, 65, 512 * 256)
    rows = max(1, min(rows, 512 * 256 * 384 * 1024 // (c * hidden * (8 if dtype == "fp32" else 1)), 512 * 256 * 1024 // max(c, hidden)))
    return dict(kind=kind, rows=rows, c=c, hidden=hidden, dtype=dtype, act=rng.choice(["silu", "silu", "gelu"]),
                residual=rng.random() < 0.5, train=not few and rng.random() < 0.6)


# ----------------------------------------------------------------------------- the inputs ---
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"case": case}

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    def rows8(n, k):
        """Normal rows in 8 bits: the largest of each is 127 steps."""
        x = randn(n, k)
        scale = x.abs().amax(-1) / 127
        return (x / scale[:, None]).round().to(torch.int8), scale * (0.5 + torch.rand(n, generator=g, device=DEV))

    if case["kind"] == "norm":
        rows, c, dt = case["rows"], case["c"], _DT[case["dtype"]]
        # a residual stream: token scales and channel offsets differ
        stream = randn(rows, c) * (0.5 + torch.rand(rows, 1, generator=g, device=DEV)) + 0.5 * randn(c)
        s["weight"] = 1 + 0.1 * randn(c)
        s["x"], s["residual"] = stream.to(dt), None
        if case["residual"]:
            s["x"], s["residual"] = (0.3 * randn(rows, c)).to(dt), s["x"]
        if case["mode"] == "train":
            s["dy"] = randn(rows, c).to(dt)
            s["dtotal"] = randn(rows, c).to(dt) if case["residual"] else None
    elif case["kind"] == "product":
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"], s["x_scale"] = rows8(rows, k)
        s["w"], s["w_scale"] = rows8(n, k)
        s["w_scale"] = s["w_scale"] / math.sqrt(k)
        if case["gated"]:
            s["w2"], s["w2_scale"] = rows8(n, k)
            s["w2_scale"] = s["w2_scale"] / math.sqrt(k)
        s["bias"] = randn(n) if case["extras"] else None
        s["residual"] = randn(rows, n).to(_DT[case["out"]]) if case["extras"] else None
    else:
        rows, c, f, dt = case["rows"], case["c"], case["hidden"], _DT[case["dtype"]]
        s["x"] = randn(rows, c).to(dt)
        s["w_gate"], s["w_up"] = (randn(f, c) / math.sqrt(c)).to(dt), (randn(f, c) / math.sqrt(c)).to(dt)
        s["w_down"] = (randn(c, f) / math.sqrt(f)).to(dt)
        s["residual"] = randn(rows, c).to(dt) if case["residual"] else None
        if case["train"]:
            s["dy"] = randn(rows, c).to(dt)
    return s


# --------------------------------------------------------------------- the plain operators ---
def _plain_norm(s):
    x, mode = s["x"], s["case"]["mode"]
    total = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    t = total.float()
    r = (t.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    h = t * r
    y = h * s["weight"]
    out = {} if s["residual"] is None else {"total": total}
    if mode == "int8":
        top = y.abs().amax(-1, keepdim=True)
        scale = top / 127
        q = torch.where(top > 0, y / scale, 0).round()
        return {**out, "y": (q * scale).to(torch.bfloat16), "scale": scale[:, 0]}
    out["y"] = y.to(x.dtype)
    if mode == "train":
        dyf = s["dy"].float()
        g = dyf * s["weight"]
        dx = r * (g - h * (g * h).mean(-1, keepdim=True))
        if s["dtotal"] is not None:
            dx = dx + s["dtotal"].float()
        out.update(dx=dx.to(x.dtype), dweight=(dyf * h).sum(0))
    return out


def _plain_act(z, act):
    if act == "silu":
        return z / (1 + (-z).exp())
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))


def _plain_act_grad(z, act):
    if act == "silu":
        sig = 1 / (1 + (-z).exp())
        return sig * (1 + z * (1 - sig))
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * (-0.5 * z * z).exp() / math.sqrt(2 * math.pi)


def _plain_product(s):
    xf = s["x"].float()

    def by(w, scale):
        return xf @ w.float().T * s["x_scale"][:, None] * scale

    y = by(s["w"], s["w_scale"])
    if s["case"]["gated"]:
        y = _plain_act(y, "silu") * by(s["w2"], s["w2_scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(_DT[s["case"]["out"]])


def _plain_mlp(s):
    case, dt = s["case"], s["x"].dtype
    act = case["act"]
    x, wg, wu, wd = (s[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    gate, up = x @ wg.T, x @ wu.T
    a = _plain_act(gate, act)
    h = a * up
    y = h @ wd.T
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not case["train"]:
        return y.to(dt)
    dy = s["dy"].float()
    dh = dy @ wd
    dgate, dup = dh * up * _plain_act_grad(gate, act), dh * a
    return {"y": y.to(dt), "dx": (dgate @ wg + dup @ wu).to(dt), "dw_gate": (dgate.T @ x).to(dt),
            "dw_up": (dup.T @ x).to(dt), "dw_down": (dy.T @ h).to(dt)}


# -------------------------------------------------------------------------------- the pass ---
def _leaf(t):
    """The same values as the input of a training step."""
    return t.detach().requires_grad_(True)


def _own_norm(s):
    from fovi_amd.arch.norm import rms_norm, rms_norm_int8
    x, residual, weight = s["x"], s["residual"], s["weight"]
    mode = s["case"]["mode"]
    if mode == "int8":
        q = rms_norm_int8(x, weight, _EPS, residual=residual)
        q, out = (q, {}) if residual is None else (q[0], {"total": q[1]})
        return {**out, "y": q.dequantize(torch.bfloat16), "scale": q.scale}
    if mode == "forward":
        y = rms_norm(x, weight, _EPS, residual=residual)
        return {"y": y} if residual is None else {"y": y[0], "total": y[1]}
    x, weight = _leaf(x), _leaf(weight)
    if residual is None:
        y = rms_norm(x, weight, _EPS)
        dx, dw = torch.autograd.grad(y, (x, weight), s["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw}
    residual = _leaf(residual)
    y, total = rms_norm(x, weight, _EPS, residual=residual)
    dx, _, dw = torch.autograd.grad((y, total), (x, residual, weight), (s["dy"], s["dtotal"]))
    return {"y": y.detach(), "total": total.detach(), "dx": dx, "dweight": dw}


def _own_product(s):
    from fovi_amd.arch.int8 import Int8Rows, gated_linear_int8, linear_int8
    x, w, dt = Int8Rows(s["x"], s["x_scale"]), Int8Rows(s["w"], s["w_scale"]), _DT[s["case"]["out"]]
    if s["case"]["gated"]:
        return gated_linear_int8(x, w, Int8Rows(s["w2"], s["w2_scale"]), activation="silu", dtype=dt)
    return linear_int8(x, w, bias=s["bias"], residual=s["residual"], dtype=dt)


def _own_mlp(s):
    from fovi_amd.arch.feed_forward import gated_mlp
    case = s["case"]
    names = ("x", "w_gate", "w_up", "w_down")
    if not case["train"]:
        return gated_mlp(*(s[n] for n in names), activation=case["act"], residual=s["residual"])
    leaves = [_leaf(s[n]) for n in names]
    y = gated_mlp(*leaves, activation=case["act"], residual=s["residual"])
    grads = torch.autograd.grad(y, leaves, s["dy"])
    return {"y": y.detach(), **dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), grads))}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "product": _own_product, "mlp": _own_mlp}[kind](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "product": _plain_product, "mlp": _plain_mlp}[kind](state)


# ------------------------------------------------------------------------------- its work ---
def work(case):
    """Inputs read once, outputs written once; the operations of the definition."""
    if case["kind"] == "norm":
        es = 4 if case["dtype"] == "fp32" else 2
        n = case["rows"] * case["c"]
        train = case["mode"] == "train"
        # x (and residual, total); y or its 8 bits and scales; dy (and dtotal), dx
        size = n * es * (3 if case["residual"] else 1) + (n + 4 * case["rows"] if case["mode"] == "int8" else n * es)
        if train:
            size += n * es * (3 if case["residual"] else 2)
        return {"bytes": size + case["c"] * (8 if train else 4), "flops": (14.0 if train else 5.0) * n}
    if case["kind"] == "product":
        m, k, n, es = case["rows"], case["k"], case["n"], 4 if case["out"] == "fp32" else 2
        two = 2 if case["gated"] else 1
        extras = n * 4 + m * n * es if case["extras"] else 0
        return {"bytes": m * (k + 4) + two * n * (k + 4) + m * n * es + extras, "flops": 2.0 * two * m * n * k}
    m, c, f, es = case["rows"], case["c"], case["hidden"], 4 if case["dtype"] == "fp32" else 2
    tokens = 2 + (1 if case["residual"] else 0) + (2 if case["train"] else 0)
    return {"bytes": es * (m * c * tokens + 3 * c * f * (2 if case["train"] else 1)),
            "flops": (18.0 if case["train"] else 6.0) * m * c * f}


# -------------------------------------------------------------------------------- its truth ---
def _exact_norm(s):
    x, w = s["x"].double(), s["weight"].double()
    c, mode = x.shape[-1], s["case"]["mode"]
    out = {}
    if s["residual"] is not None:
        total = s["x"] + s["residual"]                         # a sum of two numbers, rounded once
        out["total"], x = total.double(), total.double()
    norm = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
    rms = (norm * norm / c + _EPS).sqrt()
    y = x / rms * w
    if mode == "int8":
        top = torch.linalg.vector_norm(y, ord=math.inf, dim=-1)
        step = top[:, None] / 127
        return {**out, "y": torch.where(step > 0, torch.round(y / step) * step, 0), "scale": step[:, 0]}
    out["y"] = y
    if mode == "train":
        dy = s["dy"].double()
        dh = dy * w
        # y_i = w_i x_i / rms, d rms / d x_j = x_j / (c rms)
        dx = dh / rms - x * (dh * x).sum(-1, keepdim=True) / (c * rms ** 3)
        if s["dtotal"] is not None:
            dx += s["dtotal"].double()
        out.update(dx=dx, dweight=torch.einsum("rc,rc->c", dy, x / rms))
    return out


def _exact_product(s):
    x = s["x"].double() * s["x_scale"].double()[:, None]
    y = torch.nn.functional.linear(x, s["w"].double() * s["w_scale"].double()[:, None])
    if s["case"]["gated"]:
        y = y * torch.sigmoid(y) * torch.nn.functional.linear(x, s["w2"].double() * s["w2_scale"].double()[:, None])
    for t in (s["bias"], s["residual"]):
        if t is not None:
            y = y + t.double()
    return y


def _exact_mlp(s):
    train = s["case"]["train"]
    x, wg, wu, wd = (s[n].double().requires_grad_(train) for n in ("x", "w_gate", "w_up", "w_down"))
    f = torch.nn.functional
    act = {"silu": f.silu, "gelu": f.gelu}[s["case"]["act"]]
    with torch.set_grad_enabled(train):
        y = f.linear(act(f.linear(x, wg)) * f.linear(x, wu), wd)
        if s["residual"] is not None:
            y = y + s["residual"].double()
    if not train:
        return y
    grads = torch.autograd.grad(y, (x, wg, wu, wd), s["dy"].double())
    return {"y": y.detach(), **dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), grads))}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "product": _exact_product, "mlp": _exact_mlp}[case["kind"]](s)
