"""Cases of the operators with which queries read the tokens of several fixations: layer norm,
rotary positions on several axes, and cross attention to the tokens.

Where ``own`` is false, ``run`` computes an operator in elementary torch operations in fp32,
rounded once at the end; where it is true, it calls the framework's operators. ``exact`` gives
the definition in float64.

Kinds of case:

* ``norm``: tokens ``[rows, C]``; with ``train`` also the gradients of the tokens, weight and bias
  (parameters in fp32, as under autocast).
* ``rotary``: heads ``[B, L, H, D]`` rotated by angles ``positions[..., axis] * freqs``; with
  ``train`` also the gradient. Positions are (fixation number, row, column), the last two in
  [-1, 1], with 2 pi / 100 ** (j / n) as the frequencies of an axis of n pairs.
* ``attend``: queries ``[B, Lq, Hq, D]`` over states ``[B, Lk, Hk, D]``; ``ragged`` gives every
  image its own number of states, ``mask`` leaves pairs out, whole rows among them; with
  ``train`` also the gradients of queries, keys and values.
"""
import math

import torch

own = False

DEV = "cuda"
_DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-5


# ------------------------------------------------------------------------------ the cases ---
def listed():
    return [
        # tokens of one fixation of one image in front of a serving step: the call's latency
        dict(name="norm_tokens", kind="norm", rows=64, c=384, dtype="bf16", train=False),
        # every token of 512 views (128 images, 4 fixations) in training
        dict(name="norm_train", kind="norm", rows=512 * 256, c=384, dtype="bf16", train=True),
        # fp32 training at a width that no vector load divides
        dict(name="norm_odd", kind="norm", rows=7421, c=771, dtype="fp32", train=True),
        # the query tokens of one serving step
        dict(name="rotary_step", kind="rotary", batch=64, length=1, heads=6, dim=64, sections="8 12 12",
             pairing="half", heads_first=False, dtype="bf16", train=False),
        # keys of 4 fixations of 256 tokens of each of 128 images, with the gradient
        dict(name="rotary_views", kind="rotary", batch=128, length=1024, heads=6, dim=64, sections="8 12 12",
             pairing="half", heads_first=False, dtype="bf16", train=True),
        # fp32, part of the head, adjacent pairs, heads before tokens in memory
        dict(name="rotary_odd", kind="rotary", batch=5, length=1283, heads=5, dim=80, sections="7 11 11",
             pairing="adjacent", heads_first=True, dtype="fp32", train=True),
        # one query over the 64 tokens of one fixation: the smallest call, latency
        dict(name="attend_one", kind="attend", batch=1, lq=1, lk=64, hq=6, hk=6, dim=64, dtype="bf16",
             ragged=False, mask=False, train=False),
        # one query token of each of 128 images over what it has seen, 1 to 20 fixations of 256 tokens
        dict(name="attend_step", kind="attend", batch=128, lq=1, lk=5120, hq=6, hk=6, dim=64, dtype="bf16",
             ragged=True, mask=False, train=False),
        # four query tokens over one long row of states, shared key heads: work only along the states
        dict(name="attend_long", kind="attend", batch=1, lq=4, lk=131072, hq=16, hk=4, dim=128, dtype="bf16",
             ragged=False, mask=False, train=False),
        # inference over 4 fixations, ragged
        dict(name="attend_forward", kind="attend", batch=64, lq=257, lk=1024, hq=6, hk=6, dim=64, dtype="bf16",
             ragged=True, mask=False, train=False),
        # training over 16 fixations: the largest
        dict(name="attend_train", kind="attend", batch=32, lq=1024, lk=4096, hq=6, hk=6, dim=64, dtype="bf16",
             ragged=False, mask=False, train=True),
        # fp32 training with a mask that leaves rows empty, shared key heads, odd lengths
        dict(name="attend_masked", kind="attend", batch=8, lq=77, lk=515, hq=8, hk=2, dim=32, dtype="fp32",
             ragged=True, mask=True, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "rotary", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "norm":
        c = _log(rng, 17, 4096)
        if rng.random() < 0.5:
            c = 8 * max(1, c // 8)
        rows = min(_log(rng, 1, 512 * 256), 512 * 256 * 384 // (2 * c) if dtype == "fp32" else 512 * 256 * 384 // c)
        return dict(kind=kind, rows=rows, c=c, dtype=dtype, train=rng.random() < 0.5)
    if kind == "rotary":
        dim = rng.choice([32, 64, 64, 80, 128])
        axes = rng.choice([1, 2, 3])
        pairs = dim // 2 - (rng.randint(0, dim // 8) if rng.random() < 0.5 else 0)
        first = pairs // (axes + 1)
        sections = {1: (pairs,), 2: (pairs // 2, pairs - pairs // 2), 3: (pairs - 2 * first, first, first)}[axes]
        sections = " ".join(str(n) for n in sections)
        heads, batch = rng.randint(1, 16), _log(rng, 1, 128)
        most = 128 * 1024 * 6 * 64 // (2 if dtype == "fp32" else 1)
        length = max(1, min(_log(rng, 1, 8192), most // (heads * batch * dim)))
        return dict(kind=kind, batch=batch, length=length, heads=heads, dim=dim, sections=sections,
                    pairing=rng.choice(["half", "adjacent"]), heads_first=rng.random() < 0.3, dtype=dtype,
                    train=rng.random() < 0.5)
    while True:
        hk = rng.choice([1, 2, 4, 6, 8])
        step = rng.random() < 0.35
        case = dict(kind=kind, batch=_log(rng, 1, 128), lq=rng.randint(1, 4) if step else _log(rng, 5, 4096),
                    lk=_log(rng, 1, 131072 if step else 8192), hq=hk * rng.choice([1, 1, 2, 4]), hk=hk,
                    dim=rng.choice([32, 64, 64, 80, 128]), dtype=dtype, ragged=rng.random() < 0.5,
                    mask=not step and rng.random() < 0.3, train=not step and rng.random() < 0.5)
        w = work(dict(case, ragged=False))
        pairs = case["batch"] * case["hq"] * case["lq"] * case["lk"]
        most = 32 * 6 * 1024 * 4096 // (8 if dtype == "fp32" else 1)
        if pairs * case["dim"] <= most * 64 and pairs <= most and w["bytes"] <= 2.2e9:
            return case


# ----------------------------------------------------------------------------- the inputs ---
def _sections(case):
    """Pairs of each axis."""
    return tuple(int(n) for n in case["sections"].split())


def _lengths(case):
    """Numbers of states, evenly from a twentieth of the longest up to it."""
    b, lk = case["batch"], case["lk"]
    if not case["ragged"]:
        return [lk] * b
    lo = max(1, lk // 20)
    return [lk - (lk - lo) * i // max(1, b - 1) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    s = {"case": case}

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if case["kind"] == "norm":
        rows, c = case["rows"], case["c"]
        # a residual stream: token scales and channel offsets differ
        x = randn(rows, c) * (0.5 + torch.rand(rows, 1, generator=g, device=DEV)) + 0.5 * randn(c)
        s["x"] = x.to(dt)
        s["weight"], s["bias"] = 1 + 0.1 * randn(c), 0.1 * randn(c)
        if case["train"]:
            s["dy"] = randn(rows, c).to(dt)
    elif case["kind"] == "rotary":
        b, n, h, d = case["batch"], case["length"], case["heads"], case["dim"]

        def heads():
            return (randn(b, h, n, d).to(dt).transpose(1, 2) if case["heads_first"] else randn(b, n, h, d).to(dt))

        s["x"] = heads()
        if case["train"]:
            s["dy"] = heads()
        axes = len(_sections(case))
        pos = 2 * torch.rand(b, n, axes, generator=g, device=DEV) - 1
        pos[..., 0] = (torch.arange(n, device=DEV) // 256).float()    # the fixation's number
        s["positions"] = pos
        s["freqs"] = torch.cat([2 * math.pi * 100.0 ** (-torch.arange(m, device=DEV).float() / m)
                                for m in _sections(case)])
    else:
        b, lq, lk, hq, hk, d = (case[x] for x in ("batch", "lq", "lk", "hq", "hk", "dim"))
        # scores of a trained head spread wider than those of independent normal vectors
        s["q"] = (1.5 * randn(b, lq, hq, d)).to(dt)
        s["k"], s["v"] = randn(b, lk, hk, d).to(dt), randn(b, lk, hk, d).to(dt)
        s["kv_lengths"] = s["mask"] = None
        if case["ragged"]:
            order = torch.randperm(b, generator=g, device=DEV)
            s["kv_lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)[order]
        if case["mask"]:
            mask = torch.rand(b, 1, lq, lk, generator=g, device=DEV) < 0.7
            mask[:, :, 3::13] = False                                 # queries with nothing to read
            s["mask"] = mask
        if case["train"]:
            s["dout"] = randn(b, lq, hq, d).to(dt)
    return s


# --------------------------------------------------------------------- the plain operators ---
def _plain_norm(x, weight, bias, dy):
    xf = x.float()
    centred = xf - xf.mean(-1, keepdim=True)
    r = (centred.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    h = centred * r
    y = (h * weight + bias).to(x.dtype)
    if dy is None:
        return y
    dyf = dy.float()
    g = dyf * weight
    dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype), "dweight": (dyf * h).sum(0), "dbias": dyf.sum(0)}


def _plain_rotate(x, cos, sin, pairing):
    """``x [B, L, H, D]`` by the angles of ``cos``/``sin [B, L, 1, P]``."""
    p = cos.shape[-1]
    xf = x.float()
    turned, rest = xf[..., :2 * p], xf[..., 2 * p:]
    u, v = (turned[..., :p], turned[..., p:]) if pairing == "half" else (turned[..., ::2], turned[..., 1::2])
    a, b = u * cos - v * sin, v * cos + u * sin
    turned = torch.cat([a, b], -1) if pairing == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _plain_rotary(x, positions, freqs, sections, pairing, dy):
    axis = torch.repeat_interleave(torch.arange(len(sections), device=x.device),
                                   torch.tensor(sections, device=x.device), output_size=sum(sections))
    angle = (positions[..., axis] * freqs)[:, :, None]
    cos, sin = angle.cos(), angle.sin()
    y = _plain_rotate(x, cos, sin, pairing)
    return y if dy is None else {"y": y, "dx": _plain_rotate(dy, cos, -sin, pairing)}


def _plain_attend(q, k, v, kv_lengths, mask, dout):
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1:3]
    scale = 1 / math.sqrt(d)
    # the heads that share keys lie in the rows of one product
    qf = q.float().transpose(1, 2).reshape(b, hk, -1, d)
    kf, vf = k.float().transpose(1, 2), v.float().transpose(1, 2)
    s = (qf @ kf.transpose(2, 3) * scale).reshape(b, hq, lq, lk)
    if kv_lengths is not None:
        s = s.masked_fill(torch.arange(lk, device=q.device) >= kv_lengths[:, None, None, None], -math.inf)
    if mask is not None:
        s = s.masked_fill(~mask, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = (s - top.masked_fill(top == -math.inf, 0)).exp()
    total = e.sum(-1, keepdim=True)
    p = (e / total.masked_fill(total == 0, 1)).reshape(b, hk, -1, lk)
    o = p @ vf

    def rows(t, like):
        return t.reshape(b, hq, lq, d).transpose(1, 2).to(like.dtype)

    if dout is None:
        return rows(o, q)
    do = dout.float().transpose(1, 2).reshape(b, hk, -1, d)
    ds = p * (do @ vf.transpose(2, 3) - (do * o).sum(-1, keepdim=True)) * scale
    return {"out": rows(o, q), "dq": rows(ds @ kf, q),
            "dk": (ds.transpose(2, 3) @ qf).transpose(1, 2).to(k.dtype),
            "dv": (p.transpose(2, 3) @ do).transpose(1, 2).to(v.dtype)}


# -------------------------------------------------------------------------------- the pass ---
def _leaf(t):
    """The same values as the input of a training step."""
    return t.detach().requires_grad_(True)


def _run_own(s):
    case = s["case"]
    train = case["train"]
    if case["kind"] == "norm":
        from fovi_amd.arch.norm import layer_norm
        if not train:
            return layer_norm(s["x"], s["weight"], s["bias"], _EPS)
        x, w, b = _leaf(s["x"]), _leaf(s["weight"]), _leaf(s["bias"])
        y = layer_norm(x, w, b, _EPS)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if case["kind"] == "rotary":
        from fovi_amd.arch.rotary import rotary
        args = s["positions"], s["freqs"], _sections(case), case["pairing"]
        if not train:
            return rotary(s["x"], *args)
        x = _leaf(s["x"])
        y = rotary(x, *args)
        (dx,) = torch.autograd.grad(y, (x,), s["dy"])
        return {"y": y.detach(), "dx": dx}
    from fovi_amd.arch.attention import cross_attention
    if not train:
        return cross_attention(s["q"], s["k"], s["v"], kv_lengths=s["kv_lengths"], mask=s["mask"])
    q, k, v = _leaf(s["q"]), _leaf(s["k"]), _leaf(s["v"])
    out = cross_attention(q, k, v, kv_lengths=s["kv_lengths"], mask=s["mask"])
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def run(state):
    if own:
        return _run_own(state)
    s, case = state, state["case"]
    with torch.no_grad():
        if case["kind"] == "norm":
            return _plain_norm(s["x"], s["weight"], s["bias"], s.get("dy"))
        if case["kind"] == "rotary":
            return _plain_rotary(s["x"], s["positions"], s["freqs"], _sections(case), case["pairing"], s.get("dy"))
        return _plain_attend(s["q"], s["k"], s["v"], s["kv_lengths"], s["mask"], s.get("dout"))


# ------------------------------------------------------------------------------- its work ---
def work(case):
    """Inputs read once, outputs written once; the operations of the definition."""
    es = 4 if case["dtype"] == "fp32" else 2
    train = case["train"]
    if case["kind"] == "norm":
        n = case["rows"] * case["c"]
        return {"bytes": n * es * (4 if train else 2) + case["c"] * (16 if train else 8),
                "flops": (20.0 if train else 8.0) * n}
    if case["kind"] == "rotary":
        tokens = case["batch"] * case["length"]
        n = tokens * case["heads"] * case["dim"]
        return {"bytes": n * es * (4 if train else 2) + 4 * tokens * len(_sections(case)),
                "flops": (6.0 if train else 3.0) * n}
    b, lq, lk, hq, hk, d = (case[x] for x in ("batch", "lq", "lk", "hq", "hk", "dim"))
    states = sum(_lengths(case))
    queries = b * lq * hq * d
    kv = 2 * states * hk * d
    out = 2 * b * lk * hk * d if train else 0                     # dk and dv, in full
    masks = b * lq * lk if case["mask"] else 0
    return {"bytes": es * (queries * (4 if train else 2) + kv + out) + masks,
            "flops": (14.0 if train else 4.0) * hq * lq * d * states}


# -------------------------------------------------------------------------------- its truth ---
def _exact_norm(s):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    mean = x.mean(-1, keepdim=True)
    std = (x.var(-1, unbiased=False, keepdim=True) + _EPS).sqrt()
    h = (x - mean) / std
    y = h * w + b
    if "dy" not in s:
        return y
    dy = s["dy"].double()
    dh = dy * w
    c = x.shape[-1]
    dx = (c * dh - dh.sum(-1, keepdim=True) - h * (dh * h).sum(-1, keepdim=True)) / (c * std)
    return {"y": y, "dx": dx, "dweight": (dy * h).sum(0), "dbias": dy.sum(0)}


def _exact_rotary(s):
    case = s["case"]
    p = sum(_sections(case))
    # each pair as a complex number, turned by exp(i angle)
    parts, at = [], 0
    for axis, n in enumerate(_sections(case)):
        parts.append(s["positions"][..., axis:axis + 1].double() * s["freqs"][at:at + n].double())
        at += n
    angle = torch.cat(parts, -1)[:, :, None]

    def turn(x, angle):
        x = x.double().clone()
        at = (slice(0, p), slice(p, 2 * p)) if case["pairing"] == "half" else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
        z = torch.complex(x[..., at[0]], x[..., at[1]]) * torch.polar(torch.ones_like(angle), angle)
        x[..., at[0]], x[..., at[1]] = z.real, z.imag
        return x

    y = turn(s["x"], angle)
    return {"y": y, "dx": turn(s["dy"], -angle)} if "dy" in s else y


def _exact_attend(s):
    case = s["case"]
    b, lq, lk, hq, hk, d = (case[x] for x in ("batch", "lq", "lk", "hq", "hk", "dim"))
    lengths = [lk] * b if s["kv_lengths"] is None else s["kv_lengths"].tolist()
    train = "dout" in s
    out = {"out": torch.zeros(b, lq, hq, d, dtype=torch.float64, device=DEV)}
    if train:
        out.update(dq=torch.zeros_like(out["out"]),
                   dk=torch.zeros(b, lk, hk, d, dtype=torch.float64, device=DEV),
                   dv=torch.zeros(b, lk, hk, d, dtype=torch.float64, device=DEV))
    for i in range(b):
        n = lengths[i]
        keep = torch.ones(lq, n, dtype=torch.bool, device=DEV) if s["mask"] is None else s["mask"][i, 0, :, :n]
        some = keep.any(-1, keepdim=True)
        for h in range(hq):
            j = h * hk // hq
            q, k, v = s["q"][i, :, h].double(), s["k"][i, :n, j].double(), s["v"][i, :n, j].double()
            z = (q @ k.T / d ** 0.5).masked_fill(~keep, -math.inf)
            p = torch.where(some, torch.softmax(z.masked_fill(~some, 0), -1), 0)
            o = p @ v
            out["out"][i, :, h] = o
            if train:
                do = s["dout"][i, :, h].double()
                dp = do @ v.T
                dz = p * (dp - (p * dp).sum(-1, keepdim=True)) / d ** 0.5
                out["dq"][i, :, h] = dz @ k
                out["dk"][i, :n, j] += dz.T @ q
                out["dv"][i, :n, j] += p.T @ do
    return out if train else out["out"]


def exact(case, seed):
    if case["kind"] == "attend" and case["batch"] * case["hq"] > 2048:
        return None                                       # a loop over the heads of every image
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "rotary": _exact_rotary, "attend": _exact_attend}[case["kind"]](s)
