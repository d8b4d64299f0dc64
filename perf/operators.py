"""Cases of the token-wise operators of a transformer block: rotary positions with several axes, layer norm
(forward, backward, and the backward pass of its adaLN form) and a Linear with bias, activation and residual.

``listed()`` names the cases and ``draw()`` makes more of the same ranges; ``prepare()`` makes what a caller has in
hand, ``run()`` is one pass (with ``own`` false in elementary torch operations, with ``own`` true through
``selas_b200.ops``), ``work()`` what a pass has to read, write and compute, and ``exact()`` the result in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "quick_gelu", "silu")


def rope_case(name, batch, text, frames, height, width, start, heads, kv_heads, axes, pairs, inverse, dtype, layout, ids):
    return {"name": name, "op": "rope", "batch": batch, "text": text, "frames": frames, "height": height, "width": width, "start": start,
            "heads": heads, "kv_heads": kv_heads, "axes": axes, "pairs": pairs, "inverse": inverse, "dtype": dtype, "layout": layout, "ids": ids}


def norm_case(name, op, batch, seq, dim, x, y, w, add):
    return {"name": name, "op": op, "batch": batch, "seq": seq, "dim": dim, "x": x, "y": y, "w": w, "add": add}


def linear_case(name, m, k, n, dtype, act, bias, residual, out):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "residual": residual, "out": out}


def listed():
    return [
        # one token far along a stream: what a cached or streamed video step rotates per token; latency is all of it
        rope_case("rope, one token", 1, 0, 1, 1, 1, 70000, 24, 24, "16,56,56", "interleaved", False, "bf16", "heads", "i64"),
        # a 1024 x 1024 image behind 512 text tokens, q and k read in place from the fused projection's rows
        rope_case("rope, 1024 image", 1, 512, 1, 64, 64, 0, 24, 24, "16,56,56", "interleaved", False, "bf16", "qkv", "f32"),
        # a clip of 16 latent frames of 48 x 80 tokens: the longest sequence
        rope_case("rope, clip", 1, 0, 16, 48, 80, 0, 24, 24, "44,42,42", "interleaved", False, "bf16", "heads", "i64"),
        # the gradient's direction, pairs in halves, keys of shared heads, an odd grid, fp32
        rope_case("rope, gradient, shared keys", 2, 0, 3, 17, 23, 0, 16, 4, "16,24,24", "halves", True, "f32", "heads", "i64"),
        # a text encoder's 77 tokens of width 768: the smallest norm
        norm_case("norm, 77 text tokens", "norm", 1, 77, 768, "f16", "f16", "f16", False),
        # four 1024 x 1024 images' fp32 residual stream into the bf16 input of the next Linear
        norm_case("norm, four images", "norm", 4, 4608, 3072, "f32", "bf16", "f32", False),
        # the adaLN norm of one image backwards, joined with the residual stream's own gradient
        norm_case("modulated norm, backward", "mod_back", 1, 4608, 3072, "f32", "bf16", "bf16", True),
        # many short rows backwards, an odd count: the weight's gradient is a sum over all of them
        norm_case("norm, backward, long", "norm_back", 1, 65537, 1280, "bf16", "bf16", "f32", False),
        # the timestep embedder's first Linear for one image
        linear_case("linear, one row", 1, 256, 3072, "bf16", "silu", True, "none", "bf16"),
        # the modulation Linear of a double block for 28 steps: as many bytes as the weight has
        linear_case("linear, 28 rows", 28, 3072, 18432, "bf16", "none", True, "none", "bf16"),
        # odd sizes everywhere
        linear_case("linear, odd", 333, 1000, 1111, "f16", "gelu", True, "same", "f16"),
        # the MLP's second Linear of a 1024 x 1024 image onto the fp32 residual stream: the most arithmetic
        linear_case("linear, mlp out", 4608, 12288, 3072, "bf16", "none", True, "f32", "f32"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "norm", "norm_back", "mod_back", "linear", "linear"))
    if op == "rope":
        axes = rng.choice(("16,56,56", "44,42,42", "16,24,24", "64,64", "20,22,22", "128", "10,30,40", "64,96,96"))
        dim = sum(int(a) for a in axes.split(","))
        kv = rng.choice((1, 2, 3, 4, 8, 12, 24))
        heads = kv * rng.choice((1, 1, 2, 4))
        tokens = _log(rng, 1, 60000)
        batch = rng.choice((1, 1, 1, 2, 3))
        text = rng.randrange(0, min(513, tokens))
        height = max(1, int(math.sqrt((tokens - text) / rng.choice((1, 1, 4, 9)))))
        width = max(1, rng.randint(max(1, height - 3), height + 20))
        frames = max(1, (tokens - text) // (height * width))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        while batch * (text + frames * height * width) * (heads + kv) * dim * SIZE[dtype] > 740_000_000:
            frames, height, text = (frames + 1) // 2, (height + 1) // 2, text // 2
        return {k: v for k, v in rope_case("", batch, text, frames, height, width, rng.choice((0, 0, 0, 1000, 1_000_000)), heads, kv, axes,
                                           rng.choice(("interleaved", "halves")), rng.random() < 0.4, dtype,
                                           rng.choice(("heads", "qkv", "tokens")), rng.choice(("f32", "i64", "i32", "f64"))).items() if k != "name"}
    if op != "linear":
        dim = _log(rng, 24, 12288)
        dim = dim if rng.random() < 0.3 else max(8, dim // 8 * 8)
        rows = _log(rng, 1, min(200_000, 56_000_000 // dim))
        batch = rng.choice((1, 1, 2, 3, 5))
        types = ("f32", "bf16", "f16")
        x = rng.choice(("f32", "f32", "bf16", "f16"))
        if op == "mod_back":
            x = "f32"
            dim = max(8, dim // 4 * 4)
        c = norm_case("", op, batch, max(1, rows // batch), dim, x, "bf16" if op == "mod_back" else rng.choice(types), "bf16" if op == "mod_back" else rng.choice(types),
                      op != "norm" and rng.random() < 0.5)
        return {k: v for k, v in c.items() if k != "name"}
    m = rng.choice((1, _log(rng, 1, 64), _log(rng, 1, 8192), _log(rng, 1, 8192)))
    n = _log(rng, 16, 20000)
    k = _log(rng, 16, 14000)
    k = k if rng.random() < 0.15 else max(8, k // 8 * 8)
    n = n if rng.random() < 0.3 else max(8, n // 8 * 8)
    while 2.0 * m * n * k > 3.4e11:
        m = (m + 1) // 2
    dtype = rng.choice(("bf16", "bf16", "f16"))
    residual = rng.choice(("none", "same", "f32"))
    c = linear_case("", m, k, n, dtype, rng.choice(ACTS), rng.random() < 0.7, residual, "f32" if residual == "f32" else rng.choice((dtype, dtype, "f32")))
    return {k: v for k, v in c.items() if k != "name"}


# ---------------------------------------------------------------------------------------------- inputs


def _axes(case):
    return tuple(int(a) for a in case["axes"].split(","))


def _ids(case):
    """Position ids [L, axes]: zeros for text, then (frame, row, column); the first axis starts at `start`. With one axis it counts tokens, with two rows and columns."""
    f, h, w = case["frames"], case["height"], case["width"]
    n, axes = f * h * w, len(_axes(case))
    i = torch.arange(n, device=DEV)
    grid = {1: (i,), 2: (i // w, i % w), 3: (i // (h * w), i // w % h, i % w)}[axes]
    ids = torch.zeros(case["text"] + n, axes, dtype=torch.int64, device=DEV)
    ids[case["text"]:] = torch.stack(grid, 1)
    ids[case["text"]:, 0] += case["start"]
    return ids.to({"i64": torch.int64, "i32": torch.int32, "f32": torch.float32, "f64": torch.float64}[case["ids"]])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, dtype, std=1.0, mean=0.0):
        t = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)
        return t.mul_(std).add_(mean).to(dtype)

    if case["op"] == "rope":
        b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], sum(_axes(case))
        seq, dt = case["text"] + case["frames"] * case["height"] * case["width"], TYPES[case["dtype"]]
        if case["layout"] == "qkv":  # one fused projection's rows: q heads, k heads, v heads
            rows = normal(b, seq, h + 2 * kv, d, dtype=dt)
            q, k = rows[:, :, :h].transpose(1, 2), rows[:, :, h:h + kv].transpose(1, 2)
        elif case["layout"] == "tokens":  # separate projections' rows
            q, k = normal(b, seq, h, d, dtype=dt).transpose(1, 2), normal(b, seq, kv, d, dtype=dt).transpose(1, 2)
        else:
            q, k = normal(b, h, seq, d, dtype=dt), normal(b, kv, seq, d, dtype=dt)
        return {"case": case, "q": q, "k": k, "ids": _ids(case), "axes": _axes(case)}
    if case["op"] == "linear":
        m, k, n, dt = case["m"], case["k"], case["n"], TYPES[case["dtype"]]
        s = {"case": case, "x": normal(m, k, dtype=dt), "w": normal(n, k, dtype=dt, std=1 / math.sqrt(k)), "bias": None, "residual": None}
        if case["bias"]:
            s["bias"] = normal(n, dtype=dt, std=0.5)
        if case["residual"] != "none":
            s["residual"] = normal(m, n, dtype=dt if case["residual"] == "same" else torch.float32)
        return s
    b, seq, d = case["batch"], case["seq"], case["dim"]
    channel = 1 + 0.5 * torch.randn(d, generator=g, device=DEV).abs()  # some channels are larger, as in a residual stream
    x = (normal(b, seq, d, dtype=torch.float32) * channel + 0.2).to(TYPES[case["x"]])
    s = {"case": case, "x": x, "add": None}
    if case["op"] == "mod_back":
        s["scale"] = normal(b, d, dtype=TYPES[case["w"]], std=0.3)
    else:
        s["weight"] = normal(d, dtype=TYPES[case["w"]], std=0.3, mean=1.0)
        s["bias"] = normal(d, dtype=TYPES[case["w"]], std=0.3)
    if case["op"] != "norm":
        s["dy"] = normal(b, seq, d, dtype=TYPES[case["y"]])
        if case["add"]:
            s["add"] = normal(b, seq, d, dtype=TYPES[case["x"]])
    return s


def _eps(case):
    return 1e-6 if case["op"] == "mod_back" else 1e-5


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        from selas_b200 import ops

        if case["op"] == "rope":
            return ops.rope_axes_qk(state["q"], state["k"], state["ids"], state["axes"], 10000.0, pairs=case["pairs"], inverse=case["inverse"])
        if case["op"] == "norm":
            return ops.layer_norm(state["x"], state["weight"], state["bias"], 1e-5, out_dtype=TYPES[case["y"]])
        if case["op"] == "norm_back":
            return ops.layer_norm_backward(state["dy"], state["x"], state["weight"], 1e-5, add=state["add"])
        if case["op"] == "mod_back":
            return ops.ln_mod_backward(state["dy"], state["x"], state["scale"], add=state["add"])
        return ops.linear_act(state["x"], state["w"], state["bias"], case["act"], state["residual"], out_dtype=TYPES[case["out"]])
    if case["op"] == "rope":
        return _rope_plain(state)
    if case["op"] == "linear":
        return _linear_plain(state)
    return _norm_plain(state)


def _rope_plain(s):
    case, ids = s["case"], s["ids"]
    omega = [10000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d) for d in s["axes"]]
    angle = torch.cat([ids[:, a, None].double() * w for a, w in enumerate(omega)], 1)
    cos, sin = angle.cos().float(), angle.sin().float()
    if case["inverse"]:
        sin = -sin

    def turn(x):
        f = x.float()
        if case["pairs"] == "interleaved":
            a, b = f[..., 0::2], f[..., 1::2]
            return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2).to(x.dtype)
        a, b = f.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1).to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _norm_plain(s):
    case = s["case"]
    x = s["x"].float()
    c = x - x.mean(-1, keepdim=True)
    r = (c.square().mean(-1, keepdim=True) + _eps(case)).rsqrt()
    h = c * r
    if case["op"] == "norm":
        return (h * s["weight"].float() + s["bias"].float()).to(TYPES[case["y"]])
    dy = s["dy"].float()
    if case["op"] == "mod_back":
        g = dy * (1 + s["scale"].float()[:, None])
    else:
        g = dy * s["weight"].float()
    dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    if s["add"] is not None:
        dx = dx + s["add"].float()
    dx = dx.to(s["x"].dtype)
    if case["op"] == "mod_back":
        return dx, dy.sum(1), (dy * h).sum(1)
    return dx, (dy * h).sum((0, 1)), dy.sum((0, 1))


def _linear_plain(s):
    case = s["case"]
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    act = case["act"]
    if act == "relu":
        z = z.clamp_min(0)
    elif act == "gelu":
        z = 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    elif act == "gelu_tanh":
        z = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    elif act == "quick_gelu":
        z = z / (1 + torch.exp(-1.702 * z))
    elif act == "silu":
        z = z / (1 + torch.exp(-z))
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(TYPES[case["out"]])


# ---------------------------------------------------------------------------------------------- work


def work(case):
    if case["op"] == "rope":
        seq = case["text"] + case["frames"] * case["height"] * case["width"]
        n = case["batch"] * seq * (case["heads"] + case["kv_heads"]) * sum(_axes(case))
        ids = seq * len(_axes(case)) * (4 if case["ids"] in ("f32", "i32") else 8)
        return {"bytes": 2 * n * SIZE[case["dtype"]] + ids, "flops": 3 * n}
    if case["op"] == "linear":
        m, k, n, e = case["m"], case["k"], case["n"], SIZE[case["dtype"]]
        r = {"none": 0, "same": e, "f32": 4}[case["residual"]]
        return {"bytes": (m * k + n * k + (n if case["bias"] else 0)) * e + m * n * (r + SIZE[case["out"]]), "flops": 2 * m * n * k}
    b, seq, d = case["batch"], case["seq"], case["dim"]
    n = b * seq * d
    ex, ey, ew = SIZE[case["x"]], SIZE[case["y"]], SIZE[case["w"]]
    if case["op"] == "norm":
        return {"bytes": n * (ex + ey) + 2 * d * ew, "flops": 8 * n}
    groups = b if case["op"] == "mod_back" else 1
    return {"bytes": n * (ex + ey + ex + (ex if case["add"] else 0)) + groups * d * (ew + 8), "flops": 16 * n}


# ---------------------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        at, parts = s["ids"].to(torch.float64), []
        for a, d in enumerate(s["axes"]):
            j = torch.arange(d // 2, device=DEV, dtype=torch.float64)
            parts.append(torch.outer(at[:, a], torch.exp(j * (-2 * math.log(10000.0) / d))))
        angle = torch.cat(parts, 1)
        turn = torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle)

        def by(x):
            if case["pairs"] == "interleaved":
                z = torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous()) * turn
                return torch.view_as_real(z).flatten(-2)
            half = x.shape[-1] // 2
            z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn
            return torch.cat((z.real, z.imag), -1)

        return by(s["q"]), by(s["k"])
    if case["op"] == "linear":
        z = torch.matmul(s["x"].double(), s["w"].double().T)
        if s["bias"] is not None:
            z += s["bias"].double()
        act = case["act"]
        if act == "relu":
            z = torch.where(z > 0, z, torch.zeros_like(z))
        elif act == "gelu":
            z = z * torch.erfc(-z / math.sqrt(2.0)) / 2
        elif act == "gelu_tanh":
            u = math.sqrt(2 / math.pi) * (z + 0.044715 * z.pow(3))
            z = z * torch.sigmoid(2 * u)
        elif act == "quick_gelu":
            z = z * torch.sigmoid(1.702 * z)
        elif act == "silu":
            z = z * torch.sigmoid(z)
        return z if s["residual"] is None else z + s["residual"].double()
    x = s["x"].double().requires_grad_(case["op"] != "norm")
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    h = (x - mean) / torch.sqrt(var + _eps(case))
    if case["op"] == "norm":
        return torch.addcmul(s["bias"].double(), h, s["weight"].double())
    if case["op"] == "mod_back":
        shift = torch.zeros_like(s["scale"], dtype=torch.float64).requires_grad_(True)
        scale = s["scale"].double().requires_grad_(True)
        y = h * (1 + scale.unsqueeze(1)) + shift.unsqueeze(1)
        dx, *rest = torch.autograd.grad(y, (x, shift, scale), s["dy"].double())
    else:
        weight, bias = s["weight"].double().requires_grad_(True), s["bias"].double().requires_grad_(True)
        dx, *rest = torch.autograd.grad(h * weight + bias, (x, weight, bias), s["dy"].double())
    return (dx if s["add"] is None else dx + s["add"].double(), *rest)
