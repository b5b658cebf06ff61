"""The operators around the attention call of a transformer block, as cases that can be timed and compared.

Three operators, each with its plain form (elementary torch operations in fp32, rounded once at the end) and the call a
user makes of the library:

  norm     normalisation of a row together with the residual's addition, forward or forward + backward, or with the
           result also held in 8 bits with one scale per row
  linear   act(x W^T + b) + residual, forward or forward + backward
  linear8  the same product over 8-bit rows (e4m3) with one scale per row of x and one per row of W

`own` selects which of the two `run` computes.
"""
import math

import torch

own = False

DEVICE = "cuda"
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _norm(name, rows, dim, dtype, stream, kind, place, gate, mode):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "stream": stream, "kind": kind,
            "place": place, "gate": gate, "mode": mode}


def _linear(name, m, k, n, dtype, act, residual, mode):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "residual": residual,
            "mode": mode}


def _linear8(name, m, k, n, dtype, act, residual, quantize):
    return {"name": name, "op": "linear8", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "residual": residual,
            "quantize": quantize}


def listed():
    return [
        # one token of a pre-norm stream on its way to an 8-bit product: nothing but latency
        _norm("norm_one_token_8bit", 1, 768, "f16", "f16", "rms", "pre", 0, "8bit"),
        # residual post-norm of the first stage of a hierarchical vision model in training (64 images of 64 x 64
        # tokens, stochastic depth on): the largest stream with the shortest rows
        _norm("norm_post_train", 262144, 96, "bf16", "bf16", "layer", "post", 64, "train"),
        # a long prompt over an fp32 residual stream, the normalised rows leaving in 8 bits
        _norm("norm_prompt_8bit", 16384, 1536, "bf16", "f32", "rms", "pre", 0, "8bit"),
        # a ragged number of rows of an odd width, rows off 16-byte boundaries
        _norm("norm_odd_train", 4099, 385, "f16", "f16", "rms", "pre", 0, "train"),
        # the classifier head on one pooled image
        _linear("linear_one_row", 1, 768, 1000, "f16", "none", False, "forward"),
        # first product of the MLP, first stage, inference: bound by writing the hidden rows
        _linear("linear_gelu_wide", 262144, 96, 384, "bf16", "gelu", False, "forward"),
        # the same product two stages on, in training: as much arithmetic, an eighth of the rows
        _linear("linear_gelu_train", 16384, 384, 1536, "bf16", "gelu", False, "train"),
        # second product of the MLP with the residual's addition in its epilogue, second stage, in training
        _linear("linear_residual_train", 65536, 768, 192, "f16", "none", True, "train"),
        # a patch embedding of 14 x 14 x 3 pixels (rows of 588 elements: off 16-byte boundaries) to an odd width
        _linear("linear_odd_train", 1225, 588, 333, "bf16", "gelu", False, "train"),
        # a large square layer over a long prompt: bound by the matrix units
        _linear("linear_square", 8192, 4096, 4096, "bf16", "silu", True, "forward"),
        # a few tokens at a time through an 8-bit layer: bound by reading its weights
        _linear8("linear8_few_rows", 4, 1536, 768, "bf16", "none", True, False),
        # a long prompt through an 8-bit layer, its rows quantised on the way
        _linear8("linear8_prompt", 8192, 4096, 4096, "bf16", "gelu", False, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Mostly multiples of 8, as layers are; one in four as it falls."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.25 else max(8, (n + 4) // 8 * 8)


def draw(rng):
    op = rng.choice(("norm", "norm", "linear", "linear", "linear", "linear8"))
    if op == "norm":
        dim = _width(rng, 8, 8192)
        rows = _log_int(rng, 1, max(1, min(262144, 262144 * 96 // dim)))
        mode = rng.choice(("forward", "train", "8bit"))
        dtype = rng.choice(("bf16", "f16"))
        gate = rng.choice([g for g in (0, 1, 2, 7, 16, 64) if g == 0 or rows % g == 0])
        return {k: v for k, v in _norm("", rows, dim, dtype, rng.choice((dtype, "f32")), rng.choice(("layer", "rms")),
                                       rng.choice(("post", "pre")), gate, mode).items() if k != "name"}
    k, n = _width(rng, 8, 4096), _width(rng, 8, 4096)
    most = 8192 * 4096 * 4096 // (3 if op == "linear" else 1)
    m = _log_int(rng, 1, max(1, min(262144, most // (k * n), 262144 * 384 // max(k, n))))
    act, dtype = rng.choice(("none", "gelu", "gelu_tanh", "silu", "relu")), rng.choice(("bf16", "f16"))
    if op == "linear":
        case = _linear("", m, k, n, dtype, act, rng.random() < 0.4, rng.choice(("forward", "train")))
    else:
        case = _linear8("", m, k, n, dtype, act, rng.random() < 0.4, rng.random() < 0.5)
    return {key: v for key, v in case.items() if key != "name"}


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def rand(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale + shift).to(dtype)

    def activations(rows, dim, dtype):
        """Rows of different magnitude with a few channels that stand out, as the streams of trained models have."""
        channel = torch.exp(0.5 * torch.randn(dim, generator=g, device=DEVICE))
        row = torch.exp(0.3 * torch.randn(rows, 1, generator=g, device=DEVICE))
        return (torch.randn(rows, dim, generator=g, device=DEVICE) * channel * row).to(dtype)

    dt = DTYPES[case["dtype"]]
    s = {}
    if case["op"] == "norm":
        rows, dim, st = case["rows"], case["dim"], DTYPES[case["stream"]]
        s["x"] = activations(rows, dim, dt)
        s["shortcut"] = activations(rows, dim, st)
        s["weight"] = rand(dim, scale=0.2, shift=1.0, dtype=st)
        s["bias"] = rand(dim, scale=0.1, dtype=st) if case["kind"] == "layer" else None
        s["gate"] = None
        if case["gate"]:      # stochastic depth: one factor per sample, 0 or 1 / keep
            keep = torch.rand(case["gate"], generator=g, device=DEVICE) < 0.9
            s["gate"] = (keep.float() / 0.9).to(dt)
        s["dy"] = rand(rows, dim, dtype=st if case["place"] == "post" else dt) if case["mode"] == "train" else None
        s["dh"] = rand(rows, dim, dtype=st) if case["mode"] == "train" and case["place"] == "pre" else None
        return s
    m, k, n = case["m"], case["k"], case["n"]
    s["x"] = activations(m, k, dt)
    s["weight"] = rand(n, k, scale=k ** -0.5, dtype=dt)
    s["bias"] = rand(n, scale=0.1, dtype=dt)
    s["residual"] = activations(m, n, dt) if case["residual"] else None
    if case["op"] == "linear":
        s["dy"] = rand(m, n, dtype=dt) if case["mode"] == "train" else None
        return s
    s["weight8"], s["weight_scale"] = _plain_quantize(s.pop("weight"))
    if not case["quantize"]:
        s["x8"], s["x_scale"] = _plain_quantize(s.pop("x"))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case.get("mode") == "train":
        for name in ("x", "shortcut", "weight", "bias", "residual"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms: elementary operations in fp32, rounded once
# ---------------------------------------------------------------------------------------------------------------------
def _plain_quantize(y):
    y = y.float()
    scale = y.abs().amax(-1).clamp_min(2.0 ** -100) / F8_MAX
    return (y / scale[:, None]).to(F8), scale


def _plain_norm(s):
    case = s["case"]
    layer, post = case["kind"] == "layer", case["place"] == "post"
    x, r, w = s["x"].detach().float(), s["shortcut"].detach().float(), s["weight"].detach().float()
    b = s["bias"].detach().float() if layer else None
    g = 1.0
    if s["gate"] is not None:
        g = s["gate"].float().repeat_interleave(case["rows"] // case["gate"])[:, None]
    h = x if post else r + g * x
    centred = h - h.mean(-1, keepdim=True) if layer else h
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xhat = centred * rstd
    y = xhat * w + b if layer else xhat * w
    if post:
        y = r + g * y
    st, dt = s["shortcut"].dtype, s["x"].dtype
    if case["mode"] == "8bit":
        q, scale = _plain_quantize(y)
        return {"stream": (y if post else h).to(st), "q": q, "scale": scale}
    out = {"y": y.to(st)} if post else {"h": h.to(st), "y": y.to(dt)}
    if case["mode"] == "forward":
        return out
    dy = s["dy"].float()
    dn = g * dy if post else dy
    t = dn * w
    dh = t - xhat * (t * xhat).mean(-1, keepdim=True)
    if layer:
        dh = dh - t.mean(-1, keepdim=True)
    dh = dh * rstd
    if post:
        out["dx"], out["dshortcut"] = dh.to(dt), s["dy"]
    else:
        dh = dh + s["dh"].float()
        out["dx"], out["dshortcut"] = (g * dh).to(dt), dh.to(st)
    out["dweight"] = (dn * xhat).sum(0).to(st)
    if layer:
        out["dbias"] = dn.sum(0).to(st)
    return out


def _plain_act(z, act):
    if act == "gelu":
        return z * (0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    return z


def _plain_act_slope(z, act):
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return sig * (1.0 + z * (1.0 - sig))
    return (z > 0).float()


def _plain_linear(s):
    case = s["case"]
    dt = s["x"].dtype
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    z = x @ w.t() + b
    y = _plain_act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    out = {"y": y.to(dt)}
    if case["mode"] == "forward":
        return out
    dz = s["dy"].float()
    if case["act"] != "none":
        dz = dz * _plain_act_slope(z, case["act"])
    out["dx"] = (dz @ w).to(dt)
    out["dweight"] = (dz.t() @ x).to(dt)
    out["dbias"] = dz.sum(0).to(dt)
    if s["residual"] is not None:
        out["dresidual"] = s["dy"]
    return out


def _plain_linear8(s):
    case = s["case"]
    x8, x_scale = _plain_quantize(s["x"]) if case["quantize"] else (s["x8"], s["x_scale"])
    z = (x8.float() @ s["weight8"].float().t()) * x_scale[:, None] * s["weight_scale"][None, :] + s["bias"].float()
    y = _plain_act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(DTYPES[case["dtype"]])}


# ---------------------------------------------------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------------------------------------------------
def _own_norm(s):
    import flash_window_attention_v2_amd as fwa2
    case = s["case"]
    args = (s["x"], s["shortcut"], s["weight"], s["bias"])
    how = {"eps": EPS, "kind": case["kind"], "placement": case["place"], "gate": s["gate"]}
    if case["mode"] == "8bit":
        stream, q, scale = fwa2.residual_norm_fp8_func(*args, **how)
        return {"stream": stream, "q": q, "scale": scale}
    got = fwa2.residual_norm_func(*args, **how)
    out = {"y": got} if case["place"] == "post" else {"h": got[0], "y": got[1]}
    if case["mode"] == "forward":
        return out
    names = ["x", "shortcut", "weight"] + (["bias"] if s["bias"] is not None else [])
    if case["place"] == "post":
        grads = torch.autograd.grad(out["y"], [s[a] for a in names], s["dy"])
    else:
        grads = torch.autograd.grad((out["h"], out["y"]), [s[a] for a in names], (s["dh"], s["dy"]))
    out = {a: v.detach() for a, v in out.items()}
    out.update({"d" + a: v for a, v in zip(names, grads)})
    return out


def _own_linear(s):
    import flash_window_attention_v2_amd as fwa2
    case = s["case"]
    act = None if case["act"] == "none" else case["act"]
    y = fwa2.fused_linear_func(s["x"], s["weight"], s["bias"], act, s["residual"])
    if case["mode"] == "forward":
        return {"y": y}
    names = ["x", "weight", "bias"] + (["residual"] if s["residual"] is not None else [])
    grads = torch.autograd.grad(y, [s[a] for a in names], s["dy"])
    out = {"y": y.detach()}
    out.update({"d" + a: v for a, v in zip(names, grads)})
    return out


def _own_linear8(s):
    import flash_window_attention_v2_amd as fwa2
    case = s["case"]
    act = None if case["act"] == "none" else case["act"]
    x8, x_scale = fwa2.quantize_rows_func(s["x"]) if case["quantize"] else (s["x8"], s["x_scale"])
    return {"y": fwa2.fused_linear_fp8_func(x8, x_scale, s["weight8"], s["weight_scale"], s["bias"], act, s["residual"],
                                            out_dtype=DTYPES[case["dtype"]])}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "linear": _own_linear, "linear8": _own_linear8}[op](state)
    return {"norm": _plain_norm, "linear": _plain_linear, "linear8": _plain_linear8}[op](state)


# ---------------------------------------------------------------------------------------------------------------------
# the work of one pass, and its values in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if case["op"] == "norm":
        e, st, cells = size[case["dtype"]], size[case["stream"]], case["rows"] * case["dim"]
        post = case["place"] == "post"
        vectors = case["dim"] * st * (2 if case["kind"] == "layer" else 1)
        moved = cells * (e + st) + vectors                                         # x, shortcut
        if case["mode"] == "8bit":
            return {"bytes": moved + cells * (st + 1) + 4 * case["rows"], "flops": 12.0 * cells}
        moved += cells * st if post else cells * (st + e)                          # y, or h and y
        flops = 8.0 * cells
        if case["mode"] == "train":
            # dy, the normalised rows' source and dx; in the pre-norm form also dh and dshortcut
            moved += cells * (st + e + e) if post else cells * (e + st + st + e + (st if st != e or case["gate"] else 0))
            moved += 2 * vectors
            flops += 20.0 * cells
        return {"bytes": moved, "flops": flops}
    m, k, n = case["m"], case["k"], case["n"]
    if case["op"] == "linear8":
        moved = m * k * (2 if case["quantize"] else 1) + n * k + 4 * (m + n) + 2 * n + 2 * m * n
        return {"bytes": moved + (2 * m * n if case["residual"] else 0), "flops": 2.0 * m * n * k}
    moved = 2 * (m * k + n * k + n + m * n) + (2 * m * n if case["residual"] else 0)
    flops = 2.0 * m * n * k
    if case["mode"] == "train":
        # dy and, behind an activation, what its slope is taken at; x, W read again; dx, dW, db written
        moved += 2 * m * n * (1 if case["act"] == "none" else 3) + 4 * (m * k + n * k) + 2 * n
        flops *= 3.0
    return {"bytes": moved, "flops": flops}


def exact(case, seed):
    s = _inputs(case, seed)
    d = {k: (v.double().requires_grad_(True) if isinstance(v, torch.Tensor) and v.dtype != F8 else v) for k, v in s.items()}
    if case["op"] == "norm":
        return _exact_norm(case, d)
    act = {"none": lambda z: z, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu, "relu": torch.relu,
           "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[case["act"]]
    if case["op"] == "linear8":
        with torch.no_grad():
            if case["quantize"]:
                # the 8-bit rows are whole steps of an fp32 scale: rounded as the definition says, then taken as exact
                x8, sx = _plain_quantize(s["x"])
                x = x8.double() * sx.double()[:, None]
            else:
                x = s["x8"].double() * d["x_scale"][:, None]
            w = s["weight8"].double() * d["weight_scale"][:, None]
            y = act(torch.nn.functional.linear(x, w, d["bias"]))
            return {"y": y if d["residual"] is None else y + d["residual"]}
    y = act(torch.nn.functional.linear(d["x"], d["weight"], d["bias"]))
    if d["residual"] is not None:
        y = y + d["residual"]
    out = {"y": y.detach()}
    if case["mode"] == "train":
        names = ["x", "weight", "bias"] + (["residual"] if d["residual"] is not None else [])
        out.update({"d" + a: v for a, v in zip(names, torch.autograd.grad(y, [d[a] for a in names], d["dy"]))})
    return out


def _exact_norm(case, d):
    x, r, dim = d["x"], d["shortcut"], (case["dim"],)
    g = 1.0
    if d["gate"] is not None:
        g = d["gate"].detach().view(-1, 1, 1).expand(-1, case["rows"] // case["gate"], 1).reshape(-1, 1)

    def norm(v):
        if case["kind"] == "layer":
            return torch.nn.functional.layer_norm(v, dim, d["weight"], d["bias"], EPS)
        return torch.nn.functional.rms_norm(v, dim, d["weight"], EPS)

    if case["place"] == "post":
        h, y = None, r + g * norm(x)
    else:
        h = r + g * x
        y = norm(h)
    if case["mode"] == "8bit":
        with torch.no_grad():
            scale = y.abs().amax(-1) / F8_MAX
            return {"stream": (y if h is None else h).detach(), "q": (y / scale[:, None]).detach(), "scale": scale}
    out = {"y": y.detach()}
    if h is not None:
        out["h"] = h.detach()
    if case["mode"] == "train":
        names = ["x", "shortcut", "weight"] + (["bias"] if d["bias"] is not None else [])
        ends, seeds = ((y,), (d["dy"],)) if h is None else ((h, y), (d["dh"], d["dy"]))
        out.update({"d" + a: v for a, v in zip(names, torch.autograd.grad(ends, [d[a] for a in names], seeds))})
    return out
