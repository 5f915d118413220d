"""Timing cases of the operators of a transformer block around its attention,
each in two forms.

* ``linear``: act(x W^T + bias) * gate + residual with both operands in 8-bit
  floating point (e4m3), a power of two as scale for every 128 consecutive
  channels of a row. x comes in 16 bits, and is quantised within the call, or in
  8 bits as the operator before left it; the result is left in 16 bits or in 8.
* ``quantize``: rows of 16-bit values to such codes and scales.
* ``norm``: r = scale * x + gate * post(y), h = norm(r), modulated: what stands
  between two branches of a block; h in 16 bits or as codes and scales.
* ``rope``: RMS norm of the heads of q and k and their rotation by positions of
  several axes (time, height, width), from a grid or given token by token.

With ``own`` false ``run`` computes a case from elementary torch operations in
32 bits (angles in 64), with ``own`` true through this framework's entry points.
8-bit results are returned as the codes' values and, beside them, their scales.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
MAX_FLOPS = 2.0 * 75600 * 5120 * 13824  # of the largest product below
MAX_BYTES = 4e9
EPS = 1e-6
BLOCK = 128
THETA = 10000.0


def _linear(name, m, n, k, dtype="bf16", x8=False, out8=False, bias=True, act="none", gate=False, residual=False):
    return {"name": name, "kind": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "x8": x8, "out8": out8,
            "bias": bias, "act": act, "gate": gate, "residual": residual}


def _quantize(name, rows, k, dtype="bf16"):
    return {"name": name, "kind": "quantize", "rows": rows, "k": k, "dtype": dtype}


def _norm(name, groups, rows, channels, dtype="bf16", norm="layer", post="none", affine=False, gate=True,
          modulate=False, out8=False, scale=1.0):
    """groups: sequences or frames of `rows` tokens, each with a gate and a modulation of its own."""
    return {"name": name, "kind": "norm", "groups": groups, "rows": rows, "channels": channels, "dtype": dtype,
            "norm": norm, "post": post, "affine": affine, "gate": gate, "modulate": modulate, "out8": out8,
            "scale": scale}


def _rope(name, batch, tokens, heads, kv_heads, dim=128, dtype="bf16", height=0, width=0, halves=False, norm="all",
          far=0):
    """height, width: of a grid's frames (0: positions are given for every token). far: tokens before the first."""
    return {"name": name, "kind": "rope", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "height": height, "width": width, "halves": halves, "norm": norm, "far": far}


def listed():
    return [
        # the feed-forward products of a block at the benchmark video's 75,600 tokens: the first leaves the
        # second's operand
        _linear("linear_ffn_up", 75600, 13824, 5120, out8=True, act="gelu_tanh"),
        _linear("linear_ffn_down", 75600, 5120, 13824, x8=True, gate=True, residual=True),
        # the text embedder: 512 tokens of 4,096 channels
        _linear("linear_text", 512, 5120, 4096, act="gelu_tanh"),
        # the modulation of a block from one time step: one row
        _linear("linear_time", 1, 30720, 5120),
        # odd everywhere, f16, no axis a multiple of anything
        _linear("linear_odd", 333, 1017, 709, dtype="f16", act="silu", residual=True),
        # a benchmark video's hidden states
        _quantize("quantize_video", 75600, 5120),
        # a few odd rows: latency
        _quantize("quantize_odd", 77, 1001, dtype="f16"),
        # between the self-attention and the text attention of a block: the gated residual and an affine norm
        _norm("norm_video", 1, 75600, 5120, affine=True),
        # frames of a 480p stream, each with its own step's modulation, on their way into the 8-bit products
        _norm("norm_frames", 3, 1560, 5120, norm="rms", post="rms", modulate=True, out8=True),
        # a benchmark video's heads: 21 frames of 45 x 80 tokens
        _rope("rope_video", 1, 75600, 40, 40, height=45, width=80),
        # images of any shape in one batch, positions token by token, shared key heads
        _rope("rope_images", 2, 4099, 24, 8, dim=128, dtype="f16", halves=True, norm="head"),
        # single tokens of 32 sequences, far behind their beginnings
        _rope("rope_token", 32, 1, 32, 8, height=30, width=52, norm="head", far=1 << 26),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths of models are multiples of 64, others happen."""
    n = _log_int(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.6 else n


def _draw_linear(rng):
    while True:
        m, n, k = _log_int(rng, 1, 75600), _width(rng, 64, 13824), _width(rng, 64, 13824)
        case = _linear("", m, n, k, dtype=rng.choice(["bf16", "bf16", "f16"]), x8=rng.random() < 0.4,
                       out8=rng.random() < 0.3, bias=rng.random() < 0.7,
                       act=rng.choice(["none", "none", "gelu_tanh", "silu", "gelu"]), gate=rng.random() < 0.3,
                       residual=rng.random() < 0.4)
        if work(case)["flops"] <= MAX_FLOPS:
            return case


def _draw_quantize(rng):
    return _quantize("", _log_int(rng, 1, 75600), _width(rng, 16, 13824), rng.choice(["bf16", "bf16", "f16"]))


def _draw_norm(rng):
    while True:
        groups = rng.choice([1, 1, 2, 3, 21])
        case = _norm("", groups, max(1, _log_int(rng, 1, 75600) // groups), _width(rng, 64, 8192),
                     rng.choice(["bf16", "bf16", "f16"]), rng.choice(["layer", "rms"]),
                     rng.choice(["none", "none", "rms", "layer"]), rng.random() < 0.5, rng.random() < 0.7,
                     rng.random() < 0.6, rng.random() < 0.3, rng.choice([1.0, 1.0, 0.5, 1.4]))
        if work(case)["bytes"] <= MAX_BYTES:
            return case


def _draw_rope(rng):
    while True:
        kv = rng.choice([1, 2, 4, 8, 12, 40])
        heads = kv * (rng.choice([1, 2, 4, 5]) if kv < 40 else 1)
        grid = rng.random() < 0.6
        tokens = 1 if rng.random() < 0.25 else _log_int(rng, 2, 75600)
        batch = rng.choice([1, 2, 7, 32]) if tokens < 5000 else 1
        case = _rope("", batch, tokens, heads, kv, rng.choice([128, 128, 64, 96]), rng.choice(["bf16", "bf16", "f16"]),
                     rng.randint(1, 90) if grid else 0, rng.randint(1, 160) if grid else 0, rng.random() < 0.4,
                     rng.choice(["all", "head", "none"]), rng.choice([0, _log_int(rng, 1, 1 << 28)]))
        if heads * case["dim"] <= 8192 and work(case)["bytes"] <= MAX_BYTES:
            return case


def draw(rng):
    case = rng.choice([_draw_linear, _draw_linear, _draw_quantize, _draw_norm, _draw_rope])(rng)
    del case["name"]
    return case


# --------------------------------------------------------------------------
# sizes
# --------------------------------------------------------------------------

def _blocks(k):
    return -(-k // BLOCK)


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        size = m * (k + _blocks(k)) if case["x8"] else 2.0 * m * k
        size += n * (k + _blocks(k)) + (m * (n + _blocks(n)) if case["out8"] else 2.0 * m * n)
        size += (2.0 * m * n if case["residual"] else 0) + (2.0 * n if case["bias"] else 0)
        return {"bytes": size + (4.0 * n if case["gate"] else 0), "flops": 2.0 * m * n * k}
    if case["kind"] == "quantize":
        n, k = case["rows"], case["k"]
        return {"bytes": n * (3.0 * k + _blocks(k)), "flops": 2.0 * n * k}
    if case["kind"] == "norm":
        n, c = case["groups"] * case["rows"], case["channels"]
        vectors = case["groups"] * (case["gate"] + 2 * case["modulate"]) + case["affine"] * 2 + (case["post"] != "none")
        return {"bytes": n * (6.0 * c + (c + _blocks(c) if case["out8"] else 2.0 * c)) + 4.0 * c * vectors,
                "flops": n * c * 12.0}
    n = case["batch"] * case["tokens"]
    c = n * (case["heads"] + case["kv_heads"]) * case["dim"]
    return {"bytes": 4.0 * c + (12.0 * n if not case["height"] else 0), "flops": c * 8.0}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32) * std).to(dtype)


def _hidden(gen, rows, k, dtype):
    """Hidden states: rows of different sizes, a few channels far larger than the others."""
    x = _normal(gen, rows, k)
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device=DEVICE))
    x[:, ::97] *= 8
    return x.to(dtype)


def _to_codes(x):
    """(codes, scales) of x [rows, k] in fp32 elementary operations. The exponent e of a block is the smallest one
    with max |x| <= 448 * 2^e; powers of two are made from their bits. A block's scales of all rows lie together."""
    rows, k = x.shape
    nb = _blocks(k)
    y = x.float()
    if nb * BLOCK != k:
        y = torch.cat([y, y.new_zeros(rows, nb * BLOCK - k)], 1)
    y = y.reshape(rows, nb, BLOCK)
    top = y.abs().amax(-1)
    part, power = torch.frexp(top)
    e = torch.where(part <= 0.875, power - 9, power - 8)
    e = torch.where(top == 0, 0, e).clamp(-127, 127).to(torch.int32)
    inverse = ((127 - e) << 23).view(torch.float32)
    codes = (y * inverse[..., None]).to(torch.float8_e4m3fn).reshape(rows, nb * BLOCK)[:, :k].contiguous()
    return codes, (e + 127).to(torch.uint8).t().contiguous().view(torch.float8_e8m0fnu).t()


def _from_codes(codes, scales, dtype=torch.float32):
    s = torch.exp2((scales.view(torch.uint8).to(torch.int32) - 127).to(torch.float64)).to(dtype)
    return codes.to(dtype) * s.repeat_interleave(BLOCK, -1)[..., :codes.shape[-1]]


def _sections(dim):
    """Channels of time, height and width, as the video models split a head."""
    side = 2 * (dim // 6)
    return dim - 2 * side, side, side


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _hidden(gen, m, k, dt)
        s["x_scales"] = None
        if case["x8"]:
            s["x"], s["x_scales"] = _to_codes(s["x"])
        s["w"], s["w_scales"] = _to_codes(_normal(gen, n, k, std=1.0 / math.sqrt(k), dtype=dt))
        s["bias"] = _normal(gen, n, std=0.1, dtype=dt) if case["bias"] else None
        s["gate"] = _normal(gen, n, std=0.5) if case["gate"] else None
        s["residual"] = _normal(gen, m, n, dtype=dt) if case["residual"] else None
        return s
    if case["kind"] == "quantize":
        s["x"] = _hidden(gen, case["rows"], case["k"], dt)
        return s
    if case["kind"] == "norm":
        g, n, c = case["groups"], case["rows"], case["channels"]
        s["x"] = _hidden(gen, g * n, c, dt).view(g, n, c)
        s["y"] = _normal(gen, g, n, c, dtype=dt)
        s["gate"] = _normal(gen, g, 1, c, std=0.5) if case["gate"] else None
        s["post_weight"] = 1 + _normal(gen, c, std=0.1) if case["post"] != "none" else None
        s["weight"] = 1 + _normal(gen, c, std=0.1) if case["affine"] else None
        s["bias"] = _normal(gen, c, std=0.1) if case["affine"] and case["norm"] == "layer" else None
        # one tensor of a step's modulations, cut into pieces
        both = _normal(gen, g, 2, c, std=0.3)
        s["scale"], s["shift"] = both.chunk(2, 1) if case["modulate"] else (None, None)
        return s
    b, t, h, g, d = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    s["q"], s["k"] = _normal(gen, b, t, h, d, std=1.5, dtype=dt), _normal(gen, b, t, g, d, std=1.5, dtype=dt)
    wide = {"all": (h * d, g * d), "head": (d, d), "none": (0, 0)}[case["norm"]]
    s["q_weight"], s["k_weight"] = ((1 + _normal(gen, n, std=0.1)).to(dt) if n else None for n in wide)
    s["start"] = s["positions"] = None
    if case["height"]:
        if case["far"]:
            s["start"] = (torch.arange(b) * 1009 + case["far"]).to(torch.int32).to(DEVICE)
    else:  # images of some shape, one after another, each later in time than the last
        at = torch.arange(t, device=DEVICE)[None] + 17 * torch.arange(b, device=DEVICE)[:, None]
        side = 1 + int(math.sqrt(t))
        s["positions"] = torch.stack([at // (side * side) + case["far"], at // side % side, at % side], -1).to(torch.int32)
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _OWN[kind](s)
    return _PLAIN[kind](s)


# --------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------

def _own_linear(s):
    from dfsattn_amd import ops

    c = s["case"]
    return ops.linear_fp8(s["x"], s["w"], s["w_scales"], s["x_scales"], bias=s["bias"],
                          activation=None if c["act"] == "none" else c["act"], gate=s["gate"], residual=s["residual"],
                          out_dtype=DTYPES[c["dtype"]], quantize=c["out8"])


def _own_quantize(s):
    from dfsattn_amd import ops

    return ops.quantize_fp8(s["x"])


def _own_norm(s):
    from dfsattn_amd import ops

    c = s["case"]
    return ops.residual_norm(s["x"], s["y"], s["gate"], residual_scale=c["scale"],
                             post_norm=None if c["post"] == "none" else c["post"], post_weight=s["post_weight"],
                             norm=c["norm"], weight=s["weight"], bias=s["bias"], scale=s["scale"], shift=s["shift"],
                             eps=EPS, quantize=c["out8"])


def _own_rope(s):
    from dfsattn_amd import ops

    c = s["case"]
    axes = ops.RotaryAxes(c["dim"], _sections(c["dim"]), theta=THETA, layout="halves" if c["halves"] else "pairs")
    return ops.axial_rope(s["q"], s["k"], axes, grid=(c["height"], c["width"]) if c["height"] else None,
                          start=s["start"], positions=s["positions"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                          eps=EPS)


_OWN = {"linear": _own_linear, "quantize": _own_quantize, "norm": _own_norm, "rope": _own_rope}


# --------------------------------------------------------------------------
# plain forms, in 32 bits
# --------------------------------------------------------------------------

def _activate(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _plain_linear(s):
    c = s["case"]
    x = s["x"], s["x_scales"]
    if not c["x8"]:
        x = _to_codes(s["x"])
    y = _from_codes(*x) @ _from_codes(s["w"], s["w_scales"]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _activate(y, c["act"])
    if s["gate"] is not None:
        y = y * s["gate"]
    if s["residual"] is not None:
        y = s["residual"].float() + y
    y = y.to(DTYPES[c["dtype"]])
    return _to_codes(y) if c["out8"] else y


def _plain_quantize(s):
    return _to_codes(s["x"])


def _normalise(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    if weight is not None:
        x = x * weight
    return x if bias is None else x + bias


def _plain_norm(s):
    c = s["case"]
    y = s["y"].float()
    if c["post"] != "none":
        y = _normalise(y, c["post"], s["post_weight"], None)
    if s["gate"] is not None:
        y = y * s["gate"]
    r = (s["x"].float() * c["scale"] + y).to(s["x"].dtype)
    h = _normalise(r.float(), c["norm"], s["weight"], s["bias"])
    if s["scale"] is not None:
        h = h * (1 + s["scale"]) + s["shift"]
    h = h.to(r.dtype)
    if c["out8"]:
        codes, scales = _to_codes(h.flatten(0, 1))
        return r, codes.view(h.shape), scales.view(*h.shape[:2], -1)
    return r, h


def _positions(s):
    """[B or 1, T, 3] places of the tokens on the axes."""
    c = s["case"]
    if s["positions"] is not None:
        return s["positions"].long()
    at = torch.arange(c["tokens"], device=DEVICE)[None]
    if s["start"] is not None:
        at = at + s["start"][:, None].long()
    return torch.stack([at // (c["height"] * c["width"]), at // c["width"] % c["height"], at % c["width"]], -1)


def _plain_rope(s):
    c = s["case"]
    d = c["dim"]
    at = _positions(s).double()
    angle = torch.cat([at[..., i:i + 1] * THETA ** (-torch.arange(0, n, 2, dtype=torch.float64, device=DEVICE) / n)
                       for i, n in enumerate(_sections(d))], -1)
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    out = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.float()
        if w is not None:
            flat = y if c["norm"] == "head" else y.flatten(2)
            y = (flat / torch.sqrt((flat * flat).mean(-1, keepdim=True) + EPS) * w.float()).reshape(x.shape)
        if c["halves"]:
            a, b = y[..., :d // 2], y[..., d // 2:]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = y[..., 0::2], y[..., 1::2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        out.append(y.to(x.dtype).transpose(1, 2))
    return out


_PLAIN = {"linear": _plain_linear, "quantize": _plain_quantize, "norm": _plain_norm, "rope": _plain_rope}


# --------------------------------------------------------------------------
# definitions, in 64 bits
# --------------------------------------------------------------------------

def _unrounded(y, dtype):
    """What codes and scales stand for: y over its blocks' scales, not rounded, and the scales, which go by the largest
    values as they are stored."""
    top = torch.stack([b.abs().amax(-1) for b in y.split(BLOCK, -1)], -1).to(dtype).double()
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0)).clamp(-127, 127)
    return torch.cat([b * torch.exp2(-e[:, i:i + 1]) for i, b in enumerate(y.split(BLOCK, -1))], -1), torch.exp2(e)


def _exact_linear(s):
    c = s["case"]
    codes, scales = (s["x"], s["x_scales"]) if c["x8"] else _to_codes(s["x"])
    w = _from_codes(s["w"], s["w_scales"], torch.float64).t().contiguous()
    parts = []
    for i in range(0, c["m"], 8192):
        rows = slice(i, i + 8192)
        z = torch.mm(_from_codes(codes[rows], scales[rows], torch.float64), w)
        if s["bias"] is not None:
            z += s["bias"].double()
        if c["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif c["act"] == "gelu":
            z = z * 0.5 * torch.erfc(z * -(2 ** -0.5))
        elif c["act"] == "gelu_tanh":  # (1 + tanh(u)) / 2 = sigmoid(2 u)
            z = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
        if s["gate"] is not None:
            z = z * s["gate"].double()
        if s["residual"] is not None:
            z = z + s["residual"][rows].double()
        parts.append(_unrounded(z, DTYPES[c["dtype"]]) if c["out8"] else z)
    return tuple(torch.cat(p) for p in zip(*parts)) if c["out8"] else torch.cat(parts)


def _exact_quantize(s):
    return _unrounded(s["x"].double(), s["x"].dtype)


def _exact_norm(s):
    c = s["case"]
    x, y = s["x"].double(), s["y"].double()

    def norm(t, kind, w, b):
        var, mean = torch.var_mean(t, -1, correction=0, keepdim=True)
        if kind == "rms":
            var, mean = var + mean * mean, 0.0
        t = (t - mean) * torch.rsqrt(var + EPS)
        t = t if w is None else t * w.double()
        return t if b is None else t + b.double()

    if c["post"] != "none":
        y = norm(y, c["post"], s["post_weight"], None)
    if s["gate"] is not None:
        y = y * s["gate"].double()
    r = torch.add(y, x, alpha=c["scale"])
    h = norm(r.to(s["x"].dtype).double(), c["norm"], s["weight"], s["bias"])  # of r as it is stored
    if s["scale"] is not None:
        h = torch.addcmul(h + s["shift"].double(), h, s["scale"].double())
    if c["out8"]:
        codes, scales = _unrounded(h.flatten(0, 1), s["x"].dtype)
        return r, codes.view(h.shape), scales.view(*h.shape[:2], -1)
    return r, h


def _exact_rope(s):
    c = s["case"]
    d = c["dim"]
    at = _positions(s).double()
    speeds = [torch.exp(torch.arange(n // 2, dtype=torch.float64, device=DEVICE) * (-2 * math.log(THETA) / n))
              for n in _sections(d)]
    turn = torch.cat([torch.exp(1j * at[..., i, None] * f) for i, f in enumerate(speeds)], -1)
    out = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        if w is not None:
            axes = -1 if c["norm"] == "head" else (-2, -1)
            y = y * torch.rsqrt(y.square().mean(axes, keepdim=True) + EPS) * (
                w.double() if c["norm"] == "head" else w.double().view(-1, d))
        y = y.unflatten(-1, (2, -1)).transpose(-1, -2) if c["halves"] else y.unflatten(-1, (-1, 2))
        z = torch.view_as_real(torch.view_as_complex(y.contiguous()) * turn[:, :, None])
        z = z.transpose(-1, -2) if c["halves"] else z
        out.append(z.flatten(-2).transpose(1, 2).contiguous())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "quantize": _exact_quantize, "norm": _exact_norm, "rope": _exact_rope}[case["kind"]](s)
