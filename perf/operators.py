"""Timing cases of the operators around windowed attention, each in two forms.

* ``linear``: act(x W^T + bias) * gate + residual, the projections and the
  feed-forward products of a transformer block, from one row to a whole video.
* ``attention``: softmax attention in which a query sees the keys from ``left``
  tokens before its position to ``right`` tokens behind it and the first
  ``sinks`` tokens: whole videos, prompts, text keys, chunks and single tokens
  over a cache, which may be rolling (the tokens behind the sinks take the
  slots of the oldest).
* ``cache``: RMS norm and rotation of the heads of q and k, with k and v
  appended to such a cache.

With ``own`` false ``run`` computes a case from elementary torch operations in
32 bits, with ``own`` true through this framework's entry points.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
MAX_FLOPS = 2.0 * 75600 * 5120 * 13824  # of the largest product below
EPS = 1e-6


def _linear(name, m, n, k, dtype="bf16", bias=True, act="none", gate=False, residual=False):
    return {"name": name, "kind": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias, "act": act,
            "gate": gate, "residual": residual}


def _attention(name, batch, heads, kv_heads, lq, lk, dim=128, dtype="bf16", left=-1, right=-1, sinks=0, ragged=False,
               rolling=False):
    """left, right: -1 for no limit. ragged: every sequence has its own length. rolling: lk slots, more tokens."""
    return {"name": name, "kind": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "lq": lq,
            "lk": lk, "dim": dim, "dtype": dtype, "left": left, "right": right, "sinks": sinks, "ragged": ragged,
            "rolling": rolling}


def _cache(name, batch, tokens, heads, kv_heads, slots, dim=128, dtype="bf16", per_head=True, sinks=0, ragged=False,
           rolling=False):
    return {"name": name, "kind": "cache", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "slots": slots, "dim": dim, "dtype": dtype, "per_head": per_head, "sinks": sinks, "ragged": ragged,
            "rolling": rolling}


def listed():
    return [
        # the feed-forward products of a block at the benchmark video's 75,600 tokens
        _linear("linear_ffn_up", 75600, 13824, 5120, act="gelu_tanh"),
        _linear("linear_ffn_down", 75600, 5120, 13824, gate=True, residual=True),
        # the text embedder: 512 tokens of 4,096 channels
        _linear("linear_text", 512, 5120, 4096, act="gelu_tanh"),
        # the modulation of a block from one time step: one row
        _linear("linear_time", 1, 30720, 5120),
        # odd everywhere, f16, no axis a multiple of anything
        _linear("linear_odd", 333, 1017, 709, dtype="f16", act="silu", residual=True),
        # a whole benchmark video: one latent frame (3,600 tokens) to either side and the first frame
        _attention("attention_video", 1, 40, 40, 75600, 75600, left=3600, right=3600, sinks=3600),
        # padded prompts, causal, shared key heads, four sinks
        _attention("attention_prompt", 2, 32, 8, 8191, 8191, left=2047, right=0, sinks=4, ragged=True),
        # the next frame of a 480p stream over a rolling cache of its last five frames and the first
        _attention("attention_chunk", 1, 40, 40, 1560, 9360, left=6240, sinks=1560, rolling=True),
        # single tokens of 32 sequences over long caches
        _attention("attention_token", 32, 32, 8, 1, 16384, left=8191, right=0, sinks=64, ragged=True),
        # a few queries over a short context: latency
        _attention("attention_short", 3, 6, 2, 77, 333, dim=64, dtype="f16", left=100, right=0, sinks=3),
        # a benchmark frame's heads on their way into a rolling cache
        _cache("cache_frame", 1, 3600, 40, 40, 14400, per_head=False, sinks=3600, rolling=True),
        # single tokens of 32 sequences, each at its own place of its cache
        _cache("cache_token", 32, 1, 32, 8, 1088, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_linear(rng):
    while True:
        n, k = _log_int(rng, 64, 13824), _log_int(rng, 64, 13824)
        if rng.random() < 0.6:  # widths of models are multiples of 64, others happen
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        m = _log_int(rng, 1, 75600)
        case = _linear("", m, n, k, dtype=rng.choice(["bf16", "bf16", "f16"]), bias=rng.random() < 0.7,
                       act=rng.choice(["none", "none", "gelu_tanh", "silu", "gelu"]), gate=rng.random() < 0.3,
                       residual=rng.random() < 0.4)
        if 2.0 * m * n * k <= MAX_FLOPS:
            return case


def _draw_attention(rng):
    form = rng.choice(["video", "prompt", "text", "chunk", "token", "token"])
    dim, dtype = rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "f16"])
    while True:
        kv = rng.choice([1, 2, 4, 8, 12])
        heads = kv * rng.choice([1, 2, 4, 5])
        if form == "video":
            length = _log_int(rng, 256, 75600)
            side = _log_int(rng, 16, 8000)
            case = _attention("", 1, heads, kv, length, length, dim, dtype, left=side, right=side,
                              sinks=rng.choice([0, _log_int(rng, 1, 4000)]))
        elif form == "prompt":
            length = _log_int(rng, 1, 12000)
            case = _attention("", rng.randint(1, 4), heads, kv, length, length, dim, dtype,
                              left=rng.choice([-1, _log_int(rng, 1, 8000)]), right=0, sinks=rng.choice([0, 1, 4, 64]),
                              ragged=rng.random() < 0.5)
        elif form == "text":
            case = _attention("", 1, heads, heads, _log_int(rng, 64, 75600), _log_int(rng, 16, 512), dim, dtype,
                              ragged=rng.random() < 0.5)
        elif form == "chunk":
            tokens, keep, sinks = _log_int(rng, 2, 2000), _log_int(rng, 16, 8000), rng.choice([0, 4, 64, 1560])
            rolling = rng.random() < 0.7
            case = _attention("", rng.randint(1, 2), heads, kv, tokens, sinks + keep + tokens, dim, dtype, left=keep,
                              right=rng.choice([-1, 0]), sinks=sinks, rolling=rolling, ragged=not rolling)
        else:
            rolling = rng.random() < 0.4
            slots = _log_int(rng, 128, 32768)
            sinks = min(rng.choice([0, 4, 64]), slots // 2)
            left = slots - sinks - 1 if rolling else rng.choice([-1, _log_int(rng, 16, slots)])
            case = _attention("", rng.choice([1, 2, 7, 16, 32, 64]), heads, kv, 1, slots, dim, dtype, left=left,
                              right=0, sinks=sinks, ragged=True, rolling=rolling)
        w = work(case)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= 4e9 and _held(case) <= 4e9:
            return case


def _draw_cache(rng):
    while True:
        kv = rng.choice([1, 2, 8, 12, 40])
        heads = kv * (rng.choice([1, 2, 4, 5]) if kv < 40 else 1)
        tokens = _log_int(rng, 2, 8000) if rng.random() < 0.5 else 1
        batch = 1 if tokens > 500 else rng.choice([1, 3, 16, 32])
        dim, sinks = rng.choice([128, 128, 64]), rng.choice([0, 4, 64])
        case = _cache("", batch, tokens, heads, kv, sinks + tokens + _log_int(rng, 16, 2000), dim,
                      rng.choice(["bf16", "bf16", "f16"]), per_head=rng.random() < 0.6, sinks=sinks,
                      ragged=rng.random() < 0.6, rolling=rng.random() < 0.5)
        if heads * dim <= 8192 and _held(case) <= 1e9:
            return case


def draw(rng):
    case = rng.choice([_draw_linear, _draw_attention, _draw_cache])(rng)
    del case["name"]
    return case


# --------------------------------------------------------------------------
# sizes
# --------------------------------------------------------------------------

def _held(case):
    """Bytes of keys and values held, those that no query sees among them."""
    rows = case["lk"] if case["kind"] == "attention" else case["slots"]
    return 4.0 * case["batch"] * case["kv_heads"] * rows * case["dim"]


def _seen(lq, lk, left, right, sinks):
    """(pairs of queries and keys that see each other, keys that some query sees), queries at the end."""
    i = torch.arange(lq, dtype=torch.int64) + (lk - lq)
    hi = (i + right if right >= 0 else torch.full_like(i, lk)).clamp(max=lk - 1)
    lo = (i - left if left >= 0 else torch.zeros_like(i)).clamp(min=0)
    near = (hi - lo + 1).clamp(min=0)
    first = torch.minimum(torch.full_like(i, sinks) - 1, torch.minimum(hi, lo - 1)) + 1
    low = int(lo.min())
    return int((near + first.clamp(min=0)).sum()), max(int(hi.max()) + 1 - low, 0) + min(sinks, low)


def _lengths(case):
    """Host lengths that the case's sequences have: (of queries, of keys), before any seed: the longest is whole."""
    b = case["batch"]
    if case["kind"] == "cache":
        free = case["slots"] - case["tokens"]
        if case["rolling"]:
            return None, [case["slots"] + 37 * i for i in range(b)]
        return None, [free * (i + 1) // b if case["ragged"] else free // 2 for i in range(b)]
    lq, lk = case["lq"], case["lk"]
    if case["rolling"]:
        return [lq] * b, [lk + lk // 3 + 101 * i for i in range(b)]
    if not case["ragged"]:
        return [lq] * b, [lk] * b
    keys = [max(lk - (lk * i * 5 // (b * 8)), 1) for i in range(b)] if b > 1 else [max(lk * 5 // 8, 1)]
    if lq == lk:  # padded prompts
        return keys, keys
    if case["right"] < 0 and case["left"] < 0:  # text: every query sees the keys that are there
        return [lq] * b, keys
    return [lq] * b, [max(n, lq) for n in keys]


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        size = m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
        return {"bytes": 2.0 * size + (4.0 * n if case["gate"] else 0.0), "flops": 2.0 * m * n * k}
    b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "attention":
        ql, kl = _lengths(case)
        pairs = [_seen(n, m, case["left"], case["right"], case["sinks"]) for n, m in zip(ql, kl)]
        out = b * h * case["lq"] * d  # rows behind a sequence are written too
        return {"bytes": 2.0 * (out + sum(n * h * d for n in ql) + sum(2 * p[1] * g * d for p in pairs)),
                "flops": 4.0 * h * d * sum(p[0] for p in pairs)}
    t = b * case["tokens"]
    c = 2.0 * t * d * (h + 2 * g)
    return {"bytes": 2 * c + 4.0 * t * d, "flops": t * d * (h + g) * 8.0}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32) * std).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32).to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _normal(gen, m, k, dtype=dt)
        s["w"] = _normal(gen, n, k, std=1.0 / math.sqrt(k), dtype=dt)
        s["bias"] = _normal(gen, n, std=0.1, dtype=dt) if case["bias"] else None
        s["gate"] = _normal(gen, n, std=0.5) if case["gate"] else None
        s["residual"] = _normal(gen, m, n, dtype=dt) if case["residual"] else None
        return s
    b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    ql, kl = _lengths(case)
    if case["kind"] == "attention":
        # projections lie in token order, a cache head by head
        s["q"] = _normal(gen, b, case["lq"], h, d, dtype=dt).transpose(1, 2)
        if case["lq"] == case["lk"]:
            s["k"], s["v"] = (_normal(gen, b, case["lk"], g, d, dtype=dt).transpose(1, 2) for _ in range(2))
        else:
            s["k"], s["v"] = (_normal(gen, b, g, case["lk"], d, dtype=dt) for _ in range(2))
        lens = case["ragged"] or case["rolling"]
        s["kv_lens"] = _int32(kl) if lens else None
        s["q_lens"] = _int32(ql) if lens and ql != [case["lq"]] * b else None
        s["host_lens"] = (ql, kl)
        return s
    t = case["tokens"]
    s["q"] = _normal(gen, b, t, h, d, std=1.5, dtype=dt)
    s["k"], s["v"] = (_normal(gen, b, t, g, d, std=1.5, dtype=dt) for _ in range(2))
    s["k_cache"], s["v_cache"] = (_normal(gen, b, g, case["slots"], d, dtype=dt) for _ in range(2))
    s["q_weight"] = (1 + _normal(gen, d if case["per_head"] else h * d, std=0.1)).to(dt)
    s["k_weight"] = (1 + _normal(gen, d if case["per_head"] else g * d, std=0.1)).to(dt)
    new = [max(t - t * i // (2 * b), 1) for i in range(b)] if case["ragged"] and t > 1 else None
    s["lens"], s["host_lens"] = _int32(kl), kl
    s["new_lens"], s["host_new"] = (_int32(new) if new else None), new or [t] * b
    rows = max(kl) + t
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    s["table"] = (torch.cos(angle).float().to(DEVICE), torch.sin(angle).float().to(DEVICE))
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _OWN[kind](s)
    return _PLAIN[kind](s)


# --------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------

def _limit(n):
    return None if n < 0 else n


def _own_linear(s):
    from dfsattn_amd import ops

    c = s["case"]
    return ops.linear(s["x"], s["w"], s["bias"], activation=None if c["act"] == "none" else c["act"], gate=s["gate"],
                      residual=s["residual"])


def _own_attention(s):
    from dfsattn_amd import ops

    c = s["case"]
    return ops.window_attention(s["q"], s["k"], s["v"], left=_limit(c["left"]), right=_limit(c["right"]),
                                sinks=c["sinks"], q_lens=s["q_lens"], kv_lens=s["kv_lens"], rolling=c["rolling"])


def _own_cache(s):
    from dfsattn_amd import ops

    c = s["case"]
    q = ops.qkv_cache(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["lens"], q_weight=s["q_weight"],
                      k_weight=s["k_weight"], eps=EPS, table=s["table"], new_lens=s["new_lens"], sinks=c["sinks"],
                      rolling=c["rolling"])
    return q, s["k_cache"], s["v_cache"]


_OWN = {"linear": _own_linear, "attention": _own_attention, "cache": _own_cache}


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
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _activate(y, s["case"]["act"])
    if s["gate"] is not None:
        y = y * s["gate"]
    if s["residual"] is not None:
        y = s["residual"].float() + y
    return y.to(s["x"].dtype)


def _slot_positions(case, kv_lens):
    """[B or 1, slots] position of the token that each slot holds, -1 for none."""
    slot = torch.arange(case["lk"], device=DEVICE)[None]
    if not case["rolling"]:
        return slot
    ring = case["lk"] - case["sinks"]
    n = kv_lens[:, None].long()
    last = slot + torch.div(n - 1 - slot, ring, rounding_mode="floor") * ring
    return torch.where(slot < n, torch.where(slot < case["sinks"], slot, last), -1)


def _plain_attention(s):
    c = s["case"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, h, lq, d = q.shape
    g, lk = k.shape[1], k.shape[2]
    n_q = (torch.full((1, 1), lq, device=DEVICE) if s["q_lens"] is None else s["q_lens"][:, None]).long()
    n_k = (torch.full((1, 1), lk, device=DEVICE) if s["kv_lens"] is None else s["kv_lens"][:, None]).long()
    place = _slot_positions(c, s["kv_lens"])
    out = torch.empty((b, lq, h, d), dtype=s["q"].dtype, device=DEVICE).transpose(1, 2)
    q = q.reshape(b, g, h // g, lq, d)
    step = max(1, int(4e8 // (b * h * lk)))
    if s["kv_lens"] is None and c["left"] >= 0 and c["right"] >= 0:
        step = max(512, step)
    for i0 in range(0, lq, step):
        i1 = min(lq, i0 + step)
        kc, vc, pc = k, v, place
        if s["kv_lens"] is None:  # the keys that these queries may see
            lo = max(0, lk - lq + i0 - c["left"]) if c["left"] >= 0 else 0
            hi = min(lk, max(0, lk - lq + i1 + c["right"])) if c["right"] >= 0 else lk
            first = min(c["sinks"], lo, hi)
            kc, vc, pc = (torch.cat([t[..., :first, :], t[..., lo:hi, :]], -2) for t in (k, v, place[..., None]))
            pc = pc[..., 0]
        i = torch.arange(i0, i1, device=DEVICE)[None]
        at = (n_k - n_q + i)[:, :, None]
        key = pc[:, None, :]
        see = (key >= 0) & (key < n_k[:, :, None]) & (i < n_q)[:, :, None]
        if c["right"] >= 0:
            see = see & (key <= at + c["right"])
        if c["left"] >= 0:
            see = see & ((key >= at - c["left"]) | (key < c["sinks"]))
        n = i1 - i0
        score = q[:, :, :, i0:i1].reshape(b, g, -1, d) @ kc.transpose(-1, -2).contiguous()
        score = score.reshape(b, g, h // g, n, -1) * (1 / math.sqrt(d))
        score = score.masked_fill(~see[:, None, None], -math.inf)
        top = score.amax(-1, keepdim=True) if score.shape[-1] else score.new_zeros((*score.shape[:-1], 1))
        p = torch.exp(score - top.masked_fill(top == -math.inf, 0))
        total = p.sum(-1, keepdim=True)
        o = (p.reshape(b, g, -1, p.shape[-1]) @ vc).reshape(b, g, h // g, n, d)
        o = torch.where(total > 0, o / total, 0)
        out[:, :, i0:i1] = o.reshape(b, h, n, d).to(out.dtype)
    return out


def _norm_rotate(x, weight, per_head, cos, sin):
    """x [B, T, H, D] normalised and rotated by [B, T, 1, D/2] tables, in x's type."""
    flat = x if per_head else x.flatten(2)
    y = flat / torch.sqrt((flat * flat).mean(-1, keepdim=True) + EPS) * weight
    y = y.reshape(x.shape)
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)


def _plain_cache(s):
    c = s["case"]
    dt, t = s["q"].dtype, c["tokens"]
    at = s["lens"][:, None].long() + torch.arange(t, device=DEVICE)[None]
    cos, sin = (x[at][:, :, None] for x in s["table"])
    q = _norm_rotate(s["q"].float(), s["q_weight"].float(), c["per_head"], cos, sin).to(dt)
    k = _norm_rotate(s["k"].float(), s["k_weight"].float(), c["per_head"], cos, sin).to(dt)
    slot = at
    if c["rolling"]:
        slot = torch.where(at < c["sinks"], at, c["sinks"] + (at - c["sinks"]) % (c["slots"] - c["sinks"]))
    if s["new_lens"] is None:
        row = torch.arange(c["batch"], device=DEVICE)[:, None]
        s["k_cache"][row, :, slot] = k
        s["v_cache"][row, :, slot] = s["v"]
    else:
        q = q * (torch.arange(t, device=DEVICE)[None] < s["new_lens"][:, None])[:, :, None, None]
        for b, n in enumerate(s["host_new"]):
            s["k_cache"][b][:, slot[b, :n]] = k[b, :n].transpose(0, 1)
            s["v_cache"][b][:, slot[b, :n]] = s["v"][b, :n].transpose(0, 1)
    return q.transpose(1, 2), s["k_cache"], s["v_cache"]


_PLAIN = {"linear": _plain_linear, "attention": _plain_attention, "cache": _plain_cache}


# --------------------------------------------------------------------------
# definitions, in 64 bits
# --------------------------------------------------------------------------

def _slot_of(case, positions, slots):
    if not case["rolling"]:
        return positions
    ring = slots - case["sinks"]
    return torch.where(positions < case["sinks"], positions, (positions - case["sinks"]).remainder(ring) + case["sinks"])


def _exact_linear(s):
    w = s["w"].double().t().contiguous()
    parts = []
    for x, r in zip(s["x"].split(8192), s["residual"].split(8192) if s["residual"] is not None else [None] * 10**6):
        z = torch.mm(x.double(), w)
        if s["bias"] is not None:
            z += s["bias"].double()
        act = s["case"]["act"]
        if act == "silu":
            z = z * torch.sigmoid(z)
        elif act == "gelu":
            z = z * 0.5 * torch.erfc(z * -(2 ** -0.5))
        elif act == "gelu_tanh":  # (1 + tanh(u)) / 2 = sigmoid(2 u)
            z = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
        if s["gate"] is not None:
            z = z * s["gate"].double()
        parts.append(z if r is None else z + r.double())
    return torch.cat(parts)


def _exact_attention(s):
    c = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    b, h, lq, d = q.shape
    g, slots = k.shape[1], k.shape[2]
    out = torch.zeros((b, lq, h, d), dtype=torch.float64, device=DEVICE).transpose(1, 2)
    for bi in range(b):
        nq, nk = s["host_lens"][0][bi], s["host_lens"][1][bi]
        for i0 in range(0, nq, 1024):
            i1 = min(nq, i0 + 1024)
            at = torch.arange(nk - nq + i0, nk - nq + i1, device=DEVICE)
            lo = max(0, int(nk - nq + i0 - c["left"])) if c["left"] >= 0 else 0
            hi = min(nk, nk - nq + i1 + c["right"]) if c["right"] >= 0 else nk
            keys = torch.cat([torch.arange(min(c["sinks"], lo, max(hi, 0)), device=DEVICE),
                              torch.arange(lo, max(lo, hi), device=DEVICE)])
            if keys.numel() == 0:
                continue
            hidden = torch.zeros((i1 - i0, keys.numel()), dtype=torch.bool, device=DEVICE)
            if c["right"] >= 0:
                hidden |= keys[None] - at[:, None] > c["right"]
            if c["left"] >= 0:
                hidden |= (at[:, None] - keys[None] > c["left"]) & (keys >= c["sinks"])[None]
            slot = _slot_of(c, keys, slots)
            for gi in range(g):
                kd, vd = k[bi, gi][slot].double(), v[bi, gi][slot].double()
                for hi_ in range(gi * (h // g), (gi + 1) * (h // g)):
                    z = torch.mm(q[bi, hi_, i0:i1].double() / math.sqrt(d), kd.t().contiguous())
                    z = torch.softmax(z.masked_fill_(hidden, -math.inf), -1)
                    out[bi, hi_, i0:i1] = torch.mm(torch.nan_to_num(z), vd)
    return out


def _exact_cache(s):
    c = s["case"]
    b, t, slots, d = c["batch"], c["tokens"], c["slots"], c["dim"]
    out = []
    for name, weight in (("q", "q_weight"), ("k", "k_weight")):
        x = s[name].double()
        w = s[weight].double()
        if c["per_head"]:
            y = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / d + EPS) * w
        else:
            y = x * torch.rsqrt(x.square().sum((-2, -1), keepdim=True) / x[0, 0].numel() + EPS) * w.view(-1, d)
        z = torch.view_as_complex(y.unflatten(-1, (-1, 2)).contiguous())
        for i in range(b):
            n = s["host_lens"][i]
            turn = torch.complex(s["table"][0][n:n + t].double(), s["table"][1][n:n + t].double())
            z[i] = z[i] * turn[:, None]
        out.append(torch.view_as_real(z).flatten(-2).transpose(1, 2).contiguous())
    q, k = out
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    for i in range(b):
        n = s["host_new"][i]
        q[i, :, n:] = 0
        slot = _slot_of(c, torch.arange(n, device=DEVICE) + s["host_lens"][i], slots)
        k_cache[i].index_copy_(1, slot, k[i, :, :n])
        v_cache[i].index_copy_(1, slot, s["v"][i, :n].double().transpose(0, 1).contiguous())
    return q, k_cache, v_cache


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "attention": _exact_attention, "cache": _exact_cache}[case["kind"]](s)
