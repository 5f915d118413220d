"""64-bit definitions of ops.linear, ops.window_attention and ops.qkv_cache on
the CPU, each with an elementwise bound of what the kernels' roundings allow.

u = finfo(t).eps / 2 is one rounding to the type t, F = 2^-24 one to fp32."""
import math

import torch

F = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def activate(z, act):
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z * math.sqrt(0.5))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def linear(x, w, bias=None, act=None, gate=None, residual=None):
    """(value, bound). The sum of k + 1 terms is off by at most (k + 1) F of
    their magnitudes in any order (and an MFMA's own order adds no more), the
    activations' slopes stay below 1.13, their exponentials and quotients are
    off by relative 2^-16 (erfc's argument t carries F t into 2 t^2 F, t < 10),
    the gate and the sum with the residual round once each, and the result
    once to its type (f16 values below 2^-14 in steps of 2^-24)."""
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    if bias is not None:
        z = z + bias.double()
        mag = mag + bias.double().abs()
    y = activate(z, act)
    err = 1.13 * (x.shape[-1] + 1) * F * mag + 2.0 ** -16 * y.abs()
    if gate is not None:
        y, err = y * gate.double(), (err + F * y.abs()) * gate.double().abs()
    if residual is not None:
        y = residual.double() + y
        err = err + F * y.abs()
    return y, err + half_step(x.dtype) * (y.abs() + err) + 2.0 ** -25


def slot_of(pos, slots, sinks, rolling):
    return pos if not rolling or pos < sinks else sinks + (pos - sinks) % (slots - sinks)


def window_attention(q, k, v, left=None, right=None, sinks=0, q_lens=None, kv_lens=None, rolling=False, scale=None):
    """(out, lse, bound of out, bound of lse). Scores: a D-term fp32 sum, the
    scale and the base change are off by ds = (D + 4) F of the magnitudes, so a
    weight by relative 2 ds, and by one rounding u to the operands' type; the
    sums over n keys by n F. The output takes twice that (numerator and
    denominator) of sum p |v|, and one rounding."""
    B, H, L, D = q.shape
    G, S = k.shape[1:3]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, H, L, D, dtype=torch.float64)
    lse = torch.full((B, H, L), -math.inf, dtype=torch.float64)
    tol, lse_tol = torch.full_like(out, 2.0 ** -25), torch.full_like(lse, 1e-6)
    u = half_step(q.dtype)
    for b in range(B):
        nq = L if q_lens is None else min(max(int(q_lens[b]), 0), L)
        nk = S if kv_lens is None else max(int(kv_lens[b]), 0)
        if not rolling:
            nk = min(nk, S)
        for i in range(nq):
            p = nk - nq + i
            keys = [j for j in range(nk) if (right is None or j <= p + right)
                    and (left is None or j >= p - left or j < sinks)]
            if not keys:
                continue
            slots = [slot_of(j, S, sinks, rolling) for j in keys]
            for g in range(G):
                hs = slice(g * (H // G), (g + 1) * (H // G))
                qd, kd, vd = q[b, hs, i].double(), k[b, g, slots].double(), v[b, g, slots].double()
                s = qd @ kd.t() * scale
                ds = (D + 4) * F * float((qd.abs() @ kd.abs().t()).max()) * scale
                m = s.max(-1, keepdim=True).values
                e = torch.exp(s - m)
                tot = e.sum(-1, keepdim=True)
                out[b, hs, i] = e / tot @ vd
                lse[b, hs, i] = (m + tot.log())[:, 0]
                rel = 2 * (u + 2 * ds + (len(keys) + 8) * F)
                tol[b, hs, i] += rel * (e / tot @ vd.abs()) + u * (1 + rel) * out[b, hs, i].abs()
                lse_tol[b, hs, i] += rel + 4 * F * lse[b, hs, i].abs()
    return out, lse, tol, lse_tol


def qkv_cache(q, k, v, k_cache, v_cache, lens, q_weight=None, k_weight=None, eps=1e-6, table=None, new_lens=None,
              sinks=0, rolling=False):
    """(q, k_cache, v_cache, bound of q, bound of k_cache): the mean square of
    C channels is off by relative C F, its root and quotient by a few F, the
    rotation's products and sum by 3 F of their magnitudes; one rounding."""
    B, T, _, D = q.shape
    S = k_cache.shape[2]
    res = []
    for x, w in ((q, q_weight), (k, k_weight)):
        y = x.double()
        if w is not None:
            flat = y if w.numel() == D else y.flatten(2)
            y = (flat / torch.sqrt(flat.square().mean(-1, keepdim=True) + eps) * w.double()).reshape(x.shape)
        mag = y.abs()
        if table is not None:
            z = torch.empty_like(y)
            for b in range(B):
                c, s = (t[int(lens[b]):int(lens[b]) + T].double()[:, None] for t in table)
                a, d = y[b, ..., 0::2], y[b, ..., 1::2]
                z[b] = torch.stack([a * c - d * s, d * c + a * s], -1).flatten(-2)
                big = a.abs() + d.abs()
                mag[b] = torch.stack([big, big], -1).flatten(-2)
            y = z
        C = D if w is None or w.numel() == D else w.numel()
        res.append((y, (C + 16) * F * mag + half_step(x.dtype) * (y.abs() + 16 * F * mag) + 2.0 ** -25))
    (qd, qt), (kd, kt) = res
    kc, vc, kct = k_cache.double(), v_cache.double(), torch.zeros(k_cache.shape, dtype=torch.float64)
    for b in range(B):
        n = T if new_lens is None else int(new_lens[b])
        qd[b, n:] = 0
        for t in range(n):
            slot = slot_of(int(lens[b]) + t, S, sinks, rolling)
            if slot < S:
                kc[b, :, slot], vc[b, :, slot], kct[b, :, slot] = kd[b, t], v[b, t].double(), kt[b, t]
    return qd.transpose(1, 2), kc, vc, qt.transpose(1, 2), kct
