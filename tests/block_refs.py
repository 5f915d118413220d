"""64-bit definitions of ops.quantize_fp8, ops.linear_fp8, ops.residual_norm and
ops.axial_rope on the CPU, each with an elementwise bound of what the kernels'
roundings allow.

u = finfo(t).eps / 2 is one rounding to the type t, F = 2^-24 one to fp32."""
import math

import torch

import operator_refs as refs
from operator_refs import F, half_step

BLOCK = 128


def e4m3(v):
    """v (64 bits, at most 448) rounded to e4m3, ties to even: 3 bits behind the
    leading one, steps of 2^-9 below 2^-6."""
    _, p = torch.frexp(v.abs().clamp(min=2.0 ** -6))
    step = torch.exp2((p - 4).double())
    return torch.round(v / step) * step  # torch.round: half to even


def block_exponents(x):
    """[rows, blocks] exponents of x [rows, k] (64 bits)."""
    e = []
    for b in x.split(BLOCK, -1):
        top = torch.where(torch.isfinite(b), b.abs(), 0).amax(-1)
        m, p = torch.frexp(top)
        least = torch.where(m <= 0.875, p - 9, p - 8)  # top = m 2^p <= 448 2^e, 448 = 0.875 2^9
        e.append(torch.where(top == 0, torch.zeros_like(least), least).clamp(-127, 127))
    return torch.stack(e, -1)


def quantize(x):
    """(codes' values, scales) of x [rows, k], in 64 bits; NaN where x is not finite."""
    x = x.double()
    scales = torch.exp2(block_exponents(x).double())
    wide = scales.repeat_interleave(BLOCK, -1)[:, :x.shape[-1]]
    v = x / wide
    return torch.where(torch.isfinite(x), e4m3(torch.where(torch.isfinite(x), v, 0)), math.nan), scales


def to_tensors(codes, scales):
    """Operands of linear_fp8 from quantize's values (exact in both types)."""
    return codes.to(torch.float8_e4m3fn), (torch.log2(scales) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def values(codes, scales):
    """What codes and scales [..., k] stand for, in 64 bits."""
    s = torch.exp2(scales.view(torch.uint8).double() - 127)
    return codes.double() * s.repeat_interleave(BLOCK, -1)[..., :codes.shape[-1]]


def linear_fp8(x, w, dtype, bias=None, act=None, gate=None, residual=None):
    """(value, bound) for operands x [m, k] and w [n, k] in 64 bits, as codes and
    scales stand for them: what operator_refs.linear allows its fp32 sums and
    epilogue, one rounding to the result's type, and what the 8-bit matrix
    instructions lose by themselves. They add the products of eight consecutive
    channels after cutting each, towards zero, to a multiple of 2^-13 of the
    largest one's power of two (one product of 2^16 beside another of 1.875 *
    1.875 * 2^s: kept whole down to s = 9, to 3.5 * 2^s down to s = 4, to 3 for
    s = 3, 2 for s = 2 and 0 below; products of other eights are kept whole).
    The largest loses nothing, having 8 bits, so the sum of eight is off by less
    than 7 * 2^-13 of the largest product, which is at most the largest |x|
    times the largest |w| of the eight."""
    y, err = refs.linear(x, w, bias, act, gate, residual)

    def eights(t):
        wide = torch.nn.functional.pad(t.abs(), (0, -t.shape[-1] % 8))
        return wide.unflatten(-1, (-1, 8)).amax(-1)

    lost = 1.13 * 7 * 2.0 ** -13 * (eights(x) @ eights(w).t())  # 1.13: the activations' slopes
    err = err + (lost if gate is None else lost * gate.double().abs())
    return y, err + half_step(dtype) * (y.abs() + err) + 2.0 ** -25
