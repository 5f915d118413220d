"""Rotary positions from the grid for heads that ops.axial_rope does not take:
the fused projections' heads by the table, or in torch."""
import pytest
import torch

import block_refs as refs
from dfsattn_amd import ops
from dfsattn_amd.replace_wan import Wan_DFSAttn_Processor2_0, fused_qkv_heads
from stubs import StubAttention

pytestmark = pytest.mark.gpu


def _close(got, x, norm, rotary, heads):
    """x, the projection's output, to got [B, H, L, D]: the norm may be rounded to
    x's type before the rotation, which is off by what a rounding of either
    channel of a pair is."""
    a = rotary.axes
    xh = x.cpu().unflatten(2, (heads, -1))
    places = refs.grid_positions([0], x.shape[1], rotary.grid)
    want, tol = refs.axial_rope(xh, places, a.sections, a.theta, a.layout, norm.weight.detach().cpu(), norm.eps)
    y = xh.double()
    y = y / torch.sqrt(y.flatten(2).square().mean(-1, keepdim=True) + norm.eps)[..., None] \
        * norm.weight.detach().cpu().double().view(heads, -1)
    pair = y.unflatten(-1, (2, -1)).abs().sum(-2) if a.layout == "halves" else y.unflatten(-1, (-1, 2)).abs().sum(-1)
    pair = torch.cat([pair, pair], -1) if a.layout == "halves" else pair.repeat_interleave(2, -1)
    tol = tol + 1.01 * refs.half_step(x.dtype) * pair.transpose(1, 2)
    off = (got.cpu().double() - want).abs() - tol
    assert float(off.max()) <= 0, float(off.max())


@torch.no_grad()
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("heads,dim", [(64, 96), (65, 96), (80, 96), (31, 264)])
def test_heads_past_the_kernels(dev, heads, dim, layout):
    """64 heads of 96 channels are the kernel's most, 16 of 264."""
    print(f"rotary heads {heads} x {dim} {layout}", flush=True)
    g = torch.Generator().manual_seed(heads + dim)
    attn = StubAttention(dim=heads * dim, heads=heads)
    for norm in (attn.norm_q, attn.norm_k):
        norm.weight.copy_(1 + 0.2 * torch.randn(heads * dim, generator=g))
    attn.norm_k.eps = 1e-3
    side = 2 * (dim // 6)
    rotary = ops.GridRotary(ops.RotaryAxes(dim, (dim - 2 * side, side, side), layout=layout), (3, 4))
    q, k, v = (torch.randn(1, 30, heads * dim, generator=g).to(torch.bfloat16).to(dev) for _ in range(3))
    attn.norm_q, attn.norm_k = attn.norm_q.to(dev), attn.norm_k.to(dev)
    for token_major in (False, True):
        got = fused_qkv_heads(attn, q, k, v, rotary, token_major=token_major)
        _close(got[0], q, attn.norm_q, rotary, heads)
        _close(got[1], k, attn.norm_k, rotary, heads)
        assert torch.equal(got[2], v.unflatten(2, (heads, -1)).transpose(1, 2))


@torch.no_grad()
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("heads,dim", [(80, 96), (4, 64)])
def test_processor_hands_such_heads_on(dev, monkeypatch, heads, dim, layout):
    """What the processor's attention is given (which runs heads of 64 and 128
    alone), with the fused heads and in torch (mode "flash")."""
    import dfsattn_amd.replace_wan as wan

    print(f"processor heads {heads} x {dim} {layout}", flush=True)
    seen = []

    def attention(query, key, value, **kw):
        seen.append((query, key, value))
        return torch.zeros_like(query)

    monkeypatch.setattr(wan, "full_attention", attention)
    torch.manual_seed(5)
    attn = StubAttention(dim=heads * dim, heads=heads).to(dev, torch.bfloat16)
    side = 2 * (dim // 6)
    rotary = ops.GridRotary(ops.RotaryAxes(dim, (dim - 2 * side, side, side), layout=layout), (3, 4))
    x = torch.randn(1, 24, heads * dim, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(dev)
    for mode in ("full", "flash"):
        Wan_DFSAttn_Processor2_0(mode, 0.0, 16, 128, None, 0, [], 0, 1, 0.0, False, False)(attn, x, rotary_emb=rotary)
    _close(seen[0][0], attn.to_q(x), attn.norm_q, rotary, heads)
    _close(seen[0][1], attn.to_k(x), attn.norm_k, rotary, heads)
    y = attn.norm_q(attn.to_q(x)).unflatten(2, (heads, dim)).transpose(1, 2)
    assert torch.equal(seen[1][0], rotary.rotate(y)[0])
    assert torch.equal(seen[0][2], seen[1][2])
