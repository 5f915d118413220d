"""GridRotary where the library's kernel does not run: the processor's torch path
in both layouts, and the tables it stands for (CPU)."""
import pytest
import torch

import block_refs as refs
import dfsattn_amd.replace_wan as wan
from dfsattn_amd import ops
from stubs import StubAttention

H, D, GRID, L = 2, 32, (3, 5), 30


def _axes(layout):
    return ops.RotaryAxes(D, (8, 12, 8), (1e4, 500.0, 1e3), layout, (1.0, -0.5, 2.0))


def _expected(x, rotary):
    """[B, H, L, D]: the 64-bit definition of x [B, L, H, D], already normalised."""
    a = rotary.axes
    places = refs.grid_positions([0] * x.shape[0], x.shape[1], rotary.grid)
    return refs.axial_rope(x, places, a.sections, a.theta, a.layout, speeds=a.speeds)


@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_processor_without_the_kernel_rotates_by_places(monkeypatch, layout):
    seen = {}

    def attention(query, key, value, **kw):
        seen.update(q=query, k=key, v=value)
        return torch.zeros_like(query)

    monkeypatch.setattr(wan, "full_attention", attention)
    rotary = ops.GridRotary(_axes(layout), GRID)
    g = torch.Generator().manual_seed(1)
    attn = StubAttention(dim=H * D, heads=H)
    x = torch.randn(1, L, H * D, generator=g)
    proc = wan.Wan_DFSAttn_Processor2_0("full", 0.0, 16, 128, None, 0, [], 0, 1, 0.0, False, False)
    with torch.no_grad():
        proc(attn, x, rotary_emb=rotary)
        for name, norm, layer in (("q", attn.norm_q, attn.to_q), ("k", attn.norm_k, attn.to_k)):
            want, tol = _expected(norm(layer(x)).unflatten(2, (H, D)), rotary)
            assert seen[name].dtype == x.dtype and bool(((seen[name].double() - want).abs() <= tol).all())
        assert torch.equal(seen["v"], attn.to_v(x).unflatten(2, (H, D)).transpose(1, 2))


@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_rotate_keeps_types_and_refuses_other_heads(layout):
    rotary = ops.GridRotary(_axes(layout), GRID)
    g = torch.Generator().manual_seed(2)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.randn(2, L, H, D, generator=g).to(dtype)
        got, short = rotary.rotate(x.transpose(1, 2), x[:, :7].transpose(1, 2))
        want, tol = _expected(x, rotary)
        assert got.dtype == dtype and bool(((got.double() - want).abs() <= tol).all())
        assert torch.equal(short, got[:, :, :7])
    with pytest.raises(ValueError, match="channels"):
        rotary.rotate(torch.zeros(1, H, L, D + 8))
