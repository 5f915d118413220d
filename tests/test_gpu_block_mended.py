"""Calls of the block operators that once answered otherwise than documented."""
import pytest
import torch

from dfsattn_amd import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("quantize", [False, True])
def test_residual_norm_of_x_alone_returns_x(dev, quantize):
    """Also where x's rows, or a modulation, are laid out anew for the kernel."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 3, 64, generator=g).to(BF).to(dev)
    scale = torch.randn(4, 3, 64, generator=g).to(dev)
    for view, s in ((x, None), (x.transpose(0, 1), None), (x, scale.transpose(0, 1).contiguous().transpose(0, 1)),
                    (x[:, :, ::2], None), (x[:0].transpose(0, 1), None)):
        got = ops.residual_norm(view, scale=s, quantize=quantize)
        assert got[0] is view
        want = ops.residual_norm(view.contiguous(), scale=None if s is None else s.contiguous(), quantize=quantize)
        for a, b in zip(got[1:], want[1:]):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
