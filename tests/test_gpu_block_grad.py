"""DiTBlock's fused passes with gradients enabled: they have no backward, for
16-bit and 8-bit feed-forward layers alike."""
import pytest
import torch

from dfsattn_amd.dit import DIT_CONFIGS, build_model, install_dfs_processors, synth_inputs
from dfsattn_amd.fp8 import install_fp8

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _model(dev, layers):
    model = build_model(DIT_CONFIGS["tiny"], dev)
    model.requires_grad_(True)
    install_dfs_processors(model, mode="full")
    if "8-bit" in layers:
        install_fp8(model, attention=layers == "all 8-bit")
    if layers == "native":
        for block in model.blocks:
            block.native_ffn = True
    return model


@pytest.mark.parametrize("layers", ["16-bit", "8-bit ffn", "all 8-bit"])
def test_block_runs_and_its_backward_raises(dev, layers):
    print(f"block with gradients, {layers}", flush=True)
    model = _model(dev, layers)
    block, cfg = model.blocks[0], model.cfg
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, cfg.seq_len, cfg.dim, generator=g).to(BF).to(dev)
    ctx = torch.randn(1, cfg.text_len, cfg.dim, generator=g).to(BF).to(dev)
    temb = (0.3 * torch.randn(1, 6, cfg.dim, generator=g)).to(BF).to(dev)
    with torch.no_grad():
        want = block(x, ctx, temb, model.rotary_emb)
    got = block(x, ctx, temb, model.rotary_emb)
    assert torch.equal(got, want) and got.requires_grad and not want.requires_grad
    with pytest.raises(RuntimeError, match="no backward"):
        got.float().sum().backward()
    block.requires_grad_(False)
    assert not block(x, ctx, temb, model.rotary_emb).requires_grad
    for i in range(3):  # any input's want is enough
        ins = [x.clone(), ctx.clone(), temb.clone()]
        ins[i].requires_grad_()
        got = block(*ins, model.rotary_emb)
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="no backward"):
            got.float().sum().backward()


@pytest.mark.parametrize("layers", ["16-bit", "native", "8-bit ffn", "all 8-bit"])
def test_model_runs_with_gradients_enabled(dev, layers):
    print(f"model with gradients, {layers}", flush=True)
    model = _model(dev, layers)
    latent, ctx, _ = synth_inputs(model.cfg, dev)
    t = torch.tensor([500.0], device=dev)
    with torch.no_grad():
        want = model(latent, t, ctx)
    got = model(latent, t, ctx)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no backward"):
        got.float().sum().backward()
    # a head over frozen blocks trains
    model.requires_grad_(False)
    model.proj_out.requires_grad_(True)
    model(latent, t, ctx).float().sum().backward()
    assert bool(torch.isfinite(model.proj_out.weight.grad).all()) and float(model.proj_out.weight.grad.abs().max()) > 0
