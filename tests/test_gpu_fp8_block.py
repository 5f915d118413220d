"""The operators of a block together: DiTBlock on ops.residual_norm, its
feed-forward products on 8-bit operands, rotary positions from the grid in the
processors and in streams."""
import math

import pytest
import torch

import block_refs as refs
from dfsattn_amd import ops
from dfsattn_amd.dit import DIT_CONFIGS, build_model, install_dfs_processors, synth_inputs
from dfsattn_amd.fp8 import Fp8Linear, install_fp8
from dfsattn_amd.replace_wan import fused_qkv_heads
from dfsattn_amd.streaming import StreamCache, install_stream_processors

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _model(dev, **kw):
    model = build_model(DIT_CONFIGS["tiny"], dev)
    install_dfs_processors(model, mode="full", **kw)
    return model


def _block_inputs(dev, model, seed=0):
    g = torch.Generator().manual_seed(seed)
    cfg = model.cfg
    x = torch.randn(1, cfg.seq_len, cfg.dim, generator=g).to(BF).to(dev)
    ctx = torch.randn(1, cfg.text_len, cfg.dim, generator=g).to(BF).to(dev)
    temb = (0.3 * torch.randn(1, 6, cfg.dim, generator=g)).to(BF).to(dev)
    return x, ctx, temb


@torch.no_grad()
def test_block_keeps_its_results(dev):
    """The block's residuals and norms in one pass give what they gave in two."""
    model = _model(dev)
    block = model.blocks[0]
    x, ctx, temb = _block_inputs(dev, model)
    got = block(x, ctx, temb, model.rotary_emb)
    m = (block.scale_shift_table + temb.float()).chunk(6, 1)
    h = ops.adaln_modulate(x, block.norm1.eps, scale=m[1], shift=m[0])
    y = ops.gated_residual(x, block.attn1(h, None, None, model.rotary_emb), m[2])
    h = ops.adaln_modulate(y, block.norm2.eps, weight=block.norm2.weight.float(), bias=block.norm2.bias.float())
    y = y + block.attn2(h, ctx)
    h = ops.adaln_modulate(y, block.norm3.eps, scale=m[4], shift=m[3])
    assert torch.equal(got, ops.gated_residual(y, block._ffn_fused(h), m[5]))


@torch.no_grad()
def test_block_with_8_bit_ffn_is_its_operators(dev):
    model = _model(dev)
    block = model.blocks[1]
    x, ctx, temb = _block_inputs(dev, model, 1)
    lin1, lin2 = block.ffn[0], block.ffn[2]
    assert install_fp8(model, attention=False) == 2 * len(model.blocks)
    got = block(x, ctx, temb, model.rotary_emb)
    m = (block.scale_shift_table + temb.float()).chunk(6, 1)
    h = ops.adaln_modulate(x, block.norm1.eps, scale=m[1], shift=m[0])
    x, h = ops.residual_norm(x, block.attn1(h, None, None, model.rotary_emb), m[2], weight=block.norm2.weight,
                             bias=block.norm2.bias)
    x, h = ops.residual_norm(x, block.attn2(h, ctx), scale=m[4], shift=m[3])
    a = ops.linear_fp8(h, *ops.quantize_fp8(lin1.weight), bias=lin1.bias, activation="gelu_tanh")
    assert torch.equal(got, ops.linear_fp8(a, *ops.quantize_fp8(lin2.weight), bias=lin2.bias, gate=m[5], residual=x))


@torch.no_grad()
def test_fp8_linear_against_its_layer(dev):
    """Codes are off by 2^-4 of a value at most (and values below a block's
    normal range by half a step, 2^-10 of its scale, at most 2^-17 of its
    largest), so a product of two by 2^-3 + 2^-8, the sums as bounded before."""
    for m, n, k in ((5, 100, 300), (200, 300, 640)):
        print(f"Fp8Linear {m} x {n} x {k}", flush=True)
        g = torch.Generator().manual_seed(n)
        layer = torch.nn.Linear(k, n, dtype=BF)
        layer.weight.copy_(torch.randn(n, k, generator=g) / math.sqrt(k))
        x = torch.randn(m, k, generator=g).to(BF)
        got = Fp8Linear.from_linear(layer.to(dev))(x.to(dev))
        w, b = layer.weight.cpu().double(), layer.bias.cpu().double()
        ref = x.double() @ w.t() + b
        _, tol = refs.linear_fp8(x.double(), w, BF, layer.bias.cpu())
        top = (x.double().abs().amax(-1, keepdim=True) * w.abs().sum(-1)
               + x.double().abs().sum(-1, keepdim=True) * w.abs().amax(-1))
        tol = tol * 1.13 + (2.0 ** -3 + 2.0 ** -8) * (x.double().abs() @ w.abs().t()) + 2.0 ** -16 * top
        assert bool(((got.cpu().double() - ref).abs() <= tol).all())


@torch.no_grad()
def test_model_on_8_bit_layers(dev):
    """Every projection and product of the model on 8-bit operands: it runs, the
    same each time, and stays near the 16-bit model (each layer's products are
    off by 2^-3 of their magnitudes at most)."""
    model = _model(dev)
    latent, ctx, _ = synth_inputs(model.cfg, dev)
    t = torch.tensor([500.0], device=dev)
    before = model(latent, t, ctx)
    assert install_fp8(model) == 10 * len(model.blocks)
    after = model(latent, t, ctx)
    assert torch.equal(after, model(latent, t, ctx)) and bool(torch.isfinite(after).all())
    assert float((after - before).float().norm() / before.float().norm()) < 2.0 ** -3


@torch.no_grad()
def test_processor_with_rotary_axes(dev):
    """q and k of a processor by places on the grid and by the table, each within
    what its roundings allow of the definition; v untouched; the model's output."""
    model = _model(dev)
    attn = model.blocks[0].attn1
    cfg = model.cfg
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, cfg.seq_len, cfg.dim, generator=g).to(BF).to(dev) for _ in range(3))
    model.use_rotary_axes()
    rotary = model.rotary_axes
    got = fused_qkv_heads(attn, q, k, v, rotary, token_major=True)
    places = refs.grid_positions([0], cfg.seq_len, rotary.grid)
    for x, out, w in ((q, got[0], attn.norm_q.weight), (k, got[1], attn.norm_k.weight)):
        ref, tol = refs.axial_rope(x.cpu().unflatten(2, (cfg.heads, -1)), places, rotary.axes.sections,
                                   rotary.axes.theta, "pairs", w.cpu(), attn.norm_q.eps)
        assert bool(((out.cpu().double() - ref).abs() <= tol).all())
    assert torch.equal(got[2], v.unflatten(2, (cfg.heads, -1)).transpose(1, 2))
    attn.norm_k.eps = 1e-3
    two = fused_qkv_heads(attn, q, k, v, rotary)
    assert torch.equal(two[0], got[0]) and not torch.equal(two[1], got[1]) and two[2].is_contiguous()
    attn.norm_k.eps = attn.norm_q.eps
    latent, ctx, _ = synth_inputs(cfg, dev)
    t = torch.tensor([500.0], device=dev)
    by_places = model(latent, t, ctx)
    model.use_rotary_axes(False)
    by_table = model(latent, t, ctx)
    assert float((by_places - by_table).float().norm() / by_table.float().norm()) < 2.0 ** -6


@torch.no_grad()
def test_stream_with_rotary_axes_has_no_last_row(dev):
    """A stream by places equals one by a table while that lasts, goes on behind
    it, and far behind it where the host has moved it."""
    g = torch.Generator().manual_seed(3)
    B, H, D, chunk, grid = 2, 4, 128, 12, (3, 4)
    rotary = ops.GridRotary(ops.RotaryAxes(D, (44, 42, 42)), grid)
    freqs = rotary.table(3 * chunk).to(torch.complex64)[0, 0]
    table = (freqs.real.contiguous().to(dev), freqs.imag.contiguous().to(dev))
    w = (1 + 0.1 * torch.randn(H * D, generator=g)).to(BF).to(dev)
    one, two = (StreamCache(B, H, D, left=chunk, chunk=chunk, sinks=4, device=dev) for _ in range(2))
    for turn in range(6):
        q, k, v = (torch.randn(B, chunk, H, D, generator=g).to(BF).to(dev) for _ in range(3))
        out = one.attend(q, k, v, w, w, rotary=rotary)
        assert bool(torch.isfinite(out).all())
        if turn < 3:
            ref = two.attend(q, k, v, w, w, table=table)
            assert float((out - ref).float().norm() / ref.float().norm()) < 2.0 ** -6
            two.advance(chunk)
        one.advance(chunk)
    with pytest.raises(ValueError):
        two.attend(q, k, v, w, w, table=table)
    with pytest.raises(ValueError):
        one.attend(q, k, v, w, w, table=table, rotary=rotary)
    one.lens.fill_((1 << 30) // 12 * 12)
    assert bool(torch.isfinite(one.attend(q, k, v, w, w, rotary=rotary)).all())


@torch.no_grad()
def test_model_streams_on_8_bit_layers_with_rotary_axes(dev):
    """Frames through the model, past its grid's last one."""
    model = build_model(DIT_CONFIGS["tiny"], dev)
    install_fp8(model)
    model.use_rotary_axes()
    f, h, w = model.cfg.grid
    caches = install_stream_processors(model, left=2 * h * w, chunk=h * w, sinks=h * w)
    latent, ctx, _ = synth_inputs(model.cfg, dev)
    t = torch.tensor([500.0], device=dev)
    for i in range(f + 2):
        frame = latent[:, :, i % f:i % f + 1]
        out = model(frame, t, ctx)
        assert out.shape == frame.shape and bool(torch.isfinite(out).all())
        for c in caches:
            c.advance(h * w)


@torch.no_grad()
def test_stream_on_8_bit_layers_without_biases(dev):
    """The caches are of the layers' type, which no bias tells."""
    model = build_model(DIT_CONFIGS["tiny"], dev, torch.float16)
    for block in model.blocks:
        for name in ("to_q", "to_k", "to_v"):
            getattr(block.attn1, name).bias = None
    install_fp8(model)
    f, h, w = model.cfg.grid
    caches = install_stream_processors(model, left=h * w, chunk=h * w)
    assert all(c.k.dtype == torch.float16 and c.k.device == dev for c in caches)
    latent, ctx, _ = synth_inputs(model.cfg, dev)
    out = model(latent[:, :, :1], torch.tensor([500.0], device=dev), ctx)
    assert bool(torch.isfinite(out).all())


@torch.no_grad()
@pytest.mark.parametrize("which", [(0,), (2,), (0, 2)])
def test_ffn_with_8_bit_layers_and_the_native_products(dev, which):
    """native_ffn asks for the 16-bit products of both layers: a block with an
    8-bit one runs its layers as they are."""
    model = _model(dev)
    block = model.blocks[0]
    for i in which:
        block.ffn[i] = Fp8Linear.from_linear(block.ffn[i])
    x, ctx, temb = _block_inputs(dev, model)
    want = block(x, ctx, temb, model.rotary_emb)
    block.native_ffn = True
    assert torch.equal(block(x, ctx, temb, model.rotary_emb), want)
