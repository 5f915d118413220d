"""The window mode of full_attention and the Wan processor, the DiT block's own
FFN products and a stream over rolling caches, each against the same layer
without them."""
import pytest
import torch

import operator_refs as refs
from dfsattn_amd import ops
from dfsattn_amd.dit import DIT_CONFIGS, DiTAttention, build_model, install_dfs_processors, synth_inputs, wan_rope_freqs
from dfsattn_amd.fullattention import full_attention
from dfsattn_amd.replace_wan import Wan_DFSAttn_Processor2_0
from dfsattn_amd.streaming import StreamCache, Wan_Stream_Processor, install_stream_processors

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
STEP = 2.0 ** -9  # half a step of bf16


def _rel(a, b):
    return float((a.double() - b.double()).abs().mean() / b.double().abs().mean())


def _attention_module(dev, dim, heads, seed):
    torch.manual_seed(seed)
    m = DiTAttention(dim, heads, 1e-6, device=dev, dtype=BF)
    with torch.no_grad():
        for name, p in m.named_parameters():
            p.normal_(0, 1, generator=None).mul_(dim ** -0.5 if p.dim() == 2 else 0.1)
            if name.startswith("norm"):
                p.add_(1)
    return m


def _window_processor(window, sinks):
    return Wan_DFSAttn_Processor2_0("window", 0.0, 16, 128, None, 0, [], 0, 1, 0.0, False, False, window=window,
                                    sinks=sinks)


def test_full_attention_window_mode(dev):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 3, 170, 64, generator=g).to(BF) for _ in range(3))
    ref, _, tol, _ = refs.window_attention(q, k, v, 40, 7, 20)
    cu = torch.tensor([0, 170, 170], dtype=torch.int32)
    out = full_attention(q.to(dev), k.to(dev), v.to(dev), mode="window", cu_seqlens_q=cu, cu_seqlens_kv=cu,
                         window=(40, 7), sinks=20)
    assert bool(((out.cpu().double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("right,chunks", [(0, [40, 40, 40, 40]), (0, [7, 1, 60, 33, 59]), (None, [160])])
@torch.inference_mode()
def test_stream_equals_window_attention_of_the_whole(dev, right, chunks):
    """Chunk by chunk over a rolling cache against the window processor on all
    tokens. The two round q, k, v (the norms' kernels once and twice), P, the
    attention's output and its projection: six half steps between them at most
    on average; another window is off by far more."""
    print(f"stream right={right} chunks={chunks}", flush=True)
    dim, heads, left, sinks, n = 256, 2, 50, 10, sum(chunks)
    m = _attention_module(dev, dim, heads, 3)
    x = torch.randn(1, n, dim, device=dev, generator=torch.Generator(dev).manual_seed(1)).to(BF)
    freqs = wan_rope_freqs((4, 5, 8), dim // heads).to(dev)
    m.set_processor(_window_processor((left, right), sinks))
    whole = m(x, None, None, freqs)
    m.set_processor(_window_processor((left + 25, right), sinks))
    other = m(x, None, None, freqs)
    cache = StreamCache(1, heads, dim // heads, left, max(chunks), sinks, dev, BF)
    m.set_processor(Wan_Stream_Processor(cache, right))
    parts, at = [], 0
    for c in chunks:
        m(torch.randn_like(x[:, :c]), None, None, freqs)  # an unfinished pass, written over
        parts.append(m(x[:, at:at + c], None, None, freqs))
        cache.advance(c)
        at += c
    got = torch.cat(parts, 1)
    assert _rel(got, whole) < 6 * STEP
    assert _rel(other, whole) > 10 * _rel(got, whole)
    assert int(cache.lens) == n


@torch.inference_mode()
def test_stream_of_two_batches_keeps_them_apart(dev):
    dim, heads = 256, 2
    m = _attention_module(dev, dim, heads, 4)
    x = torch.randn(2, 60, dim, device=dev, generator=torch.Generator(dev).manual_seed(2)).to(BF)
    freqs = wan_rope_freqs((3, 4, 5), dim // heads).to(dev)

    def run(x):
        cache = StreamCache(x.shape[0], heads, dim // heads, 16, 20, 4, dev, BF)
        m.set_processor(Wan_Stream_Processor(cache))
        out = []
        for at in range(0, 60, 20):
            out.append(m(x[:, at:at + 20], None, None, freqs))
            cache.advance(20)
        return torch.cat(out, 1)

    both = run(x)
    # two rows or one take other tile sizes in the products, so sums in another order
    assert _rel(both[:1], run(x[:1].contiguous())) < 6 * STEP and _rel(both[1:], run(x[1:].contiguous())) < 6 * STEP


def test_stream_cache_refuses(dev):
    cache = StreamCache(1, 2, 64, 8, 4, 2, dev, BF)
    q = torch.zeros(1, 5, 2, 64, dtype=BF, device=dev)
    with pytest.raises(ValueError, match="chunk"):
        cache.attend(q, q, q)
    with pytest.raises(ValueError, match="advance"):
        cache.advance(5)
    with pytest.raises(ValueError):
        StreamCache(1, 2, 64, -1, 4, 0, dev, BF)


@torch.inference_mode()
def test_model_streams_its_frames(dev):
    """The tiny DiT frame by frame: output shapes, finite values, caches that
    advance; the first chunk, which sees itself alone, equals a window run on
    those frames."""
    cfg = DIT_CONFIGS["tiny"]
    model = build_model(cfg, dev)
    latent, ctx, _ = synth_inputs(cfg, dev)
    frame = cfg.grid[1] * cfg.grid[2]
    t = torch.tensor([500.0], device=dev)
    caches = install_stream_processors(model, left=2 * frame, chunk=frame, sinks=frame)
    assert len(caches) == cfg.layers
    outs = []
    for f in range(cfg.grid[0]):
        outs.append(model(latent[:, :, f:f + 1], t, ctx))
        for c in caches:
            c.advance(frame)
    assert all(o.shape == latent[:, :, :1].shape and bool(torch.isfinite(o).all()) for o in outs)
    assert all(int(c.lens) == cfg.seq_len for c in caches)
    install_dfs_processors(model, mode="window", window=(frame, None), sinks=0)
    model.rotary_emb = model.rotary_emb[:, :, :frame].contiguous()
    first = model(latent[:, :, :1], t, ctx)
    assert _rel(outs[0], first) < 2 * 16 * STEP  # two layers of at most 16 roundings each


@torch.inference_mode()
def test_block_with_its_own_ffn(dev):
    """native_ffn against the default FFN of the same block: GELU's input and
    the second product are rounded in one and not in the other."""
    cfg = DIT_CONFIGS["tiny"]
    model = build_model(cfg, dev)
    latent, ctx, _ = synth_inputs(cfg, dev)
    install_dfs_processors(model, mode="window", window=(64, 64), sinks=32)
    t = torch.tensor([500.0], device=dev)
    base = model(latent, t, ctx)
    for b in model.blocks:
        b.native_ffn = True
    own = model(latent, t, ctx)
    assert not torch.equal(base, own)
    assert _rel(own, base) < 2 * 4 * STEP  # two layers, four roundings that differ in each
    h = torch.randn(1, 77, cfg.dim, device=dev).to(BF)
    x = torch.randn(1, 77, cfg.dim, device=dev).to(BF)
    gate = torch.randn(1, 1, cfg.dim, device=dev)
    blk = model.blocks[0]
    l1, _, l2 = blk.ffn
    got = blk._ffn_native(h, x, gate)
    a = ops.linear(h, l1.weight, l1.bias, activation="gelu_tanh").cpu()
    ref, tol = refs.linear(a[0], l2.weight.cpu(), l2.bias.cpu(), None, gate[0, 0].cpu(), x[0].cpu())
    assert bool(((got[0].cpu().double() - ref).abs() <= tol).all())


@torch.inference_mode()
def test_stream_past_its_table_is_refused_and_graphs_move_on(dev):
    """A chunk past the rotary table raises before anything is written; a
    captured advance, whose replays the host does not see, leaves the place
    unknown."""
    dim, heads = 256, 2
    m = _attention_module(dev, dim, heads, 5)
    x = torch.randn(1, 8, dim, device=dev).to(BF)
    freqs = wan_rope_freqs((1, 4, 5), dim // heads).to(dev)
    cache = StreamCache(1, heads, dim // heads, 8, 8, 0, dev, BF)
    m.set_processor(Wan_Stream_Processor(cache))
    for _ in range(2):
        m(x, None, None, freqs)
        cache.advance(8)
    kept = cache.k.clone()
    with pytest.raises(ValueError, match="table"):
        m(x, None, None, freqs)  # positions 16 to 23 of 20
    assert torch.equal(kept, cache.k) and bool(torch.isfinite(m(x[:, :4], None, None, freqs)).all())
    cache.reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.advance(4)
    assert cache._position() is None
    for i in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        assert int(cache.lens) == 4 * i
    cache.reset()
    assert cache._position() == 0 and int(cache.lens) == 0
