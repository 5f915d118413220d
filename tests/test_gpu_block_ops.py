"""GPU parity of ops.residual_norm and ops.axial_rope with their 64-bit
definitions (block_refs)."""
import math

import pytest
import torch

import block_refs as refs
from dfsattn_amd import ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _randn(gen, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def _within(got, ref, tol, what=""):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    off = (got - ref).abs() - tol
    worst = int(off.argmax())
    assert float(off.max()) <= 0, (f"{what}: at {worst} got {float(got.flatten()[worst])}, want "
                                   f"{float(ref.flatten()[worst])} within {float(tol.flatten()[worst])}")


# --------------------------------------------------------------------------
# residual_norm
# --------------------------------------------------------------------------

NORM = [
    # lead, C, dtype, norm, post, weight type, gate, scale, shift (their lead shapes, None: absent), residual scale
    ((1,), 8, BF, "layer", None, None, None, None, None, 1.0),
    ((1,), 1, HF, "rms", None, F32, (), None, None, 1.0),
    ((3,), 2, BF, "layer", "layer", BF, (1,), None, (), 0.5),
    ((2, 5), 64, BF, "layer", None, F32, (2, 1), (2, 1), (2, 1), 1.0),
    ((2, 5), 77, HF, "rms", "rms", HF, (2, 1), (2, 5), (1, 5), 1.4),
    ((7,), 512, BF, "rms", None, BF, None, (), (), 1.0),
    ((3, 4, 5), 520, BF, "layer", "rms", F32, (3, 4, 1), (3, 1, 1), (4, 1), 1.0),
    ((130,), 1000, HF, "layer", "layer", F32, (), (), None, -0.25),
    ((65,), 1023, BF, "layer", None, BF, (65,), None, (), 1.0),
    ((9,), 1025, BF, "rms", "layer", F32, (), (), (), 1.0),
    ((33,), 1536, HF, "layer", None, None, (), (), (), 1.0),
    ((5,), 2049, BF, "layer", "rms", BF, (), None, None, 1.0),
    ((4, 3), 2560, BF, "rms", "rms", F32, (4, 1), (4, 1), (4, 1), 2.0),
    ((11,), 3584, HF, "layer", None, HF, (), (), (), 1.0),
    ((6,), 4100, BF, "rms", None, F32, (6,), (), None, 1.0),
    ((10,), 5120, BF, "layer", None, F32, (), (), (), 1.0),
    ((6,), 5120, HF, "rms", "rms", None, (), (), (), 1.0),
    ((3,), 6144, BF, "layer", "layer", F32, (), (), (), 1.0),
    ((3,), 7161, BF, "layer", None, F32, (), (), (), 1.0),
    ((2,), 8185, HF, "rms", "layer", BF, (2,), None, (2,), 1.0),
    ((5,), 8192, BF, "layer", "rms", F32, (), (), (), 1.0),
]


def _vectors(g, lead, C, std):
    return None if lead is None else _randn(g, *lead, C, std=std)


@pytest.mark.parametrize("lead,C,dtype,norm,post,wdt,gate,scale,shift,rs", NORM)
def test_residual_norm_matches_definition(dev, lead, C, dtype, norm, post, wdt, gate, scale, shift, rs):
    print(f"residual_norm {lead} x {C} {dtype} {norm} post={post} {wdt} gate={gate} scale={scale} shift={shift} {rs}",
          flush=True)
    g = torch.Generator().manual_seed(C + len(lead))
    x, y = _randn(g, *lead, C, dtype=dtype, std=2.0) + 0.5, _randn(g, *lead, C, dtype=dtype)
    kw = {"gate": _vectors(g, gate, C, 0.7), "residual_scale": rs, "post_norm": post,
          "post_weight": 1 + _randn(g, C, std=0.2) if post else None,
          "post_bias": _randn(g, C, dtype=HF) if post == "layer" else None}
    after = {"norm": norm, "weight": None if wdt is None else (1 + _randn(g, C, std=0.2)).to(wdt),
             "bias": None if wdt is None or norm == "rms" else _randn(g, C, dtype=wdt, std=0.3),
             "scale": _vectors(g, scale, C, 0.3), "shift": _vectors(g, shift, C, 0.3)}
    ref, tol = refs.residual(x, y, **kw)
    dv = {n: t.to(dev) if isinstance(t, torch.Tensor) else t for n, t in {**kw, **after}.items()}
    xd, yd = x.to(dev), y.to(dev)
    r, h = ops.residual_norm(xd, yd, **dv)
    assert r.dtype == h.dtype == dtype and r.is_contiguous() and h.is_contiguous()
    _within(r, ref, tol, "r")
    ref, tol = refs.norm_of(r.cpu(), **after)
    _within(h, ref, tol, "h")
    r2, codes, scales = ops.residual_norm(xd, yd, quantize=True, **dv)
    assert torch.equal(r, r2)
    want = ops.quantize_fp8(h)
    assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(scales.view(torch.uint8), want[1].view(torch.uint8))
    # x alone: its norm; in the place of x and of y
    only = {n: dv[n] for n in after}
    same, h3 = ops.residual_norm(r, **only)
    assert same is r and torch.equal(h3, h)
    for at in (xd.clone(), yd.clone()):
        a, b = (at, yd) if torch.equal(at, xd) else (xd, at)
        r4, h4 = ops.residual_norm(a, b, out=at, **dv)
        assert r4 is at and torch.equal(at, r) and torch.equal(h4, h)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,C", [(5, 256), (9000, 256), (300, 5120), (8200, 5120)])
def test_residual_norm_equals_the_two_calls(dev, rows, C, dtype):
    """What gated_residual and adaln_modulate give one after the other, bit for bit."""
    print(f"residual_norm against two calls {rows} x {C} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows + C)
    x, y = _randn(g, rows, C, dtype=dtype).to(dev), _randn(g, rows, C, dtype=dtype).to(dev)
    gate, w, b, sc, sh = (_randn(g, C).to(dev) for _ in range(5))
    r = ops.gated_residual(x, y, gate)
    for kw in ({"weight": w, "bias": b}, {"scale": sc, "shift": sh}, {"weight": w, "bias": b, "scale": sc, "shift": sh}, {}):
        got = ops.residual_norm(x, y, gate, **kw)
        assert torch.equal(got[0], r)
        assert torch.equal(got[1], ops.adaln_modulate(r, 1e-6, **kw))
    got = ops.residual_norm(x, y, scale=sc, shift=sh)
    assert torch.equal(got[0], x + y)
    assert torch.equal(got[1], ops.adaln_modulate(x + y, 1e-6, scale=sc, shift=sh))


# --------------------------------------------------------------------------
# axial_rope
# --------------------------------------------------------------------------

ROPE = [
    # B, T, H, G, D, dtype, sections, theta, layout, norm, weight type, grid or None, start
    (1, 1, 1, 1, 8, BF, (4, 2, 2), 1e4, "pairs", "none", None, (2, 3), None),
    (1, 7, 2, 2, 128, BF, (44, 42, 42), 1e4, "pairs", "all", BF, (2, 3), None),
    (2, 33, 8, 2, 128, HF, (44, 42, 42), 1e4, "halves", "head", F32, (3, 5), [5, 1 << 28]),
    (3, 5, 4, 1, 64, BF, (24, 20, 20), 1e4, "pairs", "head", HF, None, None),
    (2, 9, 12, 4, 96, BF, (32, 32, 32), 500.0, "halves", "all", F32, (4, 4), [0, 77]),
    (1, 17, 3, 5, 72, HF, (24, 24, 24), 1e4, "pairs", "head", BF, None, None),
    (2, 6, 5, 5, 80, BF, (16, 56), 1e4, "pairs", "all", BF, (9,), [1, 2]),
    (1, 11, 40, 40, 128, BF, (44, 42, 42), 1e4, "pairs", "all", BF, (45, 80), [3600]),
    (2, 3, 64, 8, 128, HF, (64, 32, 16), 1e4, "halves", "head", F32, None, None),
    (1, 4, 16, 16, 512, BF, (256, 128, 128), 1e6, "pairs", "head", F32, (2, 2), None),
    (1, 4, 3, 2, 248, BF, (120, 64), 1e4, "halves", "all", F32, (2,), [1000]),
    (2, 10, 100, 7, 32, HF, (8, 8, 8, 8), 1e4, "pairs", "none", None, (2, 3, 5), [11, 12]),
    (1, 3, 6, 6, 16, BF, (16,), 1e4, "pairs", "head", BF, (), [2147483000]),
    (1, 2, 20, 20, 40, BF, (20, 0, 10), 1e4, "pairs", "head", BF, None, None),
    (32, 1, 32, 8, 128, BF, (44, 42, 42), 1e4, "pairs", "head", BF, (30, 52), [1000 * i for i in range(32)]),
]


@pytest.mark.parametrize("B,T,H,G,D,dtype,sections,theta,layout,norm,wdt,grid,start", ROPE)
def test_axial_rope_matches_definition(dev, B, T, H, G, D, dtype, sections, theta, layout, norm, wdt, grid, start):
    print(f"axial_rope B={B} T={T} H={H} G={G} D={D} {dtype} {sections} {layout} {norm} grid={grid} start={start}",
          flush=True)
    g = torch.Generator().manual_seed(B * T + H * D)
    n = len(sections)
    axes = ops.RotaryAxes(D, sections, theta, layout)
    q, k = _randn(g, B, T, H, D, dtype=dtype, std=1.5), _randn(g, B, T, G, D, dtype=dtype, std=1.5)
    wq, wk = ((1 + _randn(g, c, std=0.2)).to(wdt) if norm != "none" else None
              for c in ((D, D) if norm == "head" else (H * D, G * D)))
    positions = None
    if grid is None:
        positions = torch.randint(-(1 << 20), 1 << 20, (B, T, n), generator=g).to(torch.int32)
        positions[:, 0] = 0
        places = positions
    else:
        places = refs.grid_positions(start or [0] * B, T, grid)
    d = [None if t is None else t.to(dev) for t in (q, k, wq, wk, positions)]
    st = None if start is None else torch.tensor(start, dtype=torch.int32).to(dev)
    kw = {"grid": grid, "start": st, "positions": d[4]}
    got = ops.axial_rope(d[0], d[1], axes, q_weight=d[2], k_weight=d[3], **kw)
    for x, w, out in ((q, wq, got[0]), (k, wk, got[1])):
        assert out.dtype == dtype and out.transpose(1, 2).is_contiguous()
        _within(out, *refs.axial_rope(x, places, sections, (theta,) * n, layout, w), "axial_rope")
    alone = ops.axial_rope(d[0], None, axes, q_weight=d[2], **kw)
    assert alone[1] is None and torch.equal(alone[0], got[0])
    if positions is not None:  # one set of positions for every sequence
        both = ops.axial_rope(d[0], d[1], axes, q_weight=d[2], k_weight=d[3], positions=d[4][0])
        _within(both[0], *refs.axial_rope(q, places[:1].expand(B, T, n), sections, (theta,) * n, layout, wq), "shared")
