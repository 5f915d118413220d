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


def test_residual_norm_rows_that_are_not_finite(dev):
    """A NaN or infinity in a row stays in it; rows of one value, whose layer
    norm is that of zeros; a channel count of every remainder by eight."""
    for C in (64, 65, 71, 2500, 2503):
        print(f"residual_norm not finite C={C}", flush=True)
        g = torch.Generator().manual_seed(C)
        x, y = _randn(g, 9, C, dtype=BF).to(dev), _randn(g, 9, C, dtype=BF).to(dev)
        whole = ops.residual_norm(x, y, norm="layer")
        x[2, C - 1], y[5, 0] = math.inf, math.nan
        got = ops.residual_norm(x, y, norm="layer")
        keep = [0, 1, 3, 4, 6, 7, 8]
        for a, b in zip(got, whole):
            assert torch.equal(a[keep], b[keep])
        assert bool(torch.isnan(got[1][[2, 5]]).all())
        r, codes, scales = ops.residual_norm(x, y, norm="layer", quantize=True)
        assert bool(torch.isnan(codes[[2, 5]].float()).all())
        flat = torch.full((3, C), 2.0, dtype=BF, device=dev)
        assert bool((ops.residual_norm(flat, flat)[1] == 0).all())


def test_residual_norm_views(dev):
    """Rows inside wider ones at any element, vectors cut from one tensor or
    expanded, what surrounds out stays, no rows."""
    g = torch.Generator().manual_seed(4)
    for C, off in ((512, 8), (512, 3), (77, 1)):
        print(f"residual_norm views C={C} offset={off}", flush=True)
        x, y = _randn(g, 2, 5, C + 16, dtype=BF), _randn(g, 2, 5, C + 16, dtype=BF)
        both = _randn(g, 2, 3, C)
        xs, ys = x.to(dev)[..., off:off + C], y.to(dev)[..., off:off + C]
        gate, scale, shift = both.to(dev).chunk(3, 1)
        room = torch.full((10 * C + 512,), 7.0, dtype=BF, device=dev)
        out = room[256:256 + 10 * C].view(2, 5, C)
        r, h = ops.residual_norm(xs, ys, gate, scale=scale, shift=shift, out=out)
        assert r is out and bool((room[:256] == 7).all()) and bool((room[256 + 10 * C:] == 7).all())
        want = ops.residual_norm(xs.contiguous(), ys.contiguous(), gate.contiguous(), scale=scale.contiguous(),
                                 shift=shift.contiguous())
        assert torch.equal(r, want[0]) and torch.equal(h, want[1])
        _within(r, *refs.residual(x[..., off:off + C], y[..., off:off + C], both[:, :1]), "r")
        one = ops.residual_norm(xs, ys, gate[:1].expand(2, 1, C))
        assert torch.equal(one[0][0], want[0][0])
        t = ops.residual_norm(xs.transpose(0, 1), ys.transpose(0, 1), gate.transpose(0, 1))
        assert torch.equal(t[0].transpose(0, 1), want[0])
    empty = ops.residual_norm(torch.zeros(0, 64, dtype=BF, device=dev), torch.zeros(0, 64, dtype=BF, device=dev), quantize=True)
    assert [tuple(e.shape) for e in empty] == [(0, 64), (0, 64), (0, 1)]


def test_axial_rope_views_and_far_positions(dev):
    """Heads inside wider rows on and off 16-byte boundaries, head-major storage;
    positions at the ends of int32."""
    g = torch.Generator().manual_seed(6)
    axes = ops.RotaryAxes(64, (24, 20, 20), 1e4)
    x = _randn(g, 2, 7, 3, 80, dtype=BF)
    places = torch.tensor([[[2 ** 31 - 1 - i, -2 ** 31 + i, 12345 * i] for i in range(7)]] * 2)
    pos = places.to(torch.int32).to(dev)
    for off in (0, 8, 3):
        print(f"axial_rope views offset={off}", flush=True)
        xd = x.to(dev)[..., off:off + 64]
        got = ops.axial_rope(xd, xd, axes, positions=pos)
        _within(got[0], *refs.axial_rope(x[..., off:off + 64], places, (24, 20, 20), (1e4,) * 3, "pairs"), "far")
        assert torch.equal(got[0], got[1])
        major = xd.transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(ops.axial_rope(major, None, axes, positions=pos)[0], got[0])
        wide = torch.zeros(2, 7, 9, dtype=torch.int32, device=dev)
        wide[..., 4:7] = pos
        assert torch.equal(ops.axial_rope(xd, None, axes, positions=wide[..., 4:7])[0], got[0])
    assert ops.axial_rope(xd[:, :0], xd[:, :0], axes, grid=(2, 2))[0].shape == (2, 3, 0, 64)


def test_block_operators_beyond_32_bits(dev):
    rows = 430000
    print("residual_norm 430,000 x 5,120", flush=True)
    g = torch.Generator().manual_seed(8)
    x, y = torch.zeros(rows, 5120, dtype=BF, device=dev), torch.zeros(rows, 5120, dtype=BF, device=dev)
    x[-2:], y[-2:] = _randn(g, 2, 5120, dtype=BF).to(dev), _randn(g, 2, 5120, dtype=BF).to(dev)
    gate = _randn(g, 5120).to(dev)
    for q in (False, True):
        got, want = ops.residual_norm(x, y, gate, quantize=q), ops.residual_norm(x[-2:], y[-2:], gate, quantize=q)
        for a, b in zip(got, want):
            assert torch.equal(a[-2:].view(torch.uint8), b.view(torch.uint8))
    del got, y
    print("axial_rope 430,000 x 40 x 128", flush=True)
    axes = ops.RotaryAxes(128, (44, 42, 42))
    got = ops.axial_rope(x.view(1, rows, 40, 128), None, axes, grid=(45, 80))[0]
    start = torch.tensor([rows - 2], dtype=torch.int32, device=dev)
    want = ops.axial_rope(x[-2:].view(1, 2, 40, 128), None, axes, grid=(45, 80), start=start)[0]
    assert torch.equal(got[:, :, -2:], want)


def _calls(dev, seed):
    """A run of the operators as a block uses them, on inputs of its own."""
    g = torch.Generator().manual_seed(seed)
    rows, C, F = 300, 640, 1100
    x, y = _randn(g, rows, C, dtype=BF).to(dev), _randn(g, rows, C, dtype=BF).to(dev)
    gate, scale, shift = (_randn(g, C).to(dev) for _ in range(3))
    w1, w2 = (ops.quantize_fp8(_randn(g, *s, dtype=BF, std=0.05).to(dev)) for s in ((F, C), (C, F)))
    b1, b2 = _randn(g, F, dtype=BF).to(dev), _randn(g, C, dtype=BF).to(dev)
    axes = ops.RotaryAxes(128, (44, 42, 42))
    start = torch.tensor([7], dtype=torch.int32, device=dev)

    def run():
        r, codes, scales = ops.residual_norm(x, y, gate, scale=scale, shift=shift, quantize=True)
        codes, scales = ops.linear_fp8(codes, *w1, scales, bias=b1, activation="gelu_tanh", quantize=True, out_dtype=BF)
        o = ops.linear_fp8(codes, *w2, scales, bias=b2, gate=gate, residual=r)
        p = ops.linear_fp8(o, *w1)
        q, k = ops.axial_rope(o.view(1, rows, 5, 128), r.view(1, rows, 5, 128), axes, grid=(5, 6), start=start)
        return r, codes.view(torch.uint8), scales.view(torch.uint8), o, p, q, k

    return run, x, start


def test_block_operators_on_another_stream_and_in_threads(dev):
    import threading

    runs = [_calls(dev, seed)[0] for seed in (1, 2)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = runs[0]()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                if not all(torch.equal(a, b) for a, b in zip(runs[i](), want[i])):
                    bad.append(i)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_block_operators_in_graphs(dev):
    """Two captured runs, replayed by turns and at once with new inputs between."""
    made = [_calls(dev, seed) for seed in (3, 4)]
    graphs, outs = [], []
    for run, _, _ in made:
        run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(4):
        for i, (run, x, start) in enumerate(made):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * turn + i)).to(BF))
            start.fill_(1000 * turn + i)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (run, _, _), got in zip(made, outs):
            assert all(torch.equal(a, b) for a, b in zip(got, run()))
