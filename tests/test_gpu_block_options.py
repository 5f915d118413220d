"""Options of ops.residual_norm and ops.axial_rope at values that tell them
apart: both eps, each axis' theta and speed. Each case first shows, on the
64-bit definition, that another option's value in their place would be seen."""
import pytest
import torch

import block_refs as refs
from dfsattn_amd import ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _randn(gen, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def _within(got, ref, tol, what):
    off = (got.cpu().double() - ref).abs() - tol
    assert float(off.max()) <= 0, f"{what}: {float(off.max())} past its bound"


def _apart(a, b, what):
    """Two (value, bound) of which a result can be within one alone."""
    assert bool(((a[0] - b[0]).abs() > a[1] + b[1]).any()), f"{what}: the case cannot tell"


@pytest.mark.parametrize("eps,post_eps", [(0.3, 0.02), (0.02, 0.3), (1e-6, 0.5), (0.5, None), (0.25, 0.0)])
@pytest.mark.parametrize("norm,post", [("layer", "rms"), ("rms", "layer"), ("layer", "layer"), ("rms", "rms")])
@pytest.mark.parametrize("rows,C,dtype", [(5, 320, BF), (3, 333, HF), (4, 5120, BF), (2, 5001, BF)])
def test_residual_norm_eps(dev, rows, C, dtype, norm, post, eps, post_eps):
    print(f"residual_norm eps {rows} x {C} {dtype} {norm} post={post} eps={eps} post_eps={post_eps}", flush=True)
    g = torch.Generator().manual_seed(C)
    # both norms see variances near the larger eps
    x, y = _randn(g, rows, C, dtype=dtype, std=0.5), _randn(g, rows, C, dtype=dtype, std=0.4)
    w, pw = 1 + _randn(g, C, std=0.2), 1 + _randn(g, C, std=0.2)
    gate = _randn(g, C, std=0.7)
    behind = eps if post_eps is None else post_eps

    def residual(e):
        return refs.residual(x, y, gate, 0.75, post, pw, None, e)

    r, h = ops.residual_norm(x.to(dev), y.to(dev), gate.to(dev), 0.75, post, pw.to(dev), post_eps=post_eps, norm=norm,
                             weight=w.to(dev), eps=eps)
    for other in [e for e in (eps, 1e-6) if abs(e - behind) > 1e-3]:
        _apart(residual(behind), residual(other), "post_eps")
    for other in [e for e in (behind, 1e-6) if abs(e - eps) > 1e-3]:
        _apart(refs.norm_of(r.cpu(), norm, w, eps=eps), refs.norm_of(r.cpu(), norm, w, eps=other), "eps")
    _within(r, *residual(behind), "r")
    _within(h, *refs.norm_of(r.cpu(), norm, w, eps=eps), "h")


@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("norm", ["head", "all"])
@pytest.mark.parametrize("B,T,H,G,D,dtype,sections,theta,speeds,grid,eps", [
    (1, 9, 4, 2, 64, BF, (24, 20, 20), (1e4, 500.0, 2.0), (0.5, 2.0, -1.0), (2, 3), 2.0),
    (2, 7, 3, 3, 128, HF, (44, 42, 42), (1e6, 1e4, 1e2), (1.0, 0.25, 3.0), None, 1.0),
    (1, 12, 40, 8, 128, BF, (44, 42, 42), (3.0, 1e4, 1e4), (-0.125, 1.0, 0.0), (2, 2), 3.0),
    (1, 6, 2, 1, 32, HF, (8, 8, 8, 8), (1e4, 1e3, 1e2, 1e1), (1.0, -2.0, 0.5, 7.0), (2, 2, 2), 0.5),
    (1, 5, 2, 2, 16, BF, (16,), (50.0,), (0.1,), (), 1e-6),
])
def test_axial_rope_axes_and_eps(dev, B, T, H, G, D, dtype, sections, theta, speeds, grid, eps, norm, layout):
    print(f"axial_rope options {B} x {T} x {H} x {D} {dtype} {layout} {norm} theta={theta} speeds={speeds} eps={eps}",
          flush=True)
    g = torch.Generator().manual_seed(D + T)
    n = len(sections)
    q, k = _randn(g, B, T, H, D, dtype=dtype, std=1.5), _randn(g, B, T, G, D, dtype=dtype, std=1.5)
    wq, wk = (1 + _randn(g, c, std=0.2) for c in ((D, D) if norm == "head" else (H * D, G * D)))
    positions = None
    if grid is None:
        positions = torch.randint(-500, 500, (B, T, n), generator=g).to(torch.int32)
        places = positions
    else:
        places = refs.grid_positions([3] * B, T, grid)
    start = None if grid is None else torch.full((B,), 3, dtype=torch.int32, device=dev)
    axes = ops.RotaryAxes(D, sections, theta, layout, speeds)

    def value(x, w, th=theta, sp=speeds, e=eps):
        return refs.axial_rope(x, places, sections, th, layout, w, e, sp)

    want = value(q, wq)
    if n > 1:
        _apart(want, value(q, wq, th=theta[::-1]), "theta")
        _apart(want, value(q, wq, th=(theta[0],) * n), "theta of the first axis for all")
        _apart(want, value(q, wq, sp=speeds[::-1]), "speeds")
    _apart(want, value(q, wq, sp=(1.0,) * n), "no speeds")
    if eps != 1e-6:
        _apart(want, value(q, wq, e=1e-6), "eps")
    got = ops.axial_rope(q.to(dev), k.to(dev), axes, grid, start, None if positions is None else positions.to(dev),
                         wq.to(dev), wk.to(dev), eps)
    _within(got[0], *want, "q")
    _within(got[1], *value(k, wk), "k")
