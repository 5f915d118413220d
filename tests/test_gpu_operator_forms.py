"""Every kernel of ops.linear and ops.window_attention against the 64-bit
definitions (operator_refs): each form that sizes can choose, in both types,
with every activation and epilogue, between guards; infinities and NaN."""
import math

import pytest
import torch

import operator_cases as cases
import operator_refs as refs
from dfsattn_amd import ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
F = refs.F


def _within(got, ref, tol, what):
    got, ref, tol = got.detach().double().cpu(), ref.cpu(), tol.cpu()
    assert got.shape == ref.shape
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    off = (got - ref).abs() - tol
    worst = int(off.argmax())
    assert float(off.max()) <= 0, (f"{what}: at {worst} got {float(got.flatten()[worst])}, want "
                                   f"{float(ref.flatten()[worst])} within {float(tol.flatten()[worst])}")


def _randn(gen, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=gen, device=gen.device) * std).to(dtype)


# --------------------------------------------------------------------------
# linear
# --------------------------------------------------------------------------

EPILOGUES = [  # bias, activation, gate, residual
    (None, None, False, False),
    ("x", "gelu_tanh", False, True),
    ("x", "gelu", True, True),
    (torch.float32, "silu", True, False),
    (torch.float32, None, True, True),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,n,k,form", cases.LINEAR)
def test_linear_forms(dev, m, n, k, form, dtype):
    """Each form with every activation: values, guards around out, out in place
    of the residual, the same bits twice. The definition in 64 bits on the GPU
    (rows and outputs picked over the result where it is large)."""
    assert cases.linear_form(m, n, k) == form
    gen = torch.Generator(dev).manual_seed(m + n + k)
    x, w = _randn(gen, m, k, dtype=dtype), _randn(gen, n, k, dtype=dtype, std=2 / math.sqrt(k))
    gate, r = torch.randn(n, generator=gen, device=dev), _randn(gen, m, n, dtype=dtype)
    rows, cols = torch.arange(0, m, 1 + m // 700, device=dev), torch.arange(0, n, 1 + n // 700, device=dev)
    rows[-1], cols[-1] = m - 1, n - 1
    for bias, act, with_gate, with_residual in EPILOGUES:
        print(f"linear form {form}: {m} x {n} x {k} {dtype} bias={bias} act={act} gate={with_gate} "
              f"residual={with_residual}", flush=True)
        b = None if bias is None else _randn(gen, n, dtype=dtype if bias == "x" else bias)
        g, res = gate if with_gate else None, r if with_residual else None
        room = torch.full((m * n + 1024,), 7.0, dtype=dtype, device=dev)
        out = room[512:512 + m * n].view(m, n)
        assert ops.linear(x, w, b, act, g, res, out) is out
        assert bool((room[:512] == 7).all()) and bool((room[512 + m * n:] == 7).all())
        ref, tol = refs.linear(x[rows], w[cols], None if b is None else b[cols], act, None if g is None else g[cols],
                               None if res is None else res[rows][:, cols])
        _within(out[rows][:, cols], ref, tol, "linear")
        assert bool(torch.isfinite(out).all())
        if with_residual:  # in its place
            room[512:512 + m * n].view(m, n).copy_(r)
            again = ops.linear(x, w, b, act, g, out, out)
            assert torch.equal(again, ops.linear(x, w, b, act, g, res))
            assert bool((room[:512] == 7).all()) and bool((room[512 + m * n:] == 7).all())
        else:
            assert torch.equal(out, ops.linear(x, w, b, act, g, res))


@pytest.mark.parametrize("m,n,k,form", [c for c in cases.LINEAR if c[1] > 60 and c[2] > 60])
def test_linear_infinities_behind_activations(dev, m, n, k, form):
    """A row with an infinity, whose sums are plus or minus infinity by the
    weights' signs, one with NaN and one of values near the type's largest:
    what the activations' formulas give, in their own rows. (Minus infinity
    times a weight of 0 is NaN in each of the three.)"""
    gen = torch.Generator(dev).manual_seed(n)
    x, w = _randn(gen, m, k, dtype=BF), _randn(gen, n, k, dtype=BF, std=2 / math.sqrt(k))
    w[:, k - 2] = w[:, k - 2].sign() + (w[:, k - 2] == 0)
    if m > 2:
        x[2] = 0
        x[2, k - 2] = 1e30  # z = +-1e30: z^3 is beyond fp32
    if m > 1:
        x[1, 1] = math.nan
    x[0, k - 2] = math.inf
    gate = torch.ones(n, device=dev)
    for act in (None, "gelu_tanh", "gelu", "silu"):
        print(f"linear infinities form {form}: {m} x {n} x {k} {act}", flush=True)
        got = ops.linear(x, w, None, act, gate).double()
        want = refs.activate(math.inf * w[:, k - 2].double(), act)
        assert torch.equal(torch.isnan(got[0]), torch.isnan(want))
        assert torch.equal(got[0].nan_to_num(nan=0), want.nan_to_num(nan=0))
        assert bool((got[0] == math.inf).any())
        if m > 1:
            assert bool(torch.isnan(got[1]).all())
        if m > 2:
            big = refs.activate(x[2, k - 2].double() * w[:, k - 2].double(), act)
            assert torch.equal(got[2], big)
        assert bool(torch.isfinite(got[3:]).all())


# --------------------------------------------------------------------------
# window_attention
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,H,G,L,S,D,left,right,sinks,rolling,form", cases.WINDOW)
def test_window_forms(dev, B, H, G, L, S, D, left, right, sinks, rolling, form, dtype):
    """Each form with and without the lse; sequences of their own lengths (the
    first, some between and the last are compared)."""
    print(f"window form {form}: B={B} H={H} G={G} L={L} S={S} D={D} {dtype} left={left} right={right} sinks={sinks} "
          f"rolling={rolling}", flush=True)
    assert cases.window_form(B, H, G, L, S, D, left, right, sinks, rolling, dtype) == form
    gen = torch.Generator(dev).manual_seed(B * S + L)
    q, k, v = (_randn(gen, B, n, s, D, dtype=dtype) for n, s in ((H, L), (G, S), (G, S)))
    lens = [S + 1000 * b + 77 if rolling else max(S - S * b // (B + 1), 1) for b in range(B)]
    ld = torch.tensor(lens, dtype=torch.int32, device=dev)
    args = dict(left=left, right=right, sinks=sinks, kv_lens=ld, rolling=rolling)
    out, lse = ops.window_attention(q, k, v, **args, want_lse=True)
    assert torch.equal(out, ops.window_attention(q, k, v, **args))
    for b in sorted({0, B // 3, B - 1}):
        one = slice(b, b + 1)
        ref, lse_ref, tol, lse_tol = refs.window_attention(q[one].cpu(), k[one].cpu(), v[one].cpu(), left, right, sinks,
                                                           None, lens[one], rolling)
        _within(out[one], ref, tol, f"out of sequence {b}")
        empty = lse_ref == -math.inf
        assert torch.equal(lse[one].cpu() == -math.inf, empty)
        # operator_refs' bound counts a rounding of the weights to the operands' type, which the lse does not have
        _within(lse[one].cpu().masked_fill(empty, 0), lse_ref.masked_fill(empty, 0),
                lse_tol - 2 * refs.half_step(dtype) * ~empty, f"lse of sequence {b}")


def _dense(q, k, v, seen, scale):
    """Softmax attention in 64 bits over the keys that `seen` [L, S] lets each
    row see, and a bound that counts as operator_refs does."""
    qd, kd, vd = q.double(), k.double(), v.double()
    s = (qd @ kd.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    big = (qd.abs() @ kd.abs().transpose(-1, -2)).masked_fill(~seen, 0).amax(-1, keepdim=True) * scale
    rel = 2 * (refs.half_step(q.dtype) + 2 * (q.shape[-1] + 4) * F * big + (k.shape[2] + 8) * F)
    out = p @ vd
    return out, torch.logsumexp(s, -1), rel * (p @ vd.abs()) + refs.half_step(q.dtype) * (1 + rel) * out.abs() + 2.0 ** -25


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("L", [1, 7, 200])
def test_window_attention_infinite_scores_and_values(dev, L, dtype):
    """A key whose scores are minus infinity has no weight, and a row that sees
    no other counts as seeing none; one whose scores are plus infinity makes its
    rows NaN; values of infinity that every row sees stay in their channel; keys
    and a row's own NaN stay with the rows that see them."""
    print(f"window infinities L={L} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(L)
    D, S, scale = 64, 300, 0.125
    q, k, v = (torch.randn(1, 2, n, D, generator=gen).to(dtype) for n in (L, S, S))
    q[..., 0] = q[..., 0].abs() + 0.5
    dead = S - 1  # the last row's own key
    k[:, :, dead, 0] = -math.inf
    at = torch.arange(S - L, S)[:, None]
    keys = torch.arange(S)[None]

    def run(q, k, v, **kw):
        out, lse = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), **kw, want_lse=True)
        return out.cpu(), lse.cpu()

    clean = k.clone()
    clean[:, :, dead] = 0
    seen = (keys <= at + 5) & (keys != dead)
    ref, lse_ref, tol = _dense(q, clean, v, seen, scale)
    out, lse = run(q, k, v, right=5)
    _within(out, ref, tol, "minus infinity")
    assert float((lse.double() - lse_ref).abs().max()) < 1e-3
    out, lse = run(q, k, v, left=0, right=0)  # rows that see their own key alone
    assert bool((out[:, :, -1] == 0).all()) and bool((lse[:, :, -1] == -math.inf).all())
    assert torch.equal(out[:, :, :-1], v[:, :, S - L:-1])
    up = k.clone()
    up[:, :, dead, 0] = math.inf
    out, _ = run(q, up, v, right=0)
    assert bool(torch.isnan(out[:, :, -1]).all())
    ref, _, tol = _dense(q, clean, v, (keys <= at) & (keys != dead), scale)
    if L > 1:
        _within(out[:, :, :-1], ref[:, :, :-1], tol[:, :, :-1], "rows before plus infinity")
    high = v.clone()
    high[:, :, 40, 9] = math.inf
    out, _ = run(q, clean, high)
    ref, _, tol = _dense(q, clean, v, torch.ones(L, S, dtype=torch.bool), scale)
    others = [c for c in range(D) if c != 9]
    assert bool((out[..., 9] == math.inf).all())
    _within(out[..., others], ref[..., others], tol[..., others], "beside infinite values")
    # hidden from every row, from all but the last, and a query of NaN
    lost = clean.clone()
    lost[:, :, 3], lost[:, :, 50, 7] = math.nan, math.inf
    lost[:, :, dead] = math.nan
    out, _ = run(q, lost, v, left=20, right=0)
    hit = ((keys >= at - 20) & (keys <= at) & ((keys == 3) | (keys == 50) | (keys == dead))).any(-1)
    ref, _, tol = _dense(q, clean, v, (keys >= at - 20) & (keys <= at), scale)
    assert bool(torch.isnan(out[:, :, (at[:, 0] == dead)]).all())
    if bool((~hit).any()):
        _within(out[:, :, ~hit], ref[:, :, ~hit], tol[:, :, ~hit], "keys of NaN that others see")
    if L > 1:
        bad = q.clone()
        bad[:, :, 2] = math.nan
        out, _ = run(bad, clean, v)
        ref, _, tol = _dense(q, clean, v, torch.ones(L, S, dtype=torch.bool), scale)
        rest = [i for i in range(L) if i != 2]
        assert bool(torch.isnan(out[:, :, 2]).all())
        _within(out[:, :, rest], ref[:, :, rest], tol[:, :, rest], "beside a query of NaN")


@pytest.mark.parametrize("L", [1, 200])
def test_window_attention_smallest_scale(dev, L):
    """At 1e-30 every key that a row sees counts the same."""
    gen = torch.Generator().manual_seed(L)
    q, k, v = (torch.randn(1, 2, n, 64, generator=gen).to(BF) for n in (L, 300, 300))
    ref, _, tol, _ = refs.window_attention(q, k, v, 100, 0, 4, scale=1e-30)
    out = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), 100, 0, 4, scale=1e-30)
    _within(out, ref, tol, "smallest scale")


# --------------------------------------------------------------------------
# broadcast inputs, a padded batch, graphs side by side
# --------------------------------------------------------------------------

@pytest.mark.parametrize("m,n,k", [(3, 140, 264), (70, 140, 264), (70, 140, 77), (4185, 1960, 264)])
def test_linear_broadcast_rows(dev, m, n, k):
    """x, weight and residual with one row for all (stride 0): the bits of
    their copies; a residual shared by two batches."""
    gen = torch.Generator(dev).manual_seed(m)
    x, w, r = _randn(gen, m, k, dtype=BF), _randn(gen, n, k, dtype=BF), _randn(gen, m, n, dtype=BF)
    one = [t[:1].expand(t.shape) for t in (x, w, r)]
    for i in range(3):
        a = [x, w, r]
        a[i] = one[i]
        print(f"broadcast {m} x {n} x {k}: operand {i}", flush=True)
        got = ops.linear(a[0], a[1], residual=a[2], activation="silu")
        a[i] = one[i].contiguous()
        assert torch.equal(got, ops.linear(a[0], a[1], residual=a[2], activation="silu"))
    both = ops.linear(torch.stack([x, x]), w, residual=r.expand(2, m, n))
    alone = ops.linear(torch.stack([x, x]), w, residual=torch.stack([r, r]))
    assert torch.equal(both, alone) and torch.equal(both[0], both[1])


@pytest.mark.parametrize("L", [1, 90])
def test_window_attention_broadcast_axes(dev, L):
    """Batches, heads and rows that are one in memory: the bits of their copies."""
    gen = torch.Generator(dev).manual_seed(L)
    base = {n: _randn(gen, 3, h, s, 64, dtype=BF) for n, h, s in (("q", 4, L), ("k", 2, 200), ("v", 2, 200))}
    lens = torch.tensor([200, 31, 130], dtype=torch.int32, device=dev)
    for name, t in base.items():
        for view in (t[:1].expand(t.shape), t[:, :1].expand(t.shape), t[:, :, :1].expand(t.shape)):
            print(f"broadcast L={L} {name} {view.stride()}", flush=True)
            args = {**base, name: view}
            got = ops.window_attention(**args, left=50, right=0, sinks=2, kv_lens=lens)
            args[name] = view.contiguous()
            assert torch.equal(got, ops.window_attention(**args, left=50, right=0, sinks=2, kv_lens=lens))


def test_padded_chunks_equal_each_sequence_alone(dev):
    """Chunks of three lengths in one padded batch, appended to rolling caches
    and attended with q_lens, against each sequence by itself; what lies behind
    a sequence's tokens is 0 in out, its slots stay."""
    gen = torch.Generator(dev).manual_seed(9)
    B, T, H, G, D, left, sinks = 3, 40, 4, 2, 64, 60, 5
    S, new, lens = sinks + left + T, [40, 7, 0], [500, 3, 90]
    q, k, v = (_randn(gen, B, T, n, D, dtype=BF) for n in (H, G, G))
    caches = [_randn(gen, B, G, S, D, dtype=BF) for _ in range(2)]
    before = [c.clone() for c in caches]
    w = torch.rand(D, device=dev, generator=gen) + 0.5
    ang = torch.rand(600, D // 2, device=dev, generator=gen)
    table = (torch.cos(ang), torch.sin(ang))

    def run(q, k, v, caches, lens, new):
        ld, nd = (torch.tensor(t, dtype=torch.int32, device=dev) for t in (lens, new))
        a = ops.qkv_cache(q, k, v, *caches, ld, w, w, table=table, new_lens=nd, sinks=sinks, rolling=True)
        return ops.window_attention(a, *caches, left, 0, sinks, q_lens=nd, kv_lens=ld + nd, rolling=True, want_lse=True)

    out, lse = run(q, k, v, caches, lens, new)
    for b in range(B):
        n = new[b]
        assert bool((out[b, :, n:] == 0).all()) and bool((lse[b, :, n:] == -math.inf).all())
        if n == 0:
            assert torch.equal(caches[0][b], before[0][b]) and torch.equal(caches[1][b], before[1][b])
            continue
        own = [c[b:b + 1].clone() for c in before]
        alone, alone_lse = run(*(t[b:b + 1, :n] for t in (q, k, v)), own, lens[b:b + 1], [n])
        assert torch.equal(own[0][0], caches[0][b]) and torch.equal(own[1][0], caches[1][b])
        # another number of rows may take other tiles, so sums in another order
        ref, _, tol, _ = refs.window_attention(
            ops.qkv_cache(*(t[b:b + 1, :n] for t in (q, k, v)), *[c.clone() for c in own],
                          torch.tensor(lens[b:b + 1], dtype=torch.int32, device=dev), w, w, table=table, sinks=sinks,
                          rolling=True).cpu(), own[0].cpu(), own[1].cpu(), left, 0, sinks, None, [lens[b] + n], True)
        _within(out[b:b + 1, :, :n], ref, tol, f"padded sequence {b}")
        _within(alone, ref, tol, f"sequence {b} alone")


def test_two_graphs_with_workspaces_of_their_own(dev):
    """Two captured calls that cut their work into parts, replayed in turn and
    on two streams at once: each has its own workspace."""
    gen = torch.Generator(dev).manual_seed(10)
    jobs = []
    for _ in range(2):
        x, w = _randn(gen, 64, 4096, dtype=BF), _randn(gen, 640, 4096, dtype=BF, std=0.02)
        q, k, v = (_randn(gen, 1, 2, n, 128, dtype=BF) for n in (130, 2600, 2600))
        jobs.append((x, w, q, k, v))
    assert cases.linear_form(64, 640, 4096) & cases.PARTS

    def run(j):
        return (ops.linear(j[0], j[1], activation="silu"), *ops.window_attention(*j[2:], right=0, want_lse=True))

    for j in jobs:
        run(j)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for j in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(j))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in jobs]
    for i in range(4):
        for j in jobs:
            j[0].normal_(generator=gen)
            j[2].normal_(generator=gen)
        want = [run(j) for j in jobs]
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
