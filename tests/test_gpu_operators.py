"""GPU parity of ops.linear, ops.window_attention and ops.qkv_cache against
their 64-bit definitions (operator_refs), within the bounds that their
roundings allow."""
import math
import threading

import pytest
import torch

import operator_refs as refs
from dfsattn_amd import _lib, ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _randn(gen, *shape, dtype, std=1.0):
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
# linear
# --------------------------------------------------------------------------

LINEAR = [
    # M, N, K, dtype, bias dtype, act, gate, residual
    (1, 64, 64, BF, BF, None, False, False),
    (1, 1, 1, BF, None, None, False, True),
    (1, 2048, 1024, BF, torch.float32, "silu", False, False),
    (3, 257, 2500, HF, HF, "gelu_tanh", True, True),
    (2, 200, 8200, BF, BF, None, False, False),
    (16, 640, 256, BF, BF, "gelu", False, True),
    (17, 96, 2048, HF, None, None, True, False),
    (33, 1000, 1032, BF, BF, "gelu_tanh", False, False),
    (64, 520, 4096, BF, None, None, False, True),
    (65, 129, 63, BF, BF, "silu", True, True),
    (100, 128, 65, HF, torch.float32, None, False, False),
    (127, 255, 511, HF, HF, "gelu", True, True),
    (128, 128, 128, BF, BF, None, False, False),
    (200, 384, 640, BF, BF, "gelu_tanh", True, True),
    (256, 256, 64, BF, None, None, False, False),
    (257, 513, 72, HF, HF, None, False, True),
    (300, 1025, 1000, BF, BF, "silu", False, False),
    (513, 1024, 1024, BF, BF, "gelu_tanh", False, True),
    (1000, 776, 136, HF, None, None, True, True),
    (2100, 2056, 192, BF, BF, None, True, True),
    (2049, 2304, 328, HF, HF, "gelu_tanh", False, False),
    (4099, 1100, 70, BF, torch.float32, "gelu_tanh", False, True),
]


@pytest.mark.parametrize("m,n,k,dtype,bias,act,gate,residual", LINEAR)
def test_linear_matches_definition(dev, m, n, k, dtype, bias, act, gate, residual):
    print(f"linear {m} x {n} x {k} {dtype} bias={bias} act={act} gate={gate} residual={residual}", flush=True)
    g = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    x, w = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype, std=2 / math.sqrt(k))
    b = None if bias is None else _randn(g, n, dtype=bias)
    gt = torch.randn(n, generator=g) if gate else None
    r = _randn(g, m, n, dtype=dtype) if residual else None
    ref, tol = refs.linear(x, w, b, act, gt, r)
    d = [None if t is None else t.to(dev) for t in (x, w, b, gt, r)]
    got = ops.linear(d[0], d[1], d[2], activation=act, gate=d[3], residual=d[4])
    assert got.dtype == dtype
    _within(got, ref, tol, "linear")
    again = ops.linear(d[0], d[1], d[2], activation=act, gate=d[3], residual=d[4])
    assert torch.equal(got, again)
    if residual:  # in place of the residual
        d[4] = ops.linear(d[0], d[1], d[2], activation=act, gate=d[3], residual=d[4], out=d[4])
        assert torch.equal(got, d[4])


@pytest.mark.parametrize("m,n,k,act", [(4200, 4200, 3000, "gelu_tanh"), (2560, 6500, 4104, None)])
def test_linear_last_tiles_in_parts(dev, m, n, k, act):
    """More large tiles than compute units: those behind the last full round
    are cut along k. Rows and outputs picked all over the result."""
    print(f"linear {m} x {n} x {k} {act}", flush=True)
    assert _lib.lib().dfs_linear_workspace_size(m, n, k, 1) > 0
    gen = torch.Generator().manual_seed(m + n + k)
    x, w = _randn(gen, m, k, dtype=BF), _randn(gen, n, k, dtype=BF, std=2 / math.sqrt(k))
    b, gate, r = _randn(gen, n, dtype=BF), torch.randn(n, generator=gen), _randn(gen, m, n, dtype=BF)
    d = [t.to(dev) for t in (x, w, b, gate, r)]
    got = ops.linear(d[0], d[1], d[2], activation=act, gate=d[3], residual=d[4])
    assert torch.equal(got, ops.linear(d[0], d[1], d[2], activation=act, gate=d[3], residual=d[4]))
    rows, cols = torch.arange(0, m, 13), torch.arange(0, n, 11)
    rows[-1], cols[-1] = m - 1, n - 1
    ref, tol = refs.linear(x[rows], w[cols], b[cols], act, gate[cols], r[rows][:, cols])
    _within(got.cpu()[rows][:, cols], ref, tol, "parts")


@pytest.mark.parametrize("m", [1, 5, 40, 130, 700])
def test_linear_strided_rows_and_batches(dev, m):
    """x inside wider rows (channels 8 and 3 in), weight inside wider rows, a
    batch axis, a residual that is a transposed view."""
    g = torch.Generator().manual_seed(m)
    k, n = 264, 136
    wide = _randn(g, 2, m, k + 24, dtype=BF)
    ww = _randn(g, n, k + 16, dtype=BF, std=0.1)
    r = _randn(g, n, 2, m, dtype=BF)
    wide_d, ww_d, r_d = wide.to(dev), ww.to(dev), r.to(dev).permute(1, 2, 0)
    for off in (8, 3):
        print(f"linear strided m={m} offset={off}", flush=True)
        x = wide[:, :, off:off + k]
        ref, tol = refs.linear(x.reshape(-1, k), ww[:, 8:8 + k], None, None, None,
                               r.permute(1, 2, 0).reshape(-1, n))
        got = ops.linear(wide_d[:, :, off:off + k], ww_d[:, 8:8 + k], residual=r_d)
        assert got.shape == (2, m, n)
        _within(got.reshape(-1, n), ref, tol, "linear strided")


def test_linear_leaves_what_surrounds_out(dev):
    """Every tile form's stores end at out's last row and column."""
    for m, n, k, dtype in ((1, 72, 64, BF), (20, 40, 64, BF), (130, 264, 72, HF), (2100, 2056, 64, BF),
                           (300, 77, 65, BF)):
        print(f"linear guard {m} x {n} x {k}", flush=True)
        g = torch.Generator().manual_seed(n)
        x, w = _randn(g, m, k, dtype=dtype).to(dev), _randn(g, n, k, dtype=dtype).to(dev)
        room = torch.full((m * n + 1024,), 7.0, dtype=dtype, device=dev)
        out = room[512:512 + m * n].view(m, n)
        ops.linear(x, w, out=out)
        assert bool((room[:512] == 7).all()) and bool((room[512 + m * n:] == 7).all())
        assert torch.equal(out, ops.linear(x, w))


def test_linear_infinities_and_nan_stay_in_their_rows(dev):
    for m, n, k in ((4, 128, 512), (300, 300, 136), (2048, 2304, 128)):
        print(f"linear inf {m} x {n} x {k}", flush=True)
        g = torch.Generator().manual_seed(m)
        x, w = _randn(g, m, k, dtype=BF), _randn(g, n, k, dtype=BF)
        x[1, 3], x[2, k - 1] = math.inf, math.nan
        got = ops.linear(x.to(dev), w.to(dev)).cpu()
        ref = (x.double() @ w.double().t())
        keep = [i for i in range(m) if i not in (1, 2)]
        assert bool(torch.isnan(got[2]).all())
        assert torch.equal(got[1].double(), ref[1])  # plus or minus infinity by the weight's sign
        assert bool(torch.isfinite(got[keep]).all())


def test_linear_empty_batch(dev):
    w = torch.zeros(8, 16, dtype=BF, device=dev)
    assert ops.linear(torch.zeros(0, 16, dtype=BF, device=dev), w).shape == (0, 8)


# --------------------------------------------------------------------------
# window_attention
# --------------------------------------------------------------------------

ATTENTION = [
    # B, H, G, L, S, D, dtype, left, right, sinks, q_lens, kv_lens, rolling
    (1, 2, 2, 1, 1, 128, BF, None, 0, 0, None, None, False),
    (1, 2, 1, 1, 300, 64, HF, None, 0, 0, None, None, False),
    (2, 8, 2, 1, 700, 128, BF, 100, 0, 5, None, [700, 33], False),
    (3, 4, 4, 1, 257, 128, HF, 64, 0, 0, None, [1, 0, 200], False),
    (2, 20, 4, 1, 130, 64, BF, 97, 0, 4, None, [1000, 57], True),
    (1, 16, 1, 1, 515, 128, BF, 500, 0, 10, None, [2000], True),
    (2, 6, 2, 3, 140, 64, HF, 50, 0, 3, None, [140, 2], False),
    (1, 12, 3, 7, 400, 128, BF, 130, 2, 130, None, None, False),
    (1, 4, 2, 17, 17, 64, BF, None, 0, 0, None, None, False),
    (2, 4, 1, 40, 40, 128, HF, 9, 0, 2, [40, 13], [40, 13], False),
    (1, 2, 2, 129, 129, 128, BF, 20, 20, 30, None, None, False),
    (1, 3, 1, 200, 200, 64, HF, 70, 0, 4, None, None, False),
    (1, 2, 1, 130, 77, 128, BF, None, None, 0, None, [50], False),
    (1, 2, 2, 150, 77, 128, HF, None, 0, 0, None, None, False),  # the first rows stand before the first key
    (1, 2, 1, 100, 420, 128, BF, 200, None, 60, None, [777], True),
    (2, 2, 2, 90, 310, 64, HF, 150, 0, 64, [90, 31], [1234, 200], True),
    (1, 1, 1, 64, 500, 128, BF, 0, 0, 0, None, None, False),
    (1, 1, 1, 140, 300, 128, BF, 0, 0, 200, None, None, False),
    (2, 2, 1, 33, 90, 128, BF, 40, 3, 7, [0, 33], [90, 0], False),
    (1, 5, 5, 260, 260, 64, BF, 128, 128, 128, None, None, False),
    # keys cut into parts: many for one sequence, with rows that see few or none of them
    (1, 4, 1, 2, 5003, 128, BF, None, 0, 0, None, None, False),
    (2, 3, 1, 1, 4100, 64, HF, None, 0, 0, None, [4100, 130], False),
    (2, 8, 1, 40, 3000, 128, BF, None, 0, 0, [40, 3], [3000, 5], False),
    (1, 2, 2, 70, 2600, 64, HF, 2400, None, 100, None, [9000], True),
    # heads for every eighth of the chip, a few rows in their last blocks
    (1, 8, 8, 150, 900, 128, BF, 500, None, 64, None, [2000], True),
    (2, 8, 4, 140, 140, 64, HF, 100, 0, 4, [140, 77], [140, 77], False),
]


@pytest.mark.parametrize("B,H,G,L,S,D,dtype,left,right,sinks,q_lens,kv_lens,rolling", ATTENTION)
def test_window_attention_matches_definition(dev, B, H, G, L, S, D, dtype, left, right, sinks, q_lens, kv_lens,
                                             rolling):
    print(f"window B={B} H={H} G={G} L={L} S={S} D={D} {dtype} left={left} right={right} sinks={sinks} "
          f"q={q_lens} kv={kv_lens} rolling={rolling}", flush=True)
    g = torch.Generator().manual_seed(L * S + H)
    q = _randn(g, B, L, H, D, dtype=dtype).transpose(1, 2)
    k, v = _randn(g, B, G, S, D, dtype=dtype), _randn(g, B, G, S, D, dtype=dtype)
    ref, lse_ref, tol, lse_tol = refs.window_attention(q, k, v, left, right, sinks, q_lens, kv_lens, rolling)
    if kv_lens is not None and not rolling:  # keys behind a sequence may hold anything
        for b, n in enumerate(kv_lens):
            k[b, :, n:], v[b, :, n:] = math.nan, math.inf
    lens = [None if t is None else torch.tensor(t, dtype=torch.int32, device=dev) for t in (q_lens, kv_lens)]
    qd, kd, vd = q.to(dev), k.to(dev), v.to(dev)
    out, lse = ops.window_attention(qd, kd, vd, left, right, sinks, *lens, rolling=rolling, want_lse=True)
    assert out.dtype == dtype and out.stride() == qd.stride()
    _within(out, ref, tol, "window out")
    lse = lse.cpu().double()
    empty = lse_ref == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool((out.cpu()[empty] == 0).all())
    _within(lse.masked_fill(empty, 0), lse_ref.masked_fill(empty, 0), lse_tol, "window lse")
    for _ in range(2):
        assert torch.equal(out, ops.window_attention(qd, kd, vd, left, right, sinks, *lens, rolling=rolling))


@pytest.mark.parametrize("L,S", [(1, 400), (6, 200), (150, 150)])
def test_window_attention_strides_scale_and_out(dev, L, S):
    """Token-major keys of a joint projection, another scale, out between
    guards, unaligned rows (copied)."""
    print(f"window strides L={L} S={S}", flush=True)
    g = torch.Generator().manual_seed(L)
    H, G, D = 4, 2, 64
    q = _randn(g, 2, L, H, D, dtype=BF).transpose(1, 2)
    kv = _randn(g, 2, S, 2, G, D, dtype=BF)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    ref, _, tol, _ = refs.window_attention(q, k, v, 90, 0, 3, scale=0.3)
    kvd, qd = kv.to(dev), q.to(dev)
    room = torch.full((2, H, L + 2, D), 5.0, dtype=BF, device=dev)
    out = ops.window_attention(qd, kvd[:, :, 0].transpose(1, 2), kvd[:, :, 1].transpose(1, 2), 90, 0, 3, scale=0.3,
                               out=room[:, :, 1:-1])
    _within(out, ref, tol, "window strided")
    assert bool((room[:, :, 0] == 5).all()) and bool((room[:, :, -1] == 5).all())
    odd = torch.empty(2, H, L, D + 2, dtype=BF, device=dev)[..., :D]
    odd.copy_(qd)
    assert torch.equal(out, ops.window_attention(odd, k.to(dev), v.to(dev), 90, 0, 3, scale=0.3))


@pytest.mark.parametrize("L", [1, 200])
def test_window_attention_large_scores_and_infinities(dev, L):
    """Scores far beyond the exponent's range, a key of minus infinite scores
    and one of plus infinite values that only some rows see."""
    print(f"window extremes L={L}", flush=True)
    g = torch.Generator().manual_seed(3)
    q, k, v = (_randn(g, 1, 2, n, 128, dtype=BF) for n in (L, 300, 300))
    q, k = q * 30, k * 30
    ref, _, tol, _ = refs.window_attention(q, k, v, 100, 0, 4)
    out = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), 100, 0, 4)
    _within(out, ref, tol, "large scores")


def test_window_attention_empty_sizes(dev):
    q = torch.ones(1, 2, 3, 64, dtype=BF, device=dev)
    k = torch.ones(1, 2, 0, 64, dtype=BF, device=dev)
    out, lse = ops.window_attention(q, k, k, want_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    assert ops.window_attention(q[:, :, :0], q, q).shape == (1, 2, 0, 64)


# --------------------------------------------------------------------------
# qkv_cache
# --------------------------------------------------------------------------

CACHE = [
    # B, T, H, G, D, S, dtype, norm ("head", "all", None), weight dtype, rotation, sinks, rolling, lens, new_lens
    (1, 1, 2, 2, 128, 4, BF, "head", BF, True, 0, False, [3], None),
    (3, 1, 8, 2, 64, 40, HF, "head", torch.float32, True, 0, False, [0, 39, 7], None),
    (2, 5, 6, 3, 128, 16, BF, "all", BF, True, 4, True, [50, 0], None),
    (2, 9, 4, 1, 64, 30, HF, "all", HF, False, 0, False, [2, 5], [9, 4]),
    (1, 13, 40, 40, 128, 64, BF, "all", BF, True, 16, True, [40], None),
    (2, 3, 1, 1, 32, 8, BF, None, None, True, 2, True, [7, 1], [0, 3]),
    (1, 7, 3, 3, 256, 9, HF, "head", BF, True, 0, False, [2], None),
    (1, 4, 16, 2, 512, 6, BF, "head", HF, False, 0, False, [1], [3]),
    (2, 2, 12, 4, 16, 5, BF, None, None, False, 0, False, [3, 2], None),
]


def _cache_inputs(B, T, H, G, D, S, dtype, norm, wdt, rotate, lens):
    g = torch.Generator().manual_seed(B * T + H * D)
    x = [_randn(g, B, T, n, D, dtype=dtype, std=3) for n in (H, G, G)]
    caches = [_randn(g, B, G, S, D, dtype=dtype) for _ in range(2)]
    w = [None if norm is None else (torch.rand(D if norm == "head" else n * D, generator=g) + 0.5).to(wdt)
         for n in (H, G)]
    ang = torch.rand(max(lens) + T, D // 2, generator=g, dtype=torch.float64) * 50
    table = (torch.cos(ang).float(), torch.sin(ang).float()) if rotate else None
    return x, caches, w, table


@pytest.mark.parametrize("B,T,H,G,D,S,dtype,norm,wdt,rotate,sinks,rolling,lens,new_lens", CACHE)
def test_qkv_cache_matches_definition(dev, B, T, H, G, D, S, dtype, norm, wdt, rotate, sinks, rolling, lens, new_lens):
    print(f"qkv_cache B={B} T={T} H={H} G={G} D={D} S={S} {dtype} norm={norm} rolling={rolling}", flush=True)
    x, caches, w, table = _cache_inputs(B, T, H, G, D, S, dtype, norm, wdt, rotate, lens)
    ref = refs.qkv_cache(*x, *caches, lens, *w, table=table, new_lens=new_lens, sinks=sinks, rolling=rolling)
    xd, cd = [t.to(dev) for t in x], [t.to(dev) for t in caches]
    wd = [None if t is None else t.to(dev) for t in w]
    td = None if table is None else tuple(t.to(dev) for t in table)
    ld = torch.tensor(lens, dtype=torch.int32, device=dev)
    nd = None if new_lens is None else torch.tensor(new_lens, dtype=torch.int32, device=dev)
    q = ops.qkv_cache(*xd, *cd, ld, *wd, table=td, new_lens=nd, sinks=sinks, rolling=rolling)
    assert q.shape == (B, H, T, D) and q.dtype == dtype
    _within(q, ref[0], ref[3], "q")
    _within(cd[0], ref[1], ref[4], "k_cache")
    assert torch.equal(cd[1].cpu().double(), ref[2])
    assert ld.tolist() == lens


def test_qkv_cache_views_and_ends(dev):
    """A joint projection's slices, caches whose rows alternate in one tensor;
    tokens past the last slot are dropped, positions past the table NaN."""
    g = torch.Generator().manual_seed(1)
    B, T, H, G, D, S = 2, 3, 4, 2, 64, 8
    qkv = _randn(g, B, T, H + 2 * G, D, dtype=BF)
    kv = torch.full((B, G, S + 1, 2, D), 9.0, dtype=BF)
    lens = [6, 2]
    ang = torch.rand(8, D // 2, generator=g, dtype=torch.float64)
    table = (torch.cos(ang).float(), torch.sin(ang).float())
    d, kvd = qkv.to(dev), kv.to(dev)
    q = ops.qkv_cache(d[:, :, :H], d[:, :, H:H + G], d[:, :, H + G:], kvd[:, :, :S, 0], kvd[:, :, :S, 1],
                      torch.tensor(lens, dtype=torch.int32, device=dev), table=tuple(t.to(dev) for t in table)).cpu()
    got = kvd.cpu()
    assert bool(torch.isnan(q[0, :, 2].float()).all())  # position 8 of 8
    assert bool((got[:, :, S] == 9).all())  # nothing behind the last slot
    wide = tuple(torch.cat([t, t[:1]]) for t in table)
    ref = refs.qkv_cache(qkv[:, :, :H], qkv[:, :, H:H + G], qkv[:, :, H + G:], kv[:, :, :S, 0], kv[:, :, :S, 1], lens,
                         table=wide)
    _within(q[:, :, :2], ref[0][:, :, :2], ref[3][:, :, :2], "q")
    _within(got[:, :, :S, 0], ref[1], ref[4], "k_cache")
    assert torch.equal(got[:, :, :S, 1].double(), ref[2])


# --------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------

def test_operators_on_another_stream(dev):
    g = torch.Generator().manual_seed(5)
    x, w = _randn(g, 300, 256, dtype=BF).to(dev), _randn(g, 512, 256, dtype=BF).to(dev)
    k = _randn(g, 1, 4, 300, 128, dtype=BF).to(dev)
    want = ops.linear(x, w)
    att = ops.window_attention(want.view(1, 300, 4, 128).transpose(1, 2), k, k, left=50, right=0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear(x, w)
        att2 = ops.window_attention(got.view(1, 300, 4, 128).transpose(1, 2), k, k, left=50, right=0)
    side.synchronize()
    assert torch.equal(want, got) and torch.equal(att, att2)


def test_operators_from_two_threads(dev):
    """Two threads on streams of their own, products in parts (a workspace each)
    and attention over a cut cache: each gets what it gets alone."""
    gen = torch.Generator().manual_seed(7)
    jobs = []
    for _ in range(2):
        x, w = _randn(gen, 64, 4096, dtype=BF).to(dev), _randn(gen, 640, 4096, dtype=BF, std=0.02).to(dev)
        q = _randn(gen, 2, 8, 1, 64, dtype=BF).to(dev)
        k, v = (_randn(gen, 2, 2, 3000, 64, dtype=BF).to(dev) for _ in range(2))
        jobs.append((x, w, q, k, v))
    assert _lib.lib().dfs_linear_workspace_size(64, 640, 4096, 1) > 0

    def run(job):
        return ops.linear(job[0], job[1], activation="silu"), ops.window_attention(*job[2:], right=0)

    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[i] = [run(jobs[i]) for _ in range(20)]
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        for y, o in got[i]:
            assert torch.equal(y, want[i][0]) and torch.equal(o, want[i][1])


def test_operators_in_a_graph(dev):
    """A layer's token over its cache (products, append, attention) captured
    once and replayed with other inputs, each replay against the eager run."""
    g = torch.Generator().manual_seed(6)
    B, H, G, D, S, C = 3, 8, 2, 64, 600, 512
    w_qkv = _randn(g, (H + 2 * G) * D, C, dtype=BF, std=0.05).to(dev)
    w_out = _randn(g, C, H * D, dtype=BF, std=0.05).to(dev)
    w_up, w_down = (_randn(g, *s, dtype=BF, std=0.05).to(dev) for s in ((1100, C), (C, 1100)))
    norm = torch.ones(D, dtype=BF, device=dev)
    ang = torch.rand(900, D // 2, generator=g)
    table = (torch.cos(ang).to(dev), torch.sin(ang).to(dev))
    x = torch.zeros(B, 1, C, dtype=BF, device=dev)
    lens = torch.zeros(B, dtype=torch.int32, device=dev)
    kc, vc = (torch.zeros(B, G, S, D, dtype=BF, device=dev) for _ in range(2))

    def layer():
        qkv = ops.linear(x, w_qkv).view(B, 1, H + 2 * G, D)
        q = ops.qkv_cache(qkv[:, :, :H], qkv[:, :, H:H + G], qkv[:, :, H + G:], kc, vc, lens, norm, norm, table=table,
                          sinks=4, rolling=True)
        o = ops.window_attention(q, kc, vc, left=500, right=0, sinks=4, kv_lens=lens + 1, rolling=True)
        y = ops.linear(o.transpose(1, 2).reshape(B, 1, H * D), w_out, residual=x)
        return ops.linear(ops.linear(y, w_up, activation="gelu_tanh"), w_down, residual=y)

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for i in range(4):
        xi = _randn(g, B, 1, C, dtype=BF).to(dev)
        li = torch.tensor([i, 590 + i, 700 + 3 * i], dtype=torch.int32, device=dev)
        ki, vi = (_randn(g, B, G, S, D, dtype=BF).to(dev) for _ in range(2))
        x.copy_(xi), lens.copy_(li), kc.copy_(ki), vc.copy_(vi)
        graph.replay()
        torch.cuda.synchronize()
        got, gk, gv = out.clone(), kc.clone(), vc.clone()
        x.copy_(xi), lens.copy_(li), kc.copy_(ki), vc.copy_(vi)
        want = layer()
        assert torch.equal(got, want) and torch.equal(gk, kc) and torch.equal(gv, vc)
        assert bool(torch.isfinite(got).all())


def test_options_given_as_tensors_are_read_at_each_call(dev):
    gen = torch.Generator().manual_seed(77)
    q, k, v = (_randn(gen, 1, 2, 40, 64, dtype=BF).to(dev) for _ in range(3))
    scale, left = torch.tensor(0.125), torch.tensor(3)
    first = ops.window_attention(q, k, v, left, 0, scale=scale)
    assert torch.equal(first, ops.window_attention(q, k, v, 3, 0, scale=0.125))
    scale.fill_(0.5)
    left.fill_(20)
    again = ops.window_attention(q, k, v, left, 0, scale=scale)
    assert torch.equal(again, ops.window_attention(q, k, v, 20, 0, scale=0.5))
    assert not torch.equal(first, again)
    wide = ops.window_attention(q, k, v, 1 << 64, 1 << 64, sinks=1 << 64)
    assert torch.equal(wide, ops.window_attention(q, k, v))


# --------------------------------------------------------------------------
# long: positions near 2^30, offsets beyond 32 bits
# --------------------------------------------------------------------------

@pytest.mark.parametrize("L", [1, 48])
def test_rolling_positions_near_two_to_the_thirty(dev, L):
    """The same slots in the same tiles, 2^30 tokens later: the same bits."""
    gen = torch.Generator().manual_seed(78)
    sinks, ring = 128, 1024
    q = _randn(gen, 2, 4, L, 128, dtype=BF).to(dev)
    k, v = (_randn(gen, 2, 2, sinks + ring, 128, dtype=BF).to(dev) for _ in range(2))
    lens = torch.tensor([5000, 7001], dtype=torch.int32, device=dev)
    args = dict(left=900, right=0, sinks=sinks, rolling=True)
    near = ops.window_attention(q, k, v, kv_lens=lens, **args)
    far = ops.window_attention(q, k, v, kv_lens=lens + (1 << 30), **args)
    assert torch.equal(near, far)
    new = _randn(gen, 2, L, 2, 128, dtype=BF).to(dev)
    k2, v2 = k.clone(), v.clone()
    a = ops.qkv_cache(q.transpose(1, 2), new, new, k, v, lens, sinks=sinks, rolling=True)
    b = ops.qkv_cache(q.transpose(1, 2), new, new, k2, v2, lens + (1 << 30), sinks=sinks, rolling=True)
    assert torch.equal(a, b) and torch.equal(k, k2) and torch.equal(v, v2)


def test_linear_offsets_beyond_32_bits(dev):
    gen = torch.Generator().manual_seed(79)
    x, w = _randn(gen, 300_000, 64, dtype=BF), _randn(gen, 8192, 64, dtype=BF)
    out = ops.linear(x.to(dev), w.to(dev))
    tail, tol = refs.linear(x[-70:], w)
    _within(out[-70:], tail, tol, "out")
    del out
    wide = torch.empty(3000, 1 << 20, dtype=BF, device=dev)
    for m, n in ((3000, 200), (8, 3000)):  # x, then w far apart
        a, b = _randn(gen, m, 64, dtype=BF), _randn(gen, n, 64, dtype=BF)
        wide[-m if m > n else -n:, 64:128] = (a if m > n else b).to(dev)
        far = wide[-max(m, n):, 64:128]
        got = ops.linear(far, b.to(dev)) if m > n else ops.linear(a.to(dev), far)
        ref, tol = refs.linear(a, b)
        _within(got, ref, tol, f"{m} x {n}")


@pytest.mark.parametrize("L", [1, 200])
def test_caches_beyond_32_bits(dev, L):
    gen = torch.Generator().manual_seed(80)
    slots, near = 18_000_128, 1152  # 4.6 GB a cache; both ends on a tile's boundary
    kc, vc = (torch.empty(1, 1, slots, 128, dtype=BF, device=dev) for _ in range(2))
    kc[:, :, -near:] = _randn(gen, 1, 1, near, 128, dtype=BF).to(dev)
    vc[:, :, -near:] = _randn(gen, 1, 1, near, 128, dtype=BF).to(dev)
    q = _randn(gen, 1, L, 2, 128, dtype=BF).to(dev)
    new = [_randn(gen, 1, L, 1, 128, dtype=BF).to(dev) for _ in range(2)]
    lens = torch.tensor([slots - L], dtype=torch.int32, device=dev)
    ks, vs = kc[:, :, -near:].clone(), vc[:, :, -near:].clone()
    qn = ops.qkv_cache(q, *new, kc, vc, lens)
    ops.qkv_cache(q, *new, ks, vs, lens - (slots - near))
    assert torch.equal(kc[:, :, -near:], ks) and torch.equal(vc[:, :, -near:], vs)
    assert torch.equal(kc[0, 0, -L:], new[0][0, :, 0])
    got = ops.window_attention(qn, kc, vc, left=500, right=0)
    ref, tol = refs.window_attention(qn.cpu(), ks.cpu(), vs.cpu(), left=500, right=0)[::2][:2]
    _within(got, ref, tol, "attention")


# --------------------------------------------------------------------------
# views whose channels share an element
# --------------------------------------------------------------------------

def _shared_channels(t):
    """Views of t's shape whose channels have stride 0: of its first channel,
    of a later one, of one element."""
    return t[..., :1].expand(t.shape), t[..., 8:9].expand(t.shape), t.flatten()[5].expand(t.shape)


@pytest.mark.parametrize("L", [2, 70])
def test_operators_take_channels_that_share_an_element(dev, L):
    gen = torch.Generator().manual_seed(81)
    base = {n: _randn(gen, 2, h, s, 64, dtype=BF).to(dev) for n, h, s in (("q", 4, L), ("k", 2, 90), ("v", 2, 90))}
    lens = torch.tensor([3, 0], dtype=torch.int32, device=dev)
    for name in base:
        for view in _shared_channels(base[name]):
            print(f"shared channels L={L} {name} {tuple(view.stride())}", flush=True)
            args = {**base, name: view}
            got = ops.window_attention(**args, left=40, right=0)
            assert torch.equal(got, ops.window_attention(**{**args, name: view.contiguous()}, left=40, right=0))
            new = {**{n: base["v" if n == "k" else "k"][:, :, :5].transpose(1, 2) for n in "qkv"},
                   name: view[:, :2, :2].transpose(1, 2)}
            new = {n: t[:, :2] for n, t in new.items()}
            assert new[name].stride(3) == 0
            caches = [[torch.zeros(2, 2, 9, 64, dtype=BF, device=dev) for _ in range(2)] for _ in range(2)]
            a = ops.qkv_cache(**new, k_cache=caches[0][0], v_cache=caches[0][1], lens=lens)
            whole = {n: t.contiguous() for n, t in new.items()}
            b = ops.qkv_cache(**whole, k_cache=caches[1][0], v_cache=caches[1][1], lens=lens)
            assert torch.equal(a, b)
            assert torch.equal(caches[0][0], caches[1][0]) and torch.equal(caches[0][1], caches[1][1])
            x = view[0, 0]
            w = base["k"][0, 0]
            assert torch.equal(ops.linear(x, w), ops.linear(x.contiguous(), w))
            assert torch.equal(ops.linear(w, x), ops.linear(w, x.contiguous()))


# --------------------------------------------------------------------------
# weights far below a row's largest
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("L,S,D,place", [(1, 4000, 64, 0), (1, 300, 128, 299), (40, 4000, 128, 0), (40, 900, 64, 450)])
@pytest.mark.parametrize("nats,spread", [(10.0, 0.3), (14.0, 0.3), (17.0, 0.3), (16.0, 0.0), (17.5, 0.0)])
def test_window_attention_keeps_small_weights(dev, L, S, D, place, nats, spread, dtype):
    """A key that takes nearly all of every row's weight and whose values are
    zero (a sink): the output is what the other keys, 10 to 18 nats below it,
    leave, and the bound is relative to that. f16 holds 11 bits down to 2^-14
    and the largest weight stands at 2^13 or more, so 18.7 nats below it."""
    print(f"small weights L={L} S={S} D={D} at {place} {nats} nats spread {spread} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(L + S)
    q, k = (_randn(gen, 1, 2, n, D, dtype=dtype, std=spread / math.sqrt(D)) for n in (L, S))
    v = _randn(gen, 1, 2, S, D, dtype=dtype).abs() + 0.5
    q[..., 0] = 1
    k[..., 0] = _randn(gen, 1, 2, S, dtype=dtype, std=spread)
    k[:, :, place, 0], v[:, :, place] = nats, 0
    ref, lse_ref, tol, lse_tol = refs.window_attention(q, k, v, scale=1.0)
    assert 0.9 < float((torch.log(ref.mean()) + nats - math.log(S)).exp()) < 2.0
    out, lse = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), scale=1.0, want_lse=True)
    _within(out, ref, tol, "small weights")
    _within(lse, lse_ref, lse_tol, "their lse")


# --------------------------------------------------------------------------
# the log-sum-exp
# --------------------------------------------------------------------------

def _fp32_lse_tol(lse_ref, lse_tol, dtype):
    """operator_refs' bound of the lse without the rounding of the weights to
    the operands' type, for which rows that see keys have 2 u in it: what the
    fp32 scores, their sum and its logarithm take."""
    return lse_tol - 2 * refs.half_step(dtype) * (lse_ref != -math.inf)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("L,D", [(1, 64), (1, 128), (8, 64), (40, 128), (300, 64)])
def test_window_attention_lse_is_fp32(dev, L, D, dtype):
    """Rows that see two keys in tiles apart, the first key and their own,
    whose score is up to 5 nats higher or lower: the weight of neither is a
    number of the operands' type."""
    print(f"lse L={L} D={D} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(L + D)
    S, B = 200 + L, 1 if L > 8 else 40
    q = torch.zeros(B, 2, L, D, dtype=dtype)
    k, v = torch.zeros(B, 2, S, D, dtype=dtype), _randn(gen, B, 2, S, D, dtype=dtype)
    q[..., 0] = 1
    k[:, :, 1:, 0] = (torch.rand(B, 2, S - 1, generator=gen) * 10 - 5).to(dtype)
    ref, lse_ref, tol, lse_tol = refs.window_attention(q, k, v, left=0, right=0, sinks=1, scale=1.0)
    out, lse = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), left=0, right=0, sinks=1, scale=1.0, want_lse=True)
    _within(out, ref, tol, "out")
    _within(lse, lse_ref, _fp32_lse_tol(lse_ref, lse_tol, dtype), "lse")


@pytest.mark.parametrize("B,H,G,L,S,D,dtype,left,right,sinks,q_lens,kv_lens,rolling", ATTENTION)
def test_window_attention_lse_is_fp32_everywhere(dev, B, H, G, L, S, D, dtype, left, right, sinks, q_lens, kv_lens,
                                                 rolling):
    """The same bound over the forms and parts; out does not depend on whether
    the lse is asked for."""
    print(f"lse B={B} H={H} G={G} L={L} S={S} D={D} {dtype} left={left} right={right} sinks={sinks} "
          f"q={q_lens} kv={kv_lens} rolling={rolling}", flush=True)
    g = torch.Generator().manual_seed(L * S + H + 1)
    q, k, v = (_randn(g, B, n, s, D, dtype=dtype) for n, s in ((H, L), (G, S), (G, S)))
    _, lse_ref, _, lse_tol = refs.window_attention(q, k, v, left, right, sinks, q_lens, kv_lens, rolling)
    lens = [None if t is None else torch.tensor(t, dtype=torch.int32, device=dev) for t in (q_lens, kv_lens)]
    args = (q.to(dev), k.to(dev), v.to(dev), left, right, sinks, *lens)
    out, lse = ops.window_attention(*args, rolling=rolling, want_lse=True)
    assert torch.equal(out, ops.window_attention(*args, rolling=rolling))
    empty = lse_ref == -math.inf
    lse = lse.cpu().double()
    assert torch.equal(lse == -math.inf, empty)
    _within(lse.masked_fill(empty, 0), lse_ref.masked_fill(empty, 0), _fp32_lse_tol(lse_ref, lse_tol, dtype), "lse")
