"""GPU parity of ops.quantize_fp8 and ops.linear_fp8 with their 64-bit
definitions (block_refs)."""
import math

import pytest
import torch

import block_refs as refs
from dfsattn_amd import ops
from test_block_ops_host import FORMS, form

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


def _hidden(gen, rows, k, dtype):
    """Rows and channels of very different sizes."""
    x = torch.randn(rows, k, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen))
    x[:, ::37] *= 30
    return x.to(dtype)


def _same_codes(got, want):
    """Codes and scales equal to quantize's 64-bit values, NaN to NaN."""
    for g, w in zip(got, want):
        g = g.cpu().double()
        assert g.shape == w.shape
        assert torch.equal(torch.isnan(g), torch.isnan(w))
        assert torch.equal(torch.nan_to_num(g), torch.nan_to_num(w))


# --------------------------------------------------------------------------
# quantize_fp8
# --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 127), (5, 129), (2, 8), (77, 1001), (300, 640), (9, 5120),
                                    (1000, 136)])
def test_quantize_matches_definition(dev, rows, k, dtype):
    print(f"quantize {rows} x {k} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows * 3 + k)
    x = _hidden(g, rows, k, dtype)
    _same_codes(ops.quantize_fp8(x.to(dev)), refs.quantize(x))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_quantize_every_value(dev, dtype):
    """All 2^16 values, each the largest of a block beside smaller ones, each a
    small one beside a large one, zeros and values that are not finite."""
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    alone = torch.zeros(1 << 16, 128, dtype=dtype)
    alone[:, 5] = every
    alone[:, 99] = torch.where(torch.isfinite(every), every * 0.37, torch.ones(()).to(dtype))
    beside = every.view(-1, 128).clone()
    beside[:, 0] = 1.75
    for x in (alone, beside, every.view(-1, 256)):
        print("quantize every value", tuple(x.shape), flush=True)
        _same_codes(ops.quantize_fp8(x.to(dev)), refs.quantize(x))


def test_quantize_views(dev):
    """Rows inside wider ones at any element, a batch axis, a transposed view, no rows."""
    g = torch.Generator().manual_seed(0)
    wide = _hidden(g, 60, 400, BF)
    for off in (0, 8, 3):
        x = wide.view(4, 15, 400)[:, :, off:off + 300]
        got = ops.quantize_fp8(wide.to(dev).view(4, 15, 400)[:, :, off:off + 300])
        assert got[0].shape == (4, 15, 300) and got[1].shape == (4, 15, 3)
        _same_codes([t.flatten(0, 1) if t.is_contiguous() else t.reshape(60, -1) for t in
                     (got[0], got[1].view(torch.uint8).reshape(60, 3).view(torch.float8_e8m0fnu))],
                    refs.quantize(x.reshape(60, 300)))
    t = wide.t()
    _same_codes(ops.quantize_fp8(wide.to(dev).t()), refs.quantize(t))
    one = ops.quantize_fp8(wide[0].to(dev))
    assert one[0].shape == (400,) and one[1].shape == (4,)
    none = ops.quantize_fp8(wide[:0].to(dev))
    assert none[0].shape == (0, 400) and none[1].shape == (0, 4)


# --------------------------------------------------------------------------
# linear_fp8
# --------------------------------------------------------------------------

LINEAR = [
    # M, N, K, dtype, x in codes, bias dtype, act, gate, residual
    (1, 64, 64, BF, False, BF, None, False, False),
    (1, 1, 1, BF, True, None, None, False, True),
    (1, 2048, 1024, BF, False, torch.float32, "silu", False, False),
    (3, 257, 2500, HF, True, HF, "gelu_tanh", True, True),
    (2, 200, 8200, BF, False, BF, None, False, False),
    (16, 640, 256, BF, True, BF, "gelu", False, True),
    (17, 96, 2048, HF, False, None, None, True, False),
    (33, 1000, 1032, BF, True, BF, "gelu_tanh", False, False),
    (64, 520, 4096, BF, False, None, None, False, True),
    (65, 129, 63, BF, True, BF, "silu", True, True),
    (100, 128, 65, HF, False, torch.float32, None, False, False),
    (127, 255, 511, HF, True, HF, "gelu", True, True),
    (128, 128, 128, BF, False, BF, None, False, False),
    (200, 384, 640, BF, True, BF, "gelu_tanh", True, True),
    (256, 256, 64, BF, False, None, None, False, False),
    (257, 513, 72, HF, True, HF, None, False, True),
    (300, 1025, 1000, BF, False, BF, "silu", False, False),
    (513, 1024, 1024, BF, True, BF, "gelu_tanh", False, True),
    (1000, 776, 136, HF, False, None, None, True, True),
    (2100, 2056, 192, BF, True, BF, None, True, True),
    (2049, 2304, 328, HF, False, HF, "gelu_tanh", False, False),
    (4099, 1100, 70, BF, True, torch.float32, "gelu_tanh", False, True),
]


@pytest.mark.parametrize("m,n,k,dtype,codes,bias,act,gate,residual", LINEAR)
def test_linear_fp8_matches_definition(dev, m, n, k, dtype, codes, bias, act, gate, residual):
    print(f"linear_fp8 {m} x {n} x {k} {dtype} codes={codes} bias={bias} act={act} gate={gate} residual={residual}",
          flush=True)
    g = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    x, w = _hidden(g, m, k, dtype), _randn(g, n, k, dtype=dtype, std=2 / math.sqrt(k))
    xq, wq = refs.quantize(x), refs.quantize(w)
    b = None if bias is None else _randn(g, n, dtype=bias)
    gt = torch.randn(n, generator=g) if gate else None
    r = _randn(g, m, n, dtype=dtype) if residual else None
    xt, wt = refs.to_tensors(*xq), refs.to_tensors(*wq)
    ref, tol = refs.linear_fp8(refs.values(*xt), refs.values(*wt), dtype, b, act, gt, r)
    d = [None if t is None else t.to(dev) for t in (*(xt if codes else (x, None)), *wt, b, gt, r)]

    def call(**kw):
        return ops.linear_fp8(d[0], d[2], d[3], d[1], bias=d[4], activation=act, gate=d[5], residual=d[6],
                              out_dtype=dtype, **kw)

    got = call()
    assert got.dtype == dtype
    _within(got, ref, tol, "linear_fp8")
    assert torch.equal(got, call())
    _same_codes(call(quantize=True), refs.quantize(got.cpu()))
    # scales whose rows lie one behind the other are read in place: the same
    d[3] = ops._scales_laid_out(d[3])
    d[1] = d[1] if d[1] is None else ops._scales_laid_out(d[1])
    assert torch.equal(got, call())
    if residual:  # in place of the residual
        d[6] = call(out=d[6])
        assert torch.equal(got, d[6])


@pytest.mark.parametrize("m,n,k,codes,act", [(4200, 4200, 3000, False, "gelu_tanh"), (2560, 6500, 4104, True, None),
                                             (4185, 1953, 264, True, "silu"), (4099, 5003, 200, False, "gelu"),
                                             (4000, 4001, 2057, True, None), (8200, 8200, 128, False, None)])
def test_linear_fp8_large_tiles(dev, m, n, k, codes, act):
    """256 x 256 tiles, whole and behind the last full round in parts; rows and
    outputs picked all over the result."""
    print(f"linear_fp8 {m} x {n} x {k} codes={codes} {act}", flush=True)
    gen = torch.Generator().manual_seed(m + n + k)
    x, w = _hidden(gen, m, k, BF), _randn(gen, n, k, dtype=BF, std=2 / math.sqrt(k))
    b, gate, r = _randn(gen, n, dtype=BF), torch.randn(n, generator=gen), _randn(gen, m, n, dtype=BF)
    xt, wt = refs.to_tensors(*refs.quantize(x)), refs.to_tensors(*refs.quantize(w))
    d = [None if t is None else t.to(dev) for t in (*(xt if codes else (x, None)), *wt, b, gate, r)]

    def call(**kw):
        return ops.linear_fp8(d[0], d[2], d[3], d[1], bias=d[4], activation=act, gate=d[5], residual=d[6], **kw)

    got = call()
    assert torch.equal(got, call())
    rows, cols = torch.arange(0, m, 13), torch.arange(0, n, 11)
    rows[-1], cols[-1] = m - 1, n - 1
    ref, tol = refs.linear_fp8(refs.values(*xt)[rows], refs.values(*wt)[cols], BF, b[cols], act, gate[cols],
                               r[rows][:, cols])
    _within(got.cpu()[rows][:, cols], ref, tol, "large tiles")
    for a, b in zip(call(quantize=True), ops.quantize_fp8(got)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    d[3], d[1] = ops._scales_laid_out(d[3]), d[1] if d[1] is None else ops._scales_laid_out(d[1])
    assert torch.equal(got, call())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,n,k,want", FORMS)
def test_linear_fp8_forms(dev, m, n, k, want, dtype):
    """Every kernel that sizes can choose, both types, all steps of the epilogue;
    x in codes and in 16 bits, the result in both; what surrounds out stays."""
    print(f"linear_fp8 form {want}: {m} x {n} x {k} {dtype}", flush=True)
    assert form(m, n, k) == want
    g = torch.Generator().manual_seed(m + 3 * n + k)
    x, w = _hidden(g, m, k, dtype), _randn(g, n, k, dtype=dtype, std=2 / math.sqrt(k))
    b, gate, r = _randn(g, n, dtype=dtype), torch.randn(n, generator=g), _randn(g, m, n, dtype=dtype)
    xt, wt = refs.to_tensors(*refs.quantize(x)), refs.to_tensors(*refs.quantize(w))
    rows, cols = torch.arange(0, m, max(1, m // 150)), torch.arange(0, n, max(1, n // 150))
    rows[-1], cols[-1] = m - 1, n - 1
    ref, tol = refs.linear_fp8(refs.values(*xt)[rows], refs.values(*wt)[cols], dtype, b[cols], "gelu_tanh", gate[cols],
                               r[rows][:, cols])
    d = [t.to(dev) for t in (x, *xt, *wt, b, gate, r)]
    room = torch.full((m * n + 512,), 7.0, dtype=dtype, device=dev)
    out = room[256:256 + m * n].view(m, n)
    for at, scales in ((d[1], d[2]), (d[0], None)):
        got = ops.linear_fp8(at, d[3], d[4], scales, bias=d[5], activation="gelu_tanh", gate=d[6], residual=d[7],
                             out_dtype=dtype, out=out)
        _within(got.cpu()[rows][:, cols], ref, tol, "form")
        assert bool((room[:256] == 7).all()) and bool((room[256 + m * n:] == 7).all())
        codes = ops.linear_fp8(at, d[3], d[4], scales, bias=d[5], activation="gelu_tanh", gate=d[6], residual=d[7],
                               out_dtype=dtype, quantize=True)
        for a, b_ in zip(codes, ops.quantize_fp8(got)):
            assert torch.equal(a.view(torch.uint8), b_.view(torch.uint8))


@pytest.mark.parametrize("m,n,k", [(2, 100, 300), (40, 200, 700), (300, 520, 1000), (913, 7811, 224)])
def test_linear_fp8_infinities_and_nan_stay_in_their_rows(dev, m, n, k):
    """Values of x that are not finite make their row NaN, others what they are
    without them; a NaN scale of w its output."""
    print(f"linear_fp8 not finite {m} x {n} x {k}", flush=True)
    g = torch.Generator().manual_seed(m)
    x, w = _hidden(g, m, k, BF), _randn(g, n, k, dtype=BF)
    wt = [t.to(dev) for t in refs.to_tensors(*refs.quantize(w))]
    whole = ops.linear_fp8(x.to(dev), *wt)
    x[0, 5], x[m - 1, k - 1] = math.inf, math.nan
    keep = torch.ones(m, dtype=torch.bool)
    keep[[0, m - 1]] = False
    got = ops.linear_fp8(x.to(dev), *wt)
    assert bool(torch.isnan(got[[0, m - 1]]).all())
    assert torch.equal(got[keep], whole[keep])
    bad = wt[1].view(torch.uint8).clone()
    bad[3, 0] = 255
    got = ops.linear_fp8(x.to(dev), wt[0], bad.view(torch.float8_e8m0fnu))
    others = torch.arange(n) != 3
    assert bool(torch.isnan(got[:, 3]).all()) and torch.equal(got[keep][:, others], whole[keep][:, others])


@pytest.mark.parametrize("m", [1, 5, 40, 130, 700])
def test_linear_fp8_strided_rows_and_batches(dev, m):
    """Codes inside wider rows on and off 16-byte boundaries, a batch axis, scales
    of any strides, a residual that is a transposed view."""
    g = torch.Generator().manual_seed(m)
    k, n = 272, 136
    x, w, r = _hidden(g, 2 * m, k, BF), _randn(g, n, k, dtype=BF, std=0.1), _randn(g, n, 2, m, dtype=BF)
    (xc, xs), (wc, ws) = refs.to_tensors(*refs.quantize(x)), refs.to_tensors(*refs.quantize(w))
    ref, tol = refs.linear_fp8(refs.values(xc, xs), refs.values(wc, ws), BF, None, None, None,
                               r.permute(1, 2, 0).reshape(-1, n))
    rd = r.to(dev).permute(1, 2, 0)
    for off in (0, 16, 3):
        print(f"linear_fp8 strided m={m} offset={off}", flush=True)

        def inside(t, pad):
            wide = torch.zeros((*t.shape[:-1], t.shape[-1] + pad), dtype=torch.uint8)
            wide[..., off:off + t.shape[-1]] = t.view(torch.uint8)
            return wide.to(dev)[..., off:off + t.shape[-1]].view(t.dtype)

        got = ops.linear_fp8(inside(xc.view(2, m, k), 48), inside(wc, 32), inside(ws, 25), inside(xs.view(2, m, -1), 27),
                             residual=rd)
        assert got.shape == (2, m, n)
        _within(got.reshape(-1, n), ref, tol, "strided")
        half = torch.zeros(2, m, k + 24, dtype=BF)
        half[:, :, off:off + k] = x.view(2, m, k)
        assert torch.equal(got, ops.linear_fp8(half.to(dev)[:, :, off:off + k], wc.to(dev), ws.to(dev), residual=rd))


def test_linear_fp8_empty_and_one(dev):
    w = ops.quantize_fp8(torch.ones(8, 16, dtype=BF, device=dev))
    assert ops.linear_fp8(torch.zeros(0, 16, dtype=BF, device=dev), *w).shape == (0, 8)
    codes, scales = ops.linear_fp8(torch.zeros(0, 16, dtype=BF, device=dev), *w, quantize=True)
    assert codes.shape == (0, 8) and scales.shape == (0, 1)
    one = ops.linear_fp8(torch.ones(16, dtype=BF, device=dev), *w)
    assert one.shape == (8,) and bool((one == 16).all())
    codes, scales = ops.linear_fp8(torch.ones(16, dtype=BF, device=dev), *w, quantize=True)
    assert codes.shape == (8,) and scales.shape == (1,)


def test_fp8_offsets_beyond_32_bits(dev):
    """More than 2^31 elements of x to quantise, and of outputs."""
    print("quantize 430,000 x 5,120", flush=True)
    x = torch.zeros(430000, 5120, dtype=BF, device=dev)
    x[-3:] = torch.randn(3, 5120, generator=torch.Generator().manual_seed(0)).to(BF).to(dev)
    codes, scales = ops.quantize_fp8(x)
    _same_codes((codes[-3:], scales[-3:]), refs.quantize(x[-3:].cpu()))
    del x, codes, scales
    print("linear_fp8 160,000 x 13,824 x 128", flush=True)
    g = torch.Generator().manual_seed(1)
    x, w = _randn(g, 160000, 128, dtype=BF), _randn(g, 13824, 128, dtype=BF, std=0.1)
    wt = [t.to(dev) for t in refs.to_tensors(*refs.quantize(w))]
    got = ops.linear_fp8(x.to(dev), *wt)
    alone = ops.linear_fp8(x[-5:].to(dev), *wt)
    ref, tol = refs.linear_fp8(refs.values(*refs.to_tensors(*refs.quantize(x[-5:]))),
                               refs.values(*(t.cpu() for t in wt)), BF)
    _within(got[-5:], ref, tol, "last rows")
    _within(alone, ref, tol, "alone")
