"""What ops.quantize_fp8, ops.linear_fp8, ops.residual_norm and ops.axial_rope
refuse, before any device is touched, and the sizes that reach each kernel of
linear_fp8."""
import copy
import dataclasses
import pickle
import random

import pytest
import torch

import block_refs as refs
from dfsattn_amd import _lib, fp8, ops
from operator_cases import FEW, PARTS, STREAM, T64, T64X128, T128, T128_DEEP, T256, WIDE

BF, HF, F32, E4, E8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=torch.uint8).view(dtype) if dtype in (E4, E8) else torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("x", [_t(4, 16, dtype=F32), _t(4, 0), torch.zeros((), dtype=BF)])
def test_quantize_refuses(x):
    with pytest.raises(ValueError):
        ops.quantize_fp8(x)


LINEAR = dict(x=_t(4, 200), weight=_t(8, 200, dtype=E4), weight_scales=_t(8, 2, dtype=E8))
CODES = dict(x=_t(4, 200, dtype=E4), x_scales=_t(4, 2, dtype=E8))


@pytest.mark.parametrize("change", [
    {"x": _t(4, 200, dtype=F32)},
    {"x": _t(4, 199)},
    {"weight": _t(8, 200)},
    {"weight": _t(8, 2, 100, dtype=E4)},
    {"weight": _t(0, 200, dtype=E4), "weight_scales": _t(0, 2, dtype=E8)},
    {"weight_scales": None},
    {"weight_scales": _t(8, 1, dtype=E8)},
    {"weight_scales": _t(8, 2, dtype=F32)},
    {"x_scales": _t(4, 2, dtype=E8)},
    {"x": _t(4, 200, dtype=E4)},
    {**CODES, "x_scales": _t(4, 1, dtype=E8)},
    {**CODES, "out_dtype": F32},
    {"out_dtype": HF},
    {"activation": "relu"},
    {"bias": _t(7)},
    {"bias": _t(8, dtype=HF)},
    {"gate": _t(8)},
    {"gate": _t(4, dtype=F32)},
    {"residual": _t(4, 7)},
    {"residual": _t(4, 8, dtype=HF)},
    {**CODES, "residual": _t(4, 8, dtype=F32)},
    {"out": _t(5, 8)},
    {"out": _t(4, 8, dtype=HF)},
    {"out": _t(4, 8), "quantize": True},
])
def test_linear_fp8_refuses(change):
    with pytest.raises(ValueError):
        ops.linear_fp8(**{**LINEAR, **change})


NORM = dict(x=_t(2, 3, 16), y=_t(2, 3, 16))


@pytest.mark.parametrize("change", [
    {"x": _t(2, 3, 16, dtype=F32)},
    {"y": _t(2, 3, 16, dtype=HF)},
    {"y": _t(6, 16)},
    {"x": _t(2, 0), "y": _t(2, 0)},
    {"x": _t(2, 8193), "y": _t(2, 8193)},
    {"norm": "group"},
    {"norm": None},
    {"post_norm": "batch"},
    {"post_weight": _t(16)},
    {"post_norm": "rms", "post_weight": _t(15)},
    {"post_norm": "rms", "post_weight": _t(16, dtype=torch.float64)},
    {"weight": _t(3, 16)},
    {"gate": _t(16)},
    {"gate": _t(3, 2, 16, dtype=F32)},
    {"gate": _t(2, 3, 1, 16, dtype=F32)},
    {"scale": _t(15, dtype=F32)},
    {"shift": _t(3, 3, 16, dtype=F32)},
    {"eps": -1.0},
    {"eps": float("nan")},
    {"post_eps": -1.0},
    {"residual_scale": float("inf")},
    {"y": None, "gate": _t(16, dtype=F32)},
    {"y": None, "residual_scale": 0.5},
    {"y": None, "out": _t(2, 3, 16)},
    {"out": _t(6, 16)},
    {"out": _t(2, 3, 16, dtype=HF)},
])
def test_residual_norm_refuses(change):
    with pytest.raises(ValueError):
        ops.residual_norm(**{**NORM, **change})


AXES = ops.RotaryAxes(64, (24, 20, 20))
ROPE = dict(q=_t(2, 3, 4, 64), k=_t(2, 3, 2, 64), axes=AXES, grid=(4, 5))


@pytest.mark.parametrize("change", [
    {"q": _t(2, 3, 4, 64, dtype=F32)},
    {"k": _t(2, 3, 2, 64, dtype=HF)},
    {"q": _t(3, 4, 64)},
    {"k": _t(2, 4, 2, 64)},
    {"k": _t(2, 3, 0, 64)},
    {"q": _t(2, 3, 4, 72), "k": _t(2, 3, 2, 72)},
    {"q": _t(2, 3, 129, 64)},
    {"axes": (24, 20, 20)},
    {"grid": None},
    {"grid": (4,)},
    {"grid": (4, 0)},
    {"positions": _t(3, 3, dtype=torch.int32)},
    {"grid": None, "positions": _t(3, 3, dtype=torch.int64)},
    {"grid": None, "positions": _t(3, 2, dtype=torch.int32)},
    {"grid": None, "positions": _t(3, 3, 3, dtype=torch.int32)},
    {"grid": None, "positions": _t(3, 3, dtype=torch.int32), "start": _t(2, dtype=torch.int32)},
    {"start": _t(3, dtype=torch.int32)},
    {"start": _t(2, dtype=torch.int64)},
    {"q_weight": _t(128)},
    {"k_weight": _t(64, 1)},
    {"k": None, "k_weight": _t(64)},
    {"eps": -1.0},
])
def test_axial_rope_refuses(change):
    with pytest.raises(ValueError):
        ops.axial_rope(**{**ROPE, **change})


@pytest.mark.parametrize("args", [(64, ()), (64, (24, 20, 21)), (64, (40, 40)), (64, (2, 2, 2, 2, 2)), (60, (20,)),
                                  (1024, (20,)), (64, (20,), 0.0), (64, (20, 20), (1e4,)), (64, (20,), 1e4, "rows"),
                                  (64, (20,), 1e4, "pairs", float("inf"))])
def test_rotary_axes_refuse(args):
    with pytest.raises(ValueError):
        ops.RotaryAxes(*args)


def test_grid_rotary_table_is_the_models():
    from dfsattn_amd.dit import wan_rope_freqs

    table = ops.GridRotary(ops.RotaryAxes(128, (44, 42, 42)), (5, 7)).table(3 * 5 * 7)
    assert torch.allclose(table, wan_rope_freqs((3, 5, 7), 128), rtol=0, atol=1e-12)
    with pytest.raises(ValueError):
        ops.GridRotary(ops.RotaryAxes(64, (64,), layout="halves"), ()).table(3)


def test_block_operators_refuse_the_cpu_and_gradients():
    for call in (lambda: ops.quantize_fp8(_t(4, 16)), lambda: ops.linear_fp8(**LINEAR),
                 lambda: ops.residual_norm(**NORM), lambda: ops.axial_rope(**ROPE)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()
    for call in (lambda: ops.quantize_fp8(_t(4, 16).requires_grad_()),
                 lambda: ops.linear_fp8(**{**LINEAR, "bias": _t(8).requires_grad_()}),
                 lambda: ops.residual_norm(**{**NORM, "weight": _t(16).requires_grad_()}),
                 lambda: ops.axial_rope(**{**ROPE, "q": _t(2, 3, 4, 64).requires_grad_()})):
        with pytest.raises(RuntimeError, match="no backward"):
            call()


def test_fp8_linear_keeps_its_bytes_through_casts():
    layer = fp8.Fp8Linear(_t(8, 200, dtype=E4), _t(8, 2, dtype=E8), _t(8)).to(HF)
    assert layer.codes.dtype == layer.scales.dtype == torch.uint8 and layer.bias.dtype == HF


def test_e4m3_rounding_of_the_reference():
    """The 64-bit rounding agrees with torch's conversion on every half-way and
    whole value that e4m3 knows, and on many others."""
    codes = torch.arange(127, dtype=torch.uint8).view(E4).double()  # 0 to 448
    mid = (codes[1:] + codes[:-1]) / 2
    v = torch.cat([codes, mid, torch.rand(4000, dtype=torch.float64) * 448, torch.rand(4000, dtype=torch.float64) / 16])
    v = v.float().double()
    assert torch.equal(refs.e4m3(v), v.float().to(E4).double())


# rows, outputs, channels, form (dfs_linear_fp8_form)
FORMS = [
    (1, 77, 8, FEW | WIDE),
    (16, 1003, 520, FEW | WIDE),
    (5, 4105, 264, FEW),
    (3, 16411, 16520, FEW | STREAM),
    (9, 20011, 520, T64),
    (13, 16411, 12008, T64 | PARTS),
    (77, 331, 328, T64),
    (33, 523, 4104, T64 | PARTS),
    (129, 7615, 168, T64X128),
    (401, 785, 5959, T64X128 | PARTS),
    (258, 6583, 171, T128_DEEP),
    (2805, 459, 12116, T128_DEEP | PARTS),
    (517, 6559, 169, T128),
    (137, 3069, 10069, T128 | PARTS),
    (913, 7811, 224, T256),
    (1785, 2357, 12148, T256 | PARTS),
]


def form(m, n, k):
    return _lib.lib().dfs_linear_fp8_form(m, n, k)


@pytest.mark.parametrize("m,n,k,want", FORMS)
def test_linear_fp8_cases_take_their_form(m, n, k, want):
    assert form(m, n, k) == want


def test_every_form_of_linear_fp8_has_a_case():
    rng, listed = random.Random(0), {c[-1] for c in FORMS}
    for _ in range(60000):
        m, n, k = (int(2 ** rng.uniform(0, e)) for e in (13, 15, 14.5))
        assert form(m, n, k) in listed, (m, n, k, form(m, n, k))
    for sizes in ((0, 1, 1), (1, -1, 1), (1, 1, 0), (1, 1, 1 << 21)):
        assert form(*sizes) == -1
        assert _lib.lib().dfs_linear_fp8_workspace_size(*sizes, 0) == -1


def test_fp8_linear_knows_its_layers_type():
    layer = fp8.Fp8Linear(_t(8, 200, dtype=E4), _t(8, 2, dtype=E8), None, HF)
    assert layer.dtype == HF and layer.to(torch.bfloat16).dtype == torch.bfloat16
    assert set(layer.state_dict()) == {"codes", "scales"}


def test_rotary_axes_are_keys_by_value():
    a, b = (ops.RotaryAxes(128, n, 1e4, "halves", 2) for n in ((44, 42, 42), [44, 42, 42]))
    copies = (b, copy.deepcopy(a), pickle.loads(pickle.dumps(a)), dataclasses.replace(a))
    assert all(a == c and hash(a) == hash(c) for c in copies)
    for other in (ops.RotaryAxes(128, (44, 42, 42), 1e4, "pairs", 2), dataclasses.replace(a, theta=1e3)):
        assert a != other and {a: 1}.get(other) is None
