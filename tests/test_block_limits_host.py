"""Sizes past what a launch holds (fewer than 2^32 threads) are refused by the C
entries before they launch. The pointers are never read: only refused calls are
made here."""
import pytest
import torch

from dfsattn_amd import _lib, ops

AT = 1 << 20  # an address for operands that nothing reads


def _call(entry, args, *names, **fields):
    a = args()
    for name in names:
        setattr(a, name, AT)
    for name, v in fields.items():
        setattr(a, name, v)
    _lib.call(entry, bytes(a), 0)


@pytest.mark.parametrize("rows,channels", [((1 << 26) - 3, 8), ((1 << 26) - 1, 64), (1 << 26, 8), (1 << 24, 9)])
def test_residual_norm_rows(rows, channels):
    """Four rows a workgroup of 256 threads, or one where a row ends inside a chunk."""
    with pytest.raises(_lib.DfsKernelError, match="rows"):
        _call("dfs_residual_norm", _lib.ResidualNormArgs, "x", "h", rows=rows, channels=channels, dtype=0, norm=1,
              x_stride=channels, h_stride=channels)


@pytest.mark.parametrize("rows,k", [((1 << 28) - 15, 128), ((1 << 28) - 1, 5), (1 << 28, 1), ((1 << 25) - 1, 1025)])
def test_quantize_fp8_blocks(rows, k):
    """Sixteen blocks of 128 channels a workgroup."""
    with pytest.raises(_lib.DfsKernelError, match="too many blocks"):
        _call("dfs_quantize_fp8", _lib.QuantizeFp8Args, "x", "values", "scales", rows=rows, k=k, dtype=0, x_stride=k,
              values_stride=k, scales_stride=rows)


@pytest.mark.parametrize("rows,n,k,codes,out8", [
    ((1 << 28) - 15, 8, 128, False, False),     # x in 16 bits
    (227745, 30391, 141313, False, False),      # x in 16 bits, w's codes laid out anew in the same launch
    ((1 << 27) - 7, 130, 16, False, True),      # the result as codes
    ((1 << 27) - 7, 130, 16, True, True),
])
def test_linear_fp8_blocks(rows, n, k, codes, out8):
    """Sixteen blocks of 128 channels a workgroup, of x and of the result."""
    names = (("x_scales",) if codes else ()) + (("out8", "out8_scales") if out8 else ("out",))
    with pytest.raises(_lib.DfsKernelError, match="too many"):
        _call("dfs_linear_fp8", _lib.LinearFp8Args, "x", "w", "w_scales", "workspace", *names, rows=rows, n=n, k=k,
              x_dtype=3 if codes else 0, dtype=0, x_stride=k, w_stride=k, x_scales_stride=rows, w_scales_stride=n,
              out_stride=n, out8_stride=n, out8_scales_stride=rows, workspace_bytes=1 << 62)


@pytest.mark.parametrize("change", [{"residual_scale": 1e39}, {"residual_scale": -3.5e38}, {"eps": 1e39}, {"eps": float("inf")},
                                    {"post_norm": "rms", "post_eps": 4e38}])
def test_residual_norm_takes_fp32_numbers(change):
    """Options are fp32 in the kernel: past its range 1e39 * 0 was not a number."""
    x = torch.zeros(2, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="fp32"):
        ops.residual_norm(x, x, **change)
    names = {"x": AT, "y": AT, "out": AT, "h": AT, "rows": 2, "channels": 16, "norm": 1, "x_stride": 16, "y_stride": 16,
             "out_stride": 16, "h_stride": 16, "residual_scale": 1.0}
    with pytest.raises(_lib.DfsKernelError, match="fp32"):
        _call("dfs_residual_norm", _lib.ResidualNormArgs, **{**names, **change, "post_norm": int("post_norm" in change)})


@pytest.mark.parametrize("eps", [1e39, float("inf")])
def test_axial_rope_takes_fp32_eps(eps):
    q = torch.zeros(1, 2, 1, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="fp32"):
        ops.axial_rope(q, None, ops.RotaryAxes(8, (8,)), (), eps=eps)
    with pytest.raises(_lib.DfsKernelError, match="fp32"):
        _call("dfs_axial_rope", _lib.AxialRopeArgs, "q", "q_out", batch=1, tokens=2, q_heads=1, head_dim=8, axes=1, eps=eps)


@pytest.mark.parametrize("grid", [(), (4,), (2, 3, 4), (0, 4), (4, -1), (1 << 30, 4)])
def test_grid_rotary_refuses_another_grid(grid):
    """A grid of the axes behind the first, as ops.axial_rope takes it: tables of
    others put the wrong places to the axes."""
    with pytest.raises(ValueError, match="grid"):
        ops.GridRotary(ops.RotaryAxes(64, (24, 20, 20)), grid)
