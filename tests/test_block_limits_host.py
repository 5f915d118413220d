"""Sizes past what a launch holds (fewer than 2^32 threads) are refused by the C
entries before they launch. The pointers are never read: only refused calls are
made here."""
import pytest

from dfsattn_amd import _lib

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
